// Attention over the 8-bit paged cache, for many rows a sequence (prompts) and
// float16 queries: tiles of 128 rows on the tensor cores.
//
// The formulas are kv_attend.cu's. A block holds RT tiles of 128 rows' queries in
// shared memory and goes over KT keys at a time: S = Q K^T into tensor
// memory, the weights P = e^(s - m) (sv / largest sv) 2^7 as float16 over S,
// O += P V with P from tensor memory. Four kinds of warps hand tiles to each
// other by mbarriers, with two places of scores, so that the products of one
// tile of keys run beside the exponentials of another:
//   four a row tile   a row a thread: scores from tensor memory, masks, m and l in
//                     32 bits
//   four              the keys' and values' bytes, which bulk copies bring to shared
//                     memory RS tiles ahead, to float16 integers (exact) in the
//                     128-byte swizzled layout; once for all row tiles
//   one               asks for the bytes, their pages and scales
//   one               one thread issues the products
// Keys lie in shared memory with their dimensions contiguous, for both products:
// K-major for the first, N-major for the second, so nothing is transposed.
//
// m is let fall behind by up to 2^8 before O is scaled again (P <= 2^15 then; P
// reaches down to 2^-31 of the largest weight). 2^7 and float16's 11 bits for P
// are the choice's cost: 2^-12 of each weight.
//
// The products cut up to 2^-23 of O off each time, always downwards: 1.2e-3 over
// 200000 keys. So O is set aside every 8192 keys and the stretches are summed by
// rounding adds (5e-5 stays, a fifth of a float16 result's own rounding), in the
// workspace, 16 bytes a thread beside its neighbours': 2.3 us a stretch. Rows of a
// thread's own, 512 bytes apart, took 11; stretches of 4096 keys keep 2e-5, and a
// prompt over 8192 keys then takes 420 us instead of 414.
//
// Bound: the softmax warps (2200 cycles of a tile's 3350: the exponentials, one
// for 4 D flops, and what goes with them, on schedulers that the conversions
// share), then a segment's beginning and end, which nothing overlaps (about 20
// us; a block has a few). Measured on one B200, 32 query and 8 key/value heads of
// 128: 512 new tokens of 4 sequences over 8192 keys (266 GFLOP) 414 us, 643
// TFLOP/s; 4096 tokens on their own (137 GFLOP) 384 us, 358 TFLOP/s; prompts of
// three sequences (207 GFLOP) 404 us. Measured and left: one block of 128 rows
// twice on an SM, each converting for itself (346 TFLOP/s on the first case);
// products issued in a fixed order (head-of-line waits: 599 us against 499);
// descriptors as 64-bit sums (907 cycles to issue eight products against 541).
#include "kv_attend.cuh"
#include "tensor.cuh"

namespace shlo {

namespace {

constexpr int kRowsT = 128;  // rows of a tile: the lanes of tensor memory

__device__ __forceinline__ float ex2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void tm_ld16(uint32_t at, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t at, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\ntcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
// 64 columns, both loads on their way at once.
__device__ __forceinline__ void tm_ld64(uint32_t at, float (&v)[32], float (&u)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
               "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
               "tcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
                 "=f"(u[0]), "=f"(u[1]), "=f"(u[2]), "=f"(u[3]), "=f"(u[4]), "=f"(u[5]), "=f"(u[6]), "=f"(u[7]), "=f"(u[8]), "=f"(u[9]), "=f"(u[10]), "=f"(u[11]), "=f"(u[12]), "=f"(u[13]), "=f"(u[14]), "=f"(u[15]), "=f"(u[16]), "=f"(u[17]), "=f"(u[18]), "=f"(u[19]), "=f"(u[20]), "=f"(u[21]), "=f"(u[22]), "=f"(u[23]), "=f"(u[24]), "=f"(u[25]), "=f"(u[26]), "=f"(u[27]), "=f"(u[28]), "=f"(u[29]), "=f"(u[30]), "=f"(u[31])
               : "r"(at), "r"(at + 32)
               : "memory");
}
__device__ __forceinline__ void tm_st16f(uint32_t at, const float (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
               "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
               : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// `bytes` (a multiple of 16, both ends on 16-byte boundaries) from this GPU's memory, counted by barrier b.
__device__ __forceinline__ void copy_bulk(uint32_t to, const int8_t *from, uint32_t bytes, uint64_t *b) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
               "r"(bytes), "r"(smem_at(b))
               : "memory");
}
// (An operand's upper half never changes, its lower half is a 32-bit sum: the
// issuing warp's few instructions between two products bound their rate.)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t a_hi, uint32_t b, uint32_t b_hi, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %6, 0;\nmov.b64 x, {%1, %2};\nmov.b64 y, {%3, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n}\n" ::"r"(d), "r"(a), "r"(a_hi), "r"(b), "r"(b_hi), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t b_hi, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 y, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(b_hi), "r"(idesc), "r"(add)
      : "memory");
}
// Two bytes (sign bit flipped) as float16 integers.
template <int SEL>
__device__ __forceinline__ uint32_t half_pair_(uint32_t x) {
  const uint32_t r = __byte_perm(x, 0x64646464u, SEL);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&r), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ float2 bcast2(float x) { return make_float2(x, x); }

template <int DP>
struct Tiles {
  static constexpr int KT = DP == 256 ? 32 : 64;   // keys a tile
  static constexpr int RT = DP == 256 ? 1 : 2;     // row tiles
  static constexpr int ROWS = RT * kRowsT;
  static constexpr int THREADS = (4 * RT + 6) * 32;
  static constexpr int O_COL = RT * 2 * KT;        // S of tile r, place b at (2 r + b) KT; P lies over S, two weights a column
  static constexpr int TM_COLS = 512;
  static constexpr int Q_BYTES = kRowsT * DP * 2, K_BYTES = KT * DP * 2;
  static constexpr int NS = 3, RS = 3;             // stages of keys and values: as float16 (the scores run two tiles ahead of the outputs), as bytes
  static constexpr int GROUPS = KT / 16;
  static constexpr int META = 2 * GROUPS + 4;      // a tile's scales of keys and of values, its holes, whether the scores need care
  static constexpr int NM = 8;                     // such sets: those asked for (RS), converted (NS) and under the softmax
  static constexpr int STRETCH = 8192 / KT;        // tiles whose products O sums up before it is set aside
  static constexpr int BATCH = 1024;
  static constexpr int MISC = 256 + (THREADS + 4) * 8 + 64 + BATCH * 4 + NM * META * 4 + 64;
  static constexpr int BYTES = 1024 + RT * Q_BYTES + 2 * NS * K_BYTES + RS * K_BYTES + MISC;
};

// Where a block sets O's earlier stretches aside, behind all blocks' partials:
// [DP / 4][row] float4, then m a row.
template <int DP>
__device__ __forceinline__ float *aside_at(const AttendArgs &a) {
  constexpr int ROWS = Tiles<DP>::ROWS;
  return a.partials + (int64_t)gridDim.x * 2 * ROWS * (DP + 2) + (int64_t)blockIdx.x * ROWS * (DP + 1);
}

template <int DP>
__global__ void __launch_bounds__(Tiles<DP>::THREADS, 1) k_kv_attend_tiles(const AttendArgs a, int min_gran) {
  using S = Tiles<DP>;
  constexpr int KT = S::KT, GROUPS = S::GROUPS, META = S::META, NM = S::NM, RT = S::RT, NS = S::NS, RS = S::RS, ROWS = S::ROWS, THREADS = S::THREADS, STRETCH = S::STRETCH;
  extern __shared__ uint8_t raw_smem[];
  uint8_t *const base = raw_smem + ((1024 - (smem_at(raw_smem) & 1023)) & 1023);
  uint8_t *const qs = base, *const ks = qs + RT * S::Q_BYTES, *const vs = ks + NS * S::K_BYTES;
  uint8_t *const raw = vs + NS * S::K_BYTES;  // [RS][keys, values][KT][D]
  // Barriers. Of a stage of bytes: there, used up. Of a stage of float16: there, used up. Of
  // a row tile and a place of scores: scores done, weights there, outputs done.
  uint64_t *const kv_full = reinterpret_cast<uint64_t *>(raw + RS * S::K_BYTES), *const kv_free = kv_full + 4, *const raw_full = kv_full + 20, *const raw_free = kv_full + 24;
  uint64_t *const qk_done = kv_full + 8, *const p_full = kv_full + 12, *const pv_done = kv_full + 16, *const drained = kv_full + 28;
  long long *const sched = reinterpret_cast<long long *>(kv_full + 32);
  Place *const place = reinterpret_cast<Place *>(sched + THREADS + 4);
  int *const batch = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(place) + 64);
  float *const meta = reinterpret_cast<float *>(batch + S::BATCH);
  unsigned *const flag = reinterpret_cast<unsigned *>(meta + NM * META);
  volatile int *const gone = reinterpret_cast<volatile int *>(flag + 1);
  uint32_t *const tm_slot = reinterpret_cast<uint32_t *>(flag + 2);
  float *const vtop_s = reinterpret_cast<float *>(flag + 3);
  int *const asked = reinterpret_cast<int *>(flag + 4);  // tiles of the segment whose bytes were asked for
  float *const fac = reinterpret_cast<float *>(qs);  // a join's factors, when no tile is under way
  static_assert(sizeof(Place) <= 64, "its room in shared memory");
  static_assert(2 * (kJoin<ROWS> + 1) * ROWS * 4 <= RT * S::Q_BYTES + (2 * NS + RS) * S::K_BYTES, "a join's factors");

  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int D = a.pool.head_dim, PT = 1 << a.page_shift;
  Line line;
  BatchArrays ba;
  if (!schedule<ROWS, KT, THREADS>(a, min_gran, sched, batch, S::BATCH, ba, line)) return;

  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      bar_init(kv_full + i, 4);
      bar_init(kv_free + i, 1);
    }
    for (int i = 0; i < RS; i++) {
      bar_init(raw_full + i, 1);
      bar_init(raw_free + i, 4);
    }
    for (int i = 0; i < 2 * RT; i++) {
      bar_init(qk_done + i, 1);
      bar_init(p_full + i, 4);
      bar_init(pv_done + i, 1);
    }
    bar_init(drained, 1);
    *gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tm_slot)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  seek<ROWS, KT, THREADS>(a, ba, line, place);
  tm_before();
  __syncthreads();
  tm_after();
  const uint32_t tm = *tm_slot;
  Place p = *place;
  Segment sg;
  // Tiles of keys of earlier segments: tile t has the stage t % NS (its barriers'
  // phase t / NS); and of each row tile, which may have had fewer: its tile t has
  // the place of scores t % 2 (phase t / 2).
  uint32_t done = 0, turns[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) turns[r] = 0;

  while (next_segment<ROWS, KT>(a, ba, p, sg)) {
    // (After a wait that was given up the units are only counted, all of them: the
    // counters are zero again for the next launch. What is joined then is not valid.)
    if (!*gone) {
    const int key0 = (sg.t.lo / KT + sg.off) * KT;
    const int32_t *table = a.batch.tables + (int64_t)sg.t.seq * a.batch.table_stride;
    auto page_at = [&](int key) -> int {  // -1: no row of the tile sees a key of these 16, or there is no page
      if (key >= sg.t.hi || key + 16 <= sg.t.lo) return -1;
      const int pg = __ldg(table + (key >> a.page_shift));
      return pg >= 0 && pg < a.pool.pages ? pg : -1;
    };
    const int rts = (sg.t.rows + kRowsT - 1) / kRowsT;  // row tiles with rows
    const int n = sg.take;
    // The asking warp's: pages and scales are held across its lanes, 32 groups of 16
    // keys (TL tiles: a stretch) at a time, and asked for a stretch ahead: on a
    // tile's own path they would be two more waits for L2.
    constexpr int TL = 32 / GROUPS;
    const int64_t tok = a.pool.token_stride;
    int pg = -1, pg_next = -1;
    int64_t off = 0, off_next = 0;  // of the group's first key
    float kscale = 0.0f, vscale = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    auto pages = [&](int j) {
      const int key = key0 + j * KT + lane * 16;
      pg_next = j + lane / GROUPS < n ? page_at(key) : -1;
      off_next = (int64_t)sg.head * a.pool.head_stride + (int64_t)max(pg_next, 0) * a.pool.page_stride + (int64_t)(key & (PT - 1)) * tok;
    };
    auto ask_scales = [&]() {
      ks_next = vs_next = 0.0f;
      if (pg_next >= 0) {
        ks_next = __ldg(a.pool.k_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pg_next * a.pool.scale_page_stride));
        vs_next = __ldg(a.pool.v_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pg_next * a.pool.scale_page_stride));
      }
    };
    auto turn = [&]() {  // to the next stretch
      pg = pg_next;
      off = off_next;
      kscale = ks_next;
      vscale = vs_next;
    };
    // The bytes of tile j into its stage. What is not there is left as it lies: any
    // byte is a finite value, and no row sees it.
    auto copy_tile = [&](int j) {
      const uint32_t rs = (done + j) % RS, to = smem_at(raw) + rs * S::K_BYTES;
      uint64_t *const bar = raw_full + rs;
      const int at = j % TL * GROUPS;
      const bool joined = tok == D;  // a group's 16 rows are one run of bytes: a lane copies one group's keys or values
      const int group = joined ? lane / 2 : lane % GROUPS;
      const int q = __shfl_sync(~0u, pg, (at + group) & 31);
      const int64_t o = __shfl_sync(~0u, off, (at + group) & 31);
      if (joined) {
        if (lane < 2 * GROUPS && q >= 0)
          copy_bulk(to + ((lane & 1) * KT + group * 16) * D, (lane & 1 ? a.pool.v : a.pool.k) + o, 16 * D, bar);
      } else {
#pragma unroll 1
        for (int i = lane; i < 2 * KT; i += 32) {  // one row a copy; GROUPS divides 32, so a lane keeps its group
          const int kv = i / KT, row = i % KT / GROUPS;
          if (q >= 0) copy_bulk(to + (kv * KT + group * 16 + row) * D, (kv ? a.pool.v : a.pool.k) + o + row * tok, D, bar);
        }
      }
    };
    // Its scales, for the softmax; and the count of its bytes, with which they are
    // handed on (a tile is complete when both the count and the bytes are there).
    auto count_tile = [&](int j, float vtop) {
      const int at = j % TL * GROUPS;
      float *mt = meta + (done + j) % NM * META;
      const float c = kscale * a.scale_log2;
      // a scale that is not finite makes the weights of the keys that are seen NaN
      const float ratio = !(fabsf(vscale) <= 3.402823466e38f) ? __int_as_float(0x7fc00000) : vtop > 0.0f ? __fdiv_rn(vscale, vtop) * 128.0f : 0.0f;
      const uint32_t group_bits = (1u << GROUPS) - 1;
      const uint32_t holes = __ballot_sync(~0u, pg < 0) >> at & group_bits, odd = __ballot_sync(~0u, !(c >= 0.0f)) >> at & group_bits;
      if (lane >= at && lane < at + GROUPS) {
        mt[lane - at] = c;
        mt[GROUPS + lane - at] = ratio;
      }
      if (lane == 0) {
        mt[2 * GROUPS] = __int_as_float((int)holes);
        mt[2 * GROUPS + 1] = __int_as_float((int)odd);
      }
      __syncwarp();
      const uint32_t bytes = 2u * (GROUPS - __popc(holes)) * 16u * (uint32_t)D;
      if (lane == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(raw_full + (done + j) % RS)), "r"(bytes) : "memory");
    };
    constexpr int ASKER = 4 * RT + 5;
    static_assert(RS <= TL / 2, "the first tiles are of one stretch, and the next one's scales are yet to ask for");
    if (warp == ASKER) {
      pages(0);
      ask_scales();
      turn();
      for (int j = 0; j < RS && j < n; j++) copy_tile(j);
      if (lane == 0) *asked = min(RS, n);
    }
    // The queries, and the largest finite scale of the segment's values.
    if (tid == 0) *vtop_s = 0.0f;
    __syncthreads();
    {
      constexpr int PIECES = DP / 8, BATCH = 4;
      const int items = rts * kRowsT * PIECES;
      for (int i0 = tid; i0 < items; i0 += BATCH * THREADS) {  // several loads on their way
        uint4 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          const int i = i0 + k * THREADS, row = i / PIECES, d = i % PIECES * 8, r = sg.t.row0 + row;
          v[k] = make_uint4(0u, 0u, 0u, 0u);
          if (row < sg.t.rows && d < D) {
            const __half *q = static_cast<const __half *>(a.q) + (int64_t)(sg.t.start + r / a.group) * a.q_token +
                              (int64_t)(sg.head * a.group + r % a.group) * a.q_head + d;
            if (a.q_wide) {
              v[k] = *reinterpret_cast<const uint4 *>(q);
            } else {
              __half h[8];
#pragma unroll
              for (int j = 0; j < 8; j++) h[j] = q[j];
              memcpy(&v[k], h, 16);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
          const int i = i0 + k * THREADS, row = i / PIECES, c = i % PIECES;
          if (i < items)
            *reinterpret_cast<uint4 *>(qs + (row / kRowsT) * S::Q_BYTES + (c / 8) * (kRowsT * 128) + (row % kRowsT) * 128 +
                                       (((c % 8) ^ (row & 7)) * 16)) = v[k];
        }
      }
      float top = 0.0f;
      for (int i = tid; i < sg.take * GROUPS; i += THREADS) {
        const int q = page_at(key0 + i * 16);
        if (q >= 0) {
          const float s = fabsf(__ldg(a.pool.v_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)q * a.pool.scale_page_stride)));
          if (s <= 3.402823466e38f) top = fmaxf(top, s);
        }
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
      if (lane == 0 && top > 0.0f) atomicMax(reinterpret_cast<int *>(vtop_s), __float_as_int(top));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    const float vtop = *vtop_s;

    if (warp == ASKER) {
      // ---- bytes, pages and scales ----
      for (int j = 0; j < RS && j < n; j++) count_tile(j, vtop);
      pages(TL);
      for (int j = RS; j < n; j++) {
        const uint32_t t = done + j;
        if (j % TL == TL / 2) ask_scales();
        if (j % TL == 0) {
          turn();
          pages(j + TL);
        }
        if (!warp_wait(raw_free + t % RS, (t / RS & 1) ^ 1, gone)) break;
        copy_tile(j);
        count_tile(j, vtop);
        if (lane == 0) *asked = j + 1;
      }
    } else
    if (warp == 4 * RT + 4) {
      // ---- products ----
      {
        // float32 sums, float16 operands; 128 rows by KT keys, and by D (the values are N-major)
        const uint32_t id_s = 1u << 4 | (uint32_t)(KT >> 3) << 17 | (uint32_t)(kRowsT >> 4) << 24;
        const uint32_t id_o = 1u << 4 | 1u << 16 | (uint32_t)(D >> 3) << 17 | (uint32_t)(kRowsT >> 4) << 24;
        const uint64_t q_op = operand(smem_at(qs), 16), k_op = operand(smem_at(ks), 16), v_op = operand(smem_at(vs), KT * 128);
        const uint32_t kq_hi = (uint32_t)(k_op >> 32), v_hi = (uint32_t)(v_op >> 32);
        // Whatever is ready is issued, of either row tile: no wait for one holds up the
        // other. The scores run at most two tiles of keys ahead of the outputs.
        int next_s[RT], next_o[RT], left = n * rts;
#pragma unroll
        for (int r = 0; r < RT; r++) next_s[r] = next_o[r] = 0;
        uint64_t t0 = 0;
        const bool hurried = a.give_up && blockIdx.x % a.give_up == 0;
        for (uint32_t idle = 0; left > 0;) {
          bool any = false;
#pragma unroll
          for (int r = 0; r < RT; r++) {
            if (r >= rts) break;
            {
              const int j = next_o[r];
              const uint32_t st = (done + j) % NS, t = turns[r] + j, b = t & 1;
              if (j < next_s[r] && __all_sync(~0u, bar_test(p_full + 2 * r + b, t >> 1 & 1))) {
                tm_after();
                const uint32_t vb = (uint32_t)v_op + st * (S::K_BYTES >> 4);
                const uint32_t d = tm + S::O_COL + r * DP, w = tm + (2 * r + b) * KT;
                if (elect_one()) {
                  mma_ts(d, w, vb, v_hi, id_o, j % STRETCH != 0);
#pragma unroll
                  for (int k = 1; k < KT / 16; k++) mma_ts(d, w + k * 8, vb + (k * 2048 >> 4), v_hi, id_o, 1);
                  tm_commit(pv_done + 2 * r + b);
                  if (rts == 1 || next_o[RT - 1 - r] > j) tm_commit(kv_free + st);  // the last row tile's
                }
                __syncwarp();
                next_o[r]++;
                left--;
                any = true;
              }
            }
            {
              const int j = next_s[r];
              const uint32_t st = (done + j) % NS, t = turns[r] + j, b = t & 1;
              // (the scores' place is free when the product that read its weights is done)
              if (j < n && (j < 2 || (next_o[r] >= j - 1 && __all_sync(~0u, bar_test(pv_done + 2 * r + b, (t >> 1 & 1) ^ 1)))) &&
                  __all_sync(~0u, bar_test(kv_full + st, (done + j) / NS & 1))) {
                tm_after();
                const uint32_t qb = (uint32_t)q_op + r * (S::Q_BYTES >> 4), kb = (uint32_t)k_op + st * (S::K_BYTES >> 4);
                const uint32_t d = tm + (2 * r + b) * KT;
                if (elect_one()) {
#pragma unroll
                  for (int k = 0; k < DP / 16; k++)
                    if (k * 16 < D)
                      mma_ss(d, qb + ((k / 4) * (kRowsT * 128) + (k % 4) * 32 >> 4), kq_hi, kb + ((k / 4) * (KT * 128) + (k % 4) * 32 >> 4), kq_hi,
                             id_s, k > 0);
                  tm_commit(qk_done + 2 * r + b);
                }
                __syncwarp();
                next_s[r]++;
                any = true;
              }
            }
          }
          if (any) {
            idle = 0;
          } else if ((++idle & 255) == 0 || hurried) {  // two seconds of nothing: give up
            uint64_t now;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (idle == 256) t0 = now;
            if (__any_sync(~0u, *gone || hurried || now - t0 > kWaitLimitNs)) {
              *gone = 1;
              break;
            }
          }
        }
      }
    } else if (warp >= 4 * RT && warp < 4 * RT + 4) {
      // ---- bytes to float16 ----
      constexpr int CH = DP / 16, KPP = 128 / CH, NI = KT / KPP;  // pieces a key, keys a pass, passes
      const int pt = tid - 128 * RT, key_in = pt / CH, ch = pt % CH;
      const bool live = ch * 16 < D;
      // where this thread's two pieces of 8 go in a stage
      const int db = ch / 4, c0 = (ch % 4) * 2, first = db & 1;  // (the pieces in an order that keeps eight lanes on eight bank groups)
      const int to1 = db * (KT * 128) + key_in * 128 + (((c0 + first) ^ (key_in & 7)) * 16);
      const int to2 = db * (KT * 128) + key_in * 128 + (((c0 + 1 - first) ^ (key_in & 7)) * 16);
      auto put = [&](uint8_t *to, const uint8_t *from) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const uint4 r = *reinterpret_cast<const uint4 *>(from + i * KPP * D);
          const uint32_t w[4] = {r.x ^ 0x80808080u, r.y ^ 0x80808080u, r.z ^ 0x80808080u, r.w ^ 0x80808080u};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            h[2 * k] = half_pair_<0x4140>(w[k]);
            h[2 * k + 1] = half_pair_<0x4342>(w[k]);
          }
          const uint4 lo4 = make_uint4(h[0], h[1], h[2], h[3]), hi4 = make_uint4(h[4], h[5], h[6], h[7]);
          *reinterpret_cast<uint4 *>(to + to1 + i * (KPP * 128)) = first ? hi4 : lo4;
          *reinterpret_cast<uint4 *>(to + to2 + i * (KPP * 128)) = first ? lo4 : hi4;
        }
      };
      for (int j = 0; j < n; j++) {
        const uint32_t t = done + j, st = t % NS, rs = t % RS;
        if (!warp_wait(raw_full + rs, t / RS & 1, gone)) break;
        if (j >= NS && !warp_wait(kv_free + st, (t / NS & 1) ^ 1, gone)) break;
        if (live) {
          const uint8_t *from = raw + rs * S::K_BYTES + key_in * D + ch * 16;
          put(ks + st * S::K_BYTES, from);
          put(vs + st * S::K_BYTES, from + KT * D);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(kv_full + st);
        if (lane == 0) bar_arrive(raw_free + rs);  // this warp has read the bytes
      }
    } else {
      // ---- weights ----
      const int rt = warp / 4, row = tid;
      if (rt < rts) {
      const int pos = sg.t.first + (sg.t.row0 + row) / a.group;
      const int lo = row_lo(a, pos), hi = row < sg.t.rows ? row_hi(a, sg.t.keys, pos) : 0;
      const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16, o_at = tm + S::O_COL + rt * DP + lanes;
      const uint32_t mine = RT == 2 && rt ? turns[RT - 1] : turns[0];
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < n; j++) {
        const uint32_t t = mine + j, b = t & 1, ph = (t >> 1) & 1, st = (done + j) % NS;
        const uint32_t s_at = tm + (2 * rt + b) * KT + lanes;
        if (__builtin_expect(j > 0 && j % STRETCH == 0, 0)) {
          // O is added to its earlier stretches, and the next product writes it anew.
          const uint32_t u = t - 1;
          if (!warp_wait(pv_done + 2 * rt + (u & 1), (u >> 1) & 1, gone)) {
            ok = false;
            break;
          }
          tm_after();
          float *const aside = aside_at<DP>(a);
          const float f = j > STRETCH ? join_factor(aside[ROWS * DP + row], m) : 0.0f;
          aside[ROWS * DP + row] = m;
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {  // 32 values' loads on their way
            float4 *const to = reinterpret_cast<float4 *>(aside) + c0 / 4 * ROWS + row, s[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
              s[x] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (j > STRETCH) s[x] = to[x * ROWS];
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
              if (c0 + h * 16 >= D) break;
              float w[16];
              tm_ld16(o_at + c0 + h * 16, w);
#pragma unroll
              for (int x = 0; x < 4; x++) {
                const float4 v = s[h * 4 + x];
                to[(h * 4 + x) * ROWS] = make_float4(__fmaf_rn(f, v.x, w[4 * x]), __fmaf_rn(f, v.y, w[4 * x + 1]),
                                                     __fmaf_rn(f, v.z, w[4 * x + 2]), __fmaf_rn(f, v.w, w[4 * x + 3]));
              }
            }
          }
        }
        if (!warp_wait(kv_full + st, (done + j) / NS & 1, gone) || !warp_wait(qk_done + 2 * rt + b, ph, gone)) {
          ok = false;
          break;
        }
        tm_after();
        const float *mt = meta + (done + j) % NM * META;
        const uint32_t holes = (uint32_t)__float_as_int(mt[2 * GROUPS]);
        const int key = key0 + j * KT;
        // With care: keys that some rows do not see, scales that are negative or no numbers.
        const bool care = key < sg.t.lo_all || key + KT > sg.t.hi_all || holes || __float_as_int(mt[2 * GROUPS + 1]);
        float v[KT / 32][32];
        if constexpr (KT == 64) tm_ld64(s_at, v[0], v[1]);
        else tm_ld32(s_at, v[0]);
        float top = -INFINITY;
        if (!care) {
#pragma unroll
          for (int g = 0; g < GROUPS; g++) {
            float x = v[g / 2][g % 2 * 16];
#pragma unroll
            for (int i = 1; i < 16; i++) x = fmaxf(x, v[g / 2][g % 2 * 16 + i]);
            top = fmaxf(top, x * mt[g]);
          }
        } else {
#pragma unroll
          for (int g = 0; g < GROUPS; g++) {
            const float c = mt[g];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int kk = key + g * 16 + i;
              float x = v[g / 2][g % 2 * 16 + i] * c;
              if (kk < lo || kk >= hi || (holes >> g & 1)) x = -INFINITY;
              v[g / 2][g % 2 * 16 + i] = x;
              top = fmaxf(top, x);
            }
          }
        }
        // Rows whose maximum rose by more than 8 (or that saw their first key) bring
        // their whole warp up to date.
        if (__any_sync(~0u, top > m + 8.0f || (m == -INFINITY && top > m))) {
          const float mn = fmaxf(m, top);
          const float f = m == -INFINITY ? 0.0f : ex2_(m - mn);
          l *= f;
          m = mn;
          if (j % STRETCH) {  // (a stretch's first product writes O)
            const uint32_t u = t - 1;
            if (!warp_wait(pv_done + 2 * rt + (u & 1), (u >> 1) & 1, gone)) {
              ok = false;
              break;
            }
            tm_after();
#pragma unroll 1
            for (int ch = 0; ch * 16 < D; ch++) {
              float w[16];
              tm_ld16(o_at + ch * 16, w);
#pragma unroll
              for (int x = 0; x < 16; x++) w[x] *= f;
              tm_st16f(o_at + ch * 16, w);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float2 sum = make_float2(0.0f, 0.0f);
        uint32_t w[KT / 2];
        const float2 sub = bcast2(-ref);
        if (!care) {
#pragma unroll
          for (int g = 0; g < GROUPS; g++) {
            const float2 c = bcast2(mt[g]), r = bcast2(mt[GROUPS + g]);
#pragma unroll
            for (int x = 0; x < 8; x++) {
              const int i = g % 2 * 16 + 2 * x;
              const float2 z = __ffma2_rn(make_float2(v[g / 2][i], v[g / 2][i + 1]), c, sub);
              const float2 e = make_float2(ex2_(z.x), ex2_(z.y));
              sum = __fadd2_rn(sum, e);
              const float2 q = __fmul2_rn(e, r);
              const __half2 h = __floats2half2_rn(q.x, q.y);
              w[g * 8 + x] = *reinterpret_cast<const uint32_t *>(&h);
            }
          }
        } else {  // (scaled already)
#pragma unroll
          for (int g = 0; g < GROUPS; g++) {
            const float2 r = bcast2(mt[GROUPS + g]);
#pragma unroll
            for (int x = 0; x < 8; x++) {
              const int i = g % 2 * 16 + 2 * x;
              const float2 s2 = make_float2(v[g / 2][i], v[g / 2][i + 1]);
              const float2 z = __fadd2_rn(s2, sub);
              const float2 e = make_float2(ex2_(z.x), ex2_(z.y));
              sum = __fadd2_rn(sum, e);
              float2 q = __fmul2_rn(e, r);  // 0 times what is not a number is not 0
              if (s2.x == -INFINITY) q.x = 0.0f;
              if (s2.y == -INFINITY) q.y = 0.0f;
              const __half2 h = __floats2half2_rn(q.x, q.y);
              w[g * 8 + x] = *reinterpret_cast<const uint32_t *>(&h);
            }
          }
        }
        l += sum.x + sum.y;
        if constexpr (KT == 64) tm_st32(s_at, w);
        else tm_st16(s_at, w);
        tm_wait_st();
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(p_full + 2 * rt + b);
      }
      if (ok) {
        const uint32_t u = mine + n - 1;
        ok = warp_wait(pv_done + 2 * rt + (u & 1), (u >> 1) & 1, gone);
      }
      tm_after();
      if (ok) {
        const bool whole = sg.take == sg.units;
        float *const part = whole ? nullptr : partial_at<ROWS, DP>(a, blockIdx.x, sg.off == 0);
        const float *const aside = aside_at<DP>(a);
        const float f_aside = n > STRETCH ? join_factor(aside[ROWS * DP + row], m) : 0.0f;
        const int r = sg.t.row0 + min(row, sg.t.rows - 1);
        __half *const to = static_cast<__half *>(a.out) + (int64_t)(sg.t.start + r / a.group) * a.out_token +
                           (int64_t)(sg.head * a.group + r % a.group) * a.out_head;
        float scale = vtop * 0x1p-7f;
        if (whole) scale = l == 0.0f ? 0.0f : scale / l;
        const bool empty = whole && l == 0.0f;  // a row that saw nothing: 0, whatever lies in O
#pragma unroll 1
        for (int ch = 0; ch * 16 < D; ch++) {
          float v[16];
          tm_ld16(o_at + ch * 16, v);
          if (row < sg.t.rows) {
            if (n > STRETCH) {
#pragma unroll
              for (int x = 0; x < 4; x++) {
                const float4 s = reinterpret_cast<const float4 *>(aside)[(ch * 4 + x) * ROWS + row];
                v[4 * x] = __fmaf_rn(f_aside, s.x, v[4 * x]);
                v[4 * x + 1] = __fmaf_rn(f_aside, s.y, v[4 * x + 1]);
                v[4 * x + 2] = __fmaf_rn(f_aside, s.z, v[4 * x + 2]);
                v[4 * x + 3] = __fmaf_rn(f_aside, s.w, v[4 * x + 3]);
              }
            }
#pragma unroll
            for (int x = 0; x < 16; x++) v[x] = empty ? 0.0f : v[x] * scale;
            if (!whole) {
#pragma unroll
              for (int x = 0; x < 4; x++)
                *reinterpret_cast<float4 *>(part + row * DP + ch * 16 + 4 * x) = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
            } else {
              __half2 h[8];
#pragma unroll
              for (int x = 0; x < 8; x++) h[x] = __floats2half2_rn(v[2 * x], v[2 * x + 1]);
              if (a.out_wide == 2) {
                uint4 w[2];
                memcpy(w, h, 32);
                *reinterpret_cast<uint4 *>(to + ch * 16) = w[0];
                *reinterpret_cast<uint4 *>(to + ch * 16 + 8) = w[1];
              } else {
#pragma unroll
                for (int x = 0; x < 8; x++) {
                  to[ch * 16 + 2 * x] = h[x].x;
                  to[ch * 16 + 2 * x + 1] = h[x].y;
                }
              }
            }
          }
        }
        if (row < sg.t.rows) {
          if (whole) {
            write_lse(a, sg.t, sg.head, row, m, l);
          } else {
            part[ROWS * DP + row] = m;
            part[ROWS * DP + ROWS + row] = l;
          }
        }
      }
      tm_before();
      }
    }
    done += n;
#pragma unroll
    for (int r = 0; r < RT; r++) turns[r] += r < rts ? n : 0;
    __syncthreads();
    tm_after();
    if (*gone) {
      // A warp gave up: the results are not valid, and the host is told. The bytes and
      // products that are on the way land before the block leaves its memory.
      if (warp == ASKER)
        for (int j = max(0, *asked - RS); j < *asked; j++) bar_drain(raw_full + (done - n + j) % RS, (done - n + j) / RS & 1);
      if (warp == 4 * RT + 4) {
        if (elect_one()) tm_commit(drained);
        __syncwarp();
        bar_drain(drained, 0);
      }
      __syncthreads();
    }
    }
    if (sg.take != sg.units) arrive<__half, ROWS, DP, THREADS>(a, sg, line, fac, flag);
  }
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(S::TM_COLS));
  if (tid == 0 && *gone && a.err) *a.err = 1;
}

// A chunk has at least so many granules (of 64 keys): its partial result, 256 rows
// of 32 bits, costs about as much as two to write and to join.
constexpr int kMinGranules = 4;

template <int DP>
int launch(AttendArgs a, int sms, int device, cudaStream_t st) {
  using S = Tiles<DP>;
  auto *kern = k_kv_attend_tiles<DP>;
  static std::atomic<uint64_t> allowed{0};
  SHLO_TRY(allow_smem((const void *)kern, S::BYTES, allowed, device));
  a.slots = (int)(((int64_t)a.batch.tokens * a.group) / S::ROWS + a.batch.seqs);
  const int64_t room = ((int64_t)a.batch.table_pages << a.page_shift) / S::KT + 1;
  int64_t most = (int64_t)a.slots * a.pool.heads;
  most = most > (1 << 20) ? most : most * room;
  int64_t grid = most < sms ? most : sms;
  if (grid > kAttendMaxBlocks) grid = kAttendMaxBlocks;
  if (grid < 1) grid = 1;
  kern<<<(unsigned)grid, S::THREADS, S::BYTES, st>>>(a, kMinGranules);
  return launch_check("kv_attend");
}

}  // namespace

size_t attend_tiles_partial_bytes(int sms) {
  const size_t blocks = sms < kAttendMaxBlocks ? sms : kAttendMaxBlocks;
  size_t rows = (size_t)Tiles<256>::ROWS * (256 + 2);
  if ((size_t)Tiles<128>::ROWS * (128 + 2) > rows) rows = (size_t)Tiles<128>::ROWS * (128 + 2);
  return blocks * 3 * rows * 4;  // two partials, and what is set aside
}

int launch_attend_tiles(const AttendArgs &a, int sms, int device, cudaStream_t st) {
  const int D = a.pool.head_dim;
  if (D <= 64) return launch<64>(a, sms, device, st);
  if (D <= 128) return launch<128>(a, sms, device, st);
  return launch<256>(a, sms, device, st);
}

}  // namespace shlo
