// Attention over the 8-bit paged cache, for many rows a sequence (prompts) and
// float16 queries: tiles of 128 rows on the tensor cores.
//
// The formulas are kv_attend.cu's. A block holds 128 rows' queries in shared
// memory and goes over KT keys at a time: S = Q K^T into tensor memory, the
// weights P = e^(s - m) (sv / largest sv) 2^7 as float16 over S, O += P V with P
// from tensor memory. Two kinds of warps hand tiles to each other by
// mbarriers:
//   0-3  a row a thread: scores from tensor memory, twice (the maximum first, then
//        the weights: 128 scores a row do not stay in registers beside a second
//        block's), masks, m and l in 32 bits
//   4-7  the keys' and values' bytes from global memory, asked for a tile ahead,
//        to float16 integers (exact) in the 128-byte swizzled layout
//   0    one thread of it issues the products (a warp of its own would cost every
//        thread 16 registers)
// Keys lie in shared memory with their dimensions contiguous, for both products:
// K-major for the first, N-major for the second, so nothing is transposed.
//
// m is let fall behind by up to 2^8 before O is scaled again (P <= 2^15 then; P
// reaches down to 2^-31 of the largest weight). 2^7 and float16's 11 bits for P
// are the choice's cost: 2^-12 of each weight.
//
// Bound: the exponentials (one for 4 DP flops) and the first product's and the
// second's turns on the tensor cores; two blocks an SM (up to 128 dimensions)
// fill each other's waits.
#include "kv_attend.cuh"

namespace shlo {

namespace {

constexpr int kRowsT = 128;
constexpr int kThreadsT = 256;

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok) : "r"(smem_at(b)), "r"(parity) : "memory");
  return ok != 0;
}
// A wait of two seconds at most; it ends early when another warp gave up.
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity, volatile int *gone) {
  if (bar_try(b, parity)) return true;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  for (uint32_t i = 1;; i++) {
    if (bar_try(b, parity)) return true;
    if ((i & 255) == 0) {
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
      if (*gone || t - t0 > 2000000000ull) {
        *gone = 1;
        return false;
      }
    }
  }
}
// The same for a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile int *gone) {
  return __all_sync(~0u, bar_wait(b, parity, gone));
}
__device__ __forceinline__ float ex2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void tm_ld32(uint32_t at, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t at, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
      "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
      "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint64_t *b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_at(b)) : "memory");
}
// Shared-memory operands in the 128-byte swizzle: rows of 128 bytes, eight rows
// a group of 1024; `lead` bytes between 64-value blocks (N-major operands).
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead) {
  return (uint64_t)((at >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
      "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a),
      "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// Two bytes (sign bit flipped) as float16 integers.
template <int SEL>
__device__ __forceinline__ uint32_t half_pair_(uint32_t x) {
  const uint32_t r = __byte_perm(x, 0x64646464u, SEL);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&r), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&v);
}

template <int DP>
struct Tiles {
  static constexpr int KT = DP == 256 ? 64 : 128;  // keys a tile
  static constexpr int PER_SM = DP == 256 ? 1 : 2;
  static constexpr int TM_COLS = DP == 256 ? 512 : 256;
  static constexpr int S_COL = 0, O_COL = KT;      // P lies over S, two weights a column
  static constexpr int Q_BYTES = kRowsT * DP * 2, K_BYTES = KT * DP * 2;
  static constexpr int GROUPS = KT / 16;
  static constexpr int BATCH = 258;
  static constexpr int MISC = 64 + (kThreadsT + 4) * 8 + 64 + BATCH * 4 + 2 * (2 * GROUPS + 2) * 4 + 64;
  static constexpr int BYTES = 1024 + Q_BYTES + 2 * K_BYTES + MISC;
};

template <int DP>
__global__ void __launch_bounds__(kThreadsT, Tiles<DP>::PER_SM) k_kv_attend_tiles(const AttendArgs a, int min_gran) {
  using S = Tiles<DP>;
  constexpr int KT = S::KT, GROUPS = S::GROUPS;
  extern __shared__ uint8_t raw_smem[];
  uint8_t *const base = raw_smem + ((1024 - (smem_at(raw_smem) & 1023)) & 1023);
  uint8_t *const qs = base, *const ks = qs + S::Q_BYTES, *const vs = ks + S::K_BYTES;
  uint64_t *const bars = reinterpret_cast<uint64_t *>(vs + S::K_BYTES);
  uint64_t *const k_full = bars, *const v_full = bars + 1, *const qk_done = bars + 2, *const p_full = bars + 3, *const pv_done = bars + 4;
  long long *const sched = reinterpret_cast<long long *>(bars + 8);
  Place *const place = reinterpret_cast<Place *>(sched + kThreadsT + 4);
  int *const batch = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(place) + 64);
  float *const meta = reinterpret_cast<float *>(batch + S::BATCH);  // [2][2 GROUPS + 2]: scales, holes
  unsigned *const flag = reinterpret_cast<unsigned *>(meta + 2 * (2 * GROUPS + 2));
  volatile int *const gone = reinterpret_cast<volatile int *>(flag + 1);
  uint32_t *const tm_slot = reinterpret_cast<uint32_t *>(flag + 2);
  float *const vtop_s = reinterpret_cast<float *>(flag + 3);
  float *const fac = reinterpret_cast<float *>(qs);  // a join's factors, when no tile is under way
  static_assert(sizeof(Place) <= 64, "its room in shared memory");
  static_assert(2 * (kJoin<kRowsT> + 1) * kRowsT * 4 <= S::Q_BYTES + 2 * S::K_BYTES, "a join's factors");

  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int D = a.pool.head_dim, PT = 1 << a.page_shift;
  Line line;
  BatchArrays ba;
  if (!schedule<kRowsT, KT, kThreadsT>(a, min_gran, sched, batch, S::BATCH, ba, line)) return;

  if (tid == 0) {
    bar_init(k_full, 4);
    bar_init(v_full, 4);
    bar_init(qk_done, 1);
    bar_init(p_full, 4);
    bar_init(pv_done, 1);
    *gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tm_slot)), "n"(S::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  seek<kRowsT, KT, kThreadsT>(a, ba, line, place);
  tm_before();
  __syncthreads();
  tm_after();
  const uint32_t tm = *tm_slot;
  const uint32_t s_at = tm + S::S_COL, o_at = tm + S::O_COL;
  Place p = *place;
  Segment sg;
  uint32_t done = 0;  // tiles of earlier segments: the barriers' phases go on

  while (next_segment<kRowsT, KT>(a, ba, p, sg)) {
    const int key0 = (sg.t.lo / KT + sg.off) * KT;
    const int32_t *table = a.batch.tables + (int64_t)sg.t.seq * a.batch.table_stride;
    auto page_at = [&](int key) -> int {  // -1: no row of the tile sees a key of these 16, or there is no page
      if (key >= sg.t.hi || key + 16 <= sg.t.lo) return -1;
      const int pg = __ldg(table + (key >> a.page_shift));
      return pg >= 0 && pg < a.pool.pages ? pg : -1;
    };
    // The queries, and the largest finite scale of the segment's values.
    if (tid == 0) *vtop_s = 0.0f;
    __syncthreads();
    {
      const int pieces = DP / 8;
      for (int i = tid; i < kRowsT * pieces; i += kThreadsT) {
        const int row = i / pieces, c = i % pieces, d = c * 8, r = sg.t.row0 + row;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < sg.t.rows && d < D) {
          const __half *q = static_cast<const __half *>(a.q) + (int64_t)(sg.t.start + r / a.group) * a.q_token +
                            (int64_t)(sg.head * a.group + r % a.group) * a.q_head + d;
          if (a.q_wide) {
            v = *reinterpret_cast<const uint4 *>(q);
          } else {
            __half h[8];
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = q[j];
            memcpy(&v, h, 16);
          }
        }
        *reinterpret_cast<uint4 *>(qs + (c / 8) * (kRowsT * 128) + row * 128 + (((c % 8) ^ (row & 7)) * 16)) = v;
      }
      float top = 0.0f;
      for (int i = tid; i < sg.take * GROUPS; i += kThreadsT) {
        const int pg = page_at(key0 + i * 16);
        if (pg >= 0) {
          const float s = fabsf(__ldg(a.pool.v_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pg * a.pool.scale_page_stride)));
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
    const int n = sg.take;

    if (warp >= 4) {
      // ---- bytes to float16 ----
      constexpr int CH = DP / 16, KPP = 128 / CH, NI = KT / KPP;  // pieces a key, keys a pass, passes
      const int pt = tid - 128, key_in = pt / CH, ch = pt % CH;
      const bool live = ch * 16 < D;
      const int64_t tok = a.pool.token_stride, hoff = (int64_t)sg.head * a.pool.head_stride + 16 * ch;
      const int db = ch / 4, c0 = (ch % 4) * 2;
      uint4 kr[NI], vr[NI];
      float ksl = 0.0f, ratio = 0.0f;
      int pg = -1;  // of group `lane` of the tile that is asked for
      auto ask_page = [&](int j) { pg = lane < GROUPS && j < n ? page_at(key0 + j * KT + lane * 16) : -1; };
      auto ask = [&](const int8_t *from, int j, uint4 (&r)[NI]) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const int key = i * KPP + key_in;
          const int q = __shfl_sync(~0u, pg, key / 16);
          if (q >= 0 && live)
            r[i] = __ldg(reinterpret_cast<const uint4 *>(from + (int64_t)q * a.pool.page_stride + hoff +
                                                         (int64_t)((key0 + j * KT + key) & (PT - 1)) * tok));
          else
            r[i] = make_uint4(0u, 0u, 0u, 0u);
        }
      };
      auto put = [&](uint8_t *to, const uint4 (&r)[NI]) {
        if (!live) return;
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const int key = i * KPP + key_in;
          uint32_t h[8];
          const uint32_t w[4] = {r[i].x ^ 0x80808080u, r[i].y ^ 0x80808080u, r[i].z ^ 0x80808080u, r[i].w ^ 0x80808080u};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            h[2 * k] = half_pair_<0x4140>(w[k]);
            h[2 * k + 1] = half_pair_<0x4342>(w[k]);
          }
          uint8_t *row = to + db * (KT * 128) + key * 128;
          const uint4 lo4 = make_uint4(h[0], h[1], h[2], h[3]), hi4 = make_uint4(h[4], h[5], h[6], h[7]);
          // the two pieces in an order that keeps eight lanes on eight bank groups
          const int first = db & 1;
          *reinterpret_cast<uint4 *>(row + (((c0 + first) ^ (key & 7)) * 16)) = first ? hi4 : lo4;
          *reinterpret_cast<uint4 *>(row + (((c0 + 1 - first) ^ (key & 7)) * 16)) = first ? lo4 : hi4;
        }
      };
      auto ask_scales = [&]() {
        ksl = 0.0f;
        ratio = 0.0f;
        if (pg >= 0) {
          ksl = __ldg(a.pool.k_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pg * a.pool.scale_page_stride));
          const float s = __ldg(a.pool.v_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pg * a.pool.scale_page_stride));
          // a scale that is not finite makes the weights of the keys that are seen NaN
          ratio = !(fabsf(s) <= 3.402823466e38f) ? __int_as_float(0x7fc00000) : vtop > 0.0f ? __fdiv_rn(s, vtop) * 128.0f : 0.0f;
        }
      };
      ask_page(0);
      ask(a.pool.k, 0, kr);
      ask_scales();
      ask(a.pool.v, 0, vr);
      for (int j = 0; j < n; j++) {
        const uint32_t ph = (done + j) & 1;
        if (j && !warp_wait(qk_done, ph ^ 1, gone)) break;  // the keys before these are used up
        put(ks, kr);
        // The softmax is a tile behind at most: two sets of scales.
        float *mt = meta + ph * (2 * GROUPS + 2);
        if (warp == 4) {
          if (lane < GROUPS) {
            mt[lane] = ksl * a.scale_log2;
            mt[GROUPS + lane] = ratio;
          }
          const uint32_t holes = __ballot_sync(~0u, lane < GROUPS && pg < 0);
          if (lane == 0) mt[2 * GROUPS] = __int_as_float((int)holes);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(k_full);
        ask_page(j + 1);
        if (j + 1 < n) {
          ask(a.pool.k, j + 1, kr);
          ask_scales();
        }
        if (j && !warp_wait(pv_done, ph ^ 1, gone)) break;
        put(vs, vr);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(v_full);
        if (j + 1 < n) ask(a.pool.v, j + 1, vr);
      }
    } else {
      // ---- weights ----
      const int row = tid, pos = sg.t.first + (sg.t.row0 + row) / a.group;
      const int lo = row_lo(a, pos), hi = row < sg.t.rows ? row_hi(a, sg.t.keys, pos) : 0;
      const uint32_t lanes = (uint32_t)(warp * 32) << 16;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      // One thread's: float32 sums, float16 operands; 128 rows by KT keys, and by D
      // (the values are N-major).
      const uint32_t id_s = 1u << 4 | (uint32_t)(KT >> 3) << 17 | (uint32_t)(kRowsT >> 4) << 24;
      const uint32_t id_o = 1u << 4 | 1u << 16 | (uint32_t)(D >> 3) << 17 | (uint32_t)(kRowsT >> 4) << 24;
      // (every warp has waited for the keys: see below)
      auto scores = [&]() {
        tm_after();
        for (int k = 0; k < D / 16; k++) {
          const uint32_t off = (k % 4) * 32;
          mma_ss(s_at, operand(smem_at(qs) + (k / 4) * (kRowsT * 128) + off, 16),
                 operand(smem_at(ks) + (k / 4) * (KT * 128) + off, 16), id_s, k > 0);
        }
        tm_commit(qk_done);
      };
      auto outputs = [&](int j) {
        const uint32_t ph = (done + j) & 1;
        if (!bar_wait(p_full, ph, gone) || !bar_wait(v_full, ph, gone)) return;
        tm_after();
        for (int k = 0; k < KT / 16; k++)
          mma_ts(o_at, s_at + k * 8, operand(smem_at(vs) + k * 2048, KT * 128), id_o, j > 0 || k > 0);
        tm_commit(pv_done);
        // S takes P's place: the next scores wait for the product that reads P
        if (j + 1 < n && bar_wait(pv_done, ph, gone)) scores();
      };
      // A warp waits for a tile's keys (their scales lie beside them) before it lets
      // the product that reads them start: later, the barrier might be two phases
      // on and look as if it had yet to come.
      ok = warp_wait(k_full, done & 1, gone);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (tid == 0 && ok) scores();
      __syncwarp();
      for (int j = 0; j < n && ok; j++) {
        const uint32_t ph = (done + j) & 1;
        if (!warp_wait(qk_done, ph, gone)) {
          ok = false;
          break;
        }
        tm_after();
        const float *mt = meta + ph * (2 * GROUPS + 2);
        const uint32_t holes = (uint32_t)__float_as_int(mt[2 * GROUPS]);
        const int key = key0 + j * KT;
        const bool edge = key < sg.t.lo_all || key + KT > sg.t.hi_all || holes;
        auto masked = [&](float (&v)[32], int chunk) {
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float c = mt[chunk * 2 + g];
#pragma unroll
            for (int x = 0; x < 16; x++) v[g * 16 + x] *= c;
          }
          if (edge) {
#pragma unroll
            for (int x = 0; x < 32; x++) {
              const int kk = key + chunk * 32 + x;
              if (kk < lo || kk >= hi || (holes >> (chunk * 2 + x / 16) & 1)) v[x] = -INFINITY;
            }
          }
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int ch = 0; ch < KT / 32; ch++) {  // (unrolled, the loops overflow the instruction cache)
          float v[32];
          tm_ld32(s_at + lanes + ch * 32, v);
          masked(v, ch);
#pragma unroll
          for (int x = 0; x < 32; x++) top = fmaxf(top, v[x]);
        }
        // Rows whose maximum rose by more than 8 (or that saw their first key) bring
        // their whole warp up to date.
        if (__any_sync(~0u, top > m + 8.0f || (m == -INFINITY && top > m))) {
          const float mn = fmaxf(m, top);
          const float f = m == -INFINITY ? 0.0f : ex2_(m - mn);
          l *= f;
          m = mn;
          if (j) {  // (the first product writes O)
#pragma unroll 1
            for (int ch = 0; ch * 32 < D; ch++) {
              float v[32];
              tm_ld32(o_at + lanes + ch * 32, v);
#pragma unroll
              for (int x = 0; x < 32; x++) v[x] *= f;
              tm_st32(o_at + lanes + ch * 32, v);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
        for (int ch = 0; ch < KT / 32; ch++) {
          float v[32];
          tm_ld32(s_at + lanes + ch * 32, v);
          masked(v, ch);
          uint32_t w[16];
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float r = mt[GROUPS + ch * 2 + g];
#pragma unroll
            for (int x = 0; x < 8; x++) {
              const int i = g * 16 + 2 * x;
              const float e0 = ex2_(v[i] - ref), e1 = ex2_(v[i + 1] - ref);
              l += e0;
              l += e1;
              float p0 = e0 * r, p1 = e1 * r;
              if (edge) {  // 0 times what is not a number
                if (v[i] == -INFINITY) p0 = 0.0f;
                if (v[i + 1] == -INFINITY) p1 = 0.0f;
              }
              const __half2 h = __floats2half2_rn(p0, p1);
              w[g * 8 + x] = *reinterpret_cast<const uint32_t *>(&h);
            }
          }
          tm_st16(s_at + lanes + ch * 16, w);
        }
        tm_wait_st();
        tm_before();
        if (j + 1 < n && !warp_wait(k_full, ph ^ 1, gone)) ok = false;
        __syncwarp();
        if (lane == 0) bar_arrive(p_full);
        if (tid == 0) outputs(j);
        __syncwarp();
      }
      ok = ok && warp_wait(pv_done, (done + n - 1) & 1, gone);
      tm_after();
      const bool whole = sg.take == sg.units;
      float *part = whole ? nullptr : partial_at<kRowsT, DP>(a, blockIdx.x, sg.off == 0);
      const float unscale = vtop * 0x1p-7f;
      if (ok) {
#pragma unroll 1
        for (int ch = 0; ch < DP / 32; ch++) {
          if (ch * 32 < D) {
            float v[32];
            tm_ld32(o_at + lanes + ch * 32, v);
            if (row < sg.t.rows) {
#pragma unroll
              for (int x = 0; x < 8; x++) {
                const float4 r = make_float4(v[4 * x] * unscale, v[4 * x + 1] * unscale, v[4 * x + 2] * unscale, v[4 * x + 3] * unscale);
                const int d = ch * 32 + 4 * x;
                if (d < D) {
                  if (whole) write_out<__half>(a, sg.t, sg.head, row, d, r, l);
                  else *reinterpret_cast<float4 *>(part + row * DP + d) = r;
                }
              }
            }
          }
        }
        if (row < sg.t.rows) {
          if (whole) {
            write_lse(a, sg.t, sg.head, row, m, l);
          } else {
            part[kRowsT * DP + row] = m;
            part[kRowsT * DP + kRowsT + row] = l;
          }
        }
      }
      tm_before();
    }
    done += n;
    __syncthreads();
    tm_after();
    if (*gone) break;
    if (sg.take != sg.units) arrive<__half, kRowsT, DP, kThreadsT>(a, sg, line, fac, flag);
  }
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(S::TM_COLS));
  if (tid == 0 && *gone && a.err) *a.err = 1;
}

template <int DP>
int launch(AttendArgs a, int sms, cudaStream_t st) {
  using S = Tiles<DP>;
  auto *kern = k_kv_attend_tiles<DP>;
  SHLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
  a.slots = (int)(((int64_t)a.batch.tokens * a.group) / kRowsT + a.batch.seqs);
  const int64_t room = ((int64_t)a.batch.table_pages << a.page_shift) / S::KT + 1;
  int64_t most = (int64_t)a.slots * a.pool.heads;
  most = most > (1 << 20) ? most : most * room;
  const int64_t full = (int64_t)sms * S::PER_SM;
  int64_t grid = most < full ? most : full;
  if (grid > kAttendMaxBlocks) grid = kAttendMaxBlocks;
  if (grid < 1) grid = 1;
  kern<<<(unsigned)grid, kThreadsT, S::BYTES, st>>>(a, 1);
  return launch_check("kv_attend");
}

}  // namespace

size_t attend_tiles_partial_bytes(int sms) {
  auto of = [&](int dp, int per_sm) {
    const int blocks = sms * per_sm < kAttendMaxBlocks ? sms * per_sm : kAttendMaxBlocks;
    return (size_t)blocks * 2 * kRowsT * (dp + 2) * 4;
  };
  size_t most = of(64, Tiles<64>::PER_SM);
  if (of(128, Tiles<128>::PER_SM) > most) most = of(128, Tiles<128>::PER_SM);
  if (of(256, Tiles<256>::PER_SM) > most) most = of(256, Tiles<256>::PER_SM);
  return most;
}

int launch_attend_tiles(const AttendArgs &a, int sms, cudaStream_t st) {
  const int D = a.pool.head_dim;
  if (D <= 64) return launch<64>(a, sms, st);
  if (D <= 128) return launch<128>(a, sms, st);
  return launch<256>(a, sms, st);
}

}  // namespace shlo
