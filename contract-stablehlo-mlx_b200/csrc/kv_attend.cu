// Attention over the 8-bit paged cache, for few rows a sequence: one new token
// (or a few) times the query heads that share a key/value head.
//
//   s_t = scale * sk_t * (q . k_t),  out = sum_t e^(s_t - m) sv_t v_t / l,
//   lse = ln sum_t e^(s_t),
// over the keys t a row sees: t < length, t <= its position (causal), above
// position - window, in a page that the table holds. A row that sees none has
// out 0 and lse -inf. sk, sv: the scale of t's page and head.
//
// Bound: the cache's bytes, read once. A warp takes 16 keys at a time straight
// from global memory into matrix-instruction fragments: the 8-bit values become
// float16 integers exactly (a byte under the exponent of 1024, minus 1152), the
// scales are applied to the scores and to the weights. Keys are the M side of
// both products (S^T = K Q^T, O^T = V^T P^T), so 8 rows fill the N side and no
// lane idles for a group of 8 query heads; a row's dimensions and the keys of a
// tile may be taken in any order, so each lane reads 16 contiguous bytes.
//
// Measured on one B200, 128-wide heads, four query heads to a key/value head,
// float16: 64 sequences x 8192 keys (1.07 GB) 219 us, 4.91 TB/s; 64 ragged ones
// (505 MB) 119 us; two of 150 to 200 thousand keys (343 MB) 89 us; one of 256
// keys 12 us. A loop without the products takes as long: the rest over the bytes
// is the start (the line, the first pages and pieces, 8 us), a block's cuts
// between units (8 us each, which the SM's other blocks cover as long as they
// are not at one too) and the last blocks' ends. Two or four blocks an SM
// measured 231 and 227 us for the first.
//
// Precision. Scores, maxima, sums and outputs are kept in 32 bits, outputs as
// rounding adds of sixteen keys' products (sums that the matrix instructions
// carry on lose up to 2^-23 of themselves each time, always downwards: 3e-4 over
// 200000 keys; the adds cost 0.5 %). The weights
// are rounded to float16 for the second product, as e^(s - m) (sv / largest sv
// so far, rounded down to a power of two) 2^14: below 2^15 and, since float16
// reaches down to 2^-24, exact to 2^-38 of the largest weight (of the largest
// value's scale among the keys of the tile of rows: a page whose scale is 2^28
// times a row's others costs that row's bits). For float32 queries q and the
// weights are split into two float16 terms each (22 bits), q after scaling each
// row by a power of two to below 2^14.
#include "kv_attend.cuh"

namespace shlo {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two bytes of x (sign bit flipped) as float16 integers: 0x6400 | u is 1024 + u.
template <int SEL>
__device__ __forceinline__ uint32_t half_pair(uint32_t x) {
  const uint32_t r = __byte_perm(x, 0x64646464u, SEL);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&r), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
// Copy N bytes from global to this lane's place in shared memory, past L1; zeros where `ok` is false.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const int8_t *src) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const int8_t *src, bool ok) {
  const int n = ok ? N : 0;
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(p) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(p) : "memory");
  return r;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// DP: the head width rounded up to 64, 128 or 256; NT: row tiles of 8; TERMS: 1
// (float16 queries) or 2 (float32). A step is 16 MT keys of a warp: its keys'
// and its values' bytes are a piece each, in one ring of R pieces (keys 0, values
// 0, keys 1, ...): the piece R on is asked for as soon as one is used up. A lane
// copies the bytes it will read itself to a place of its own (so the ring needs
// no barrier and no reads conflict): the ring, not the warps' number, covers the
// memory's latency.
template <typename T, int DP, int NT>
struct Shape {
  static constexpr int TERMS = sizeof(T) == 2 ? 1 : 2;
  static constexpr int ROWS = 8 * NT;
  static constexpr int MT = DP == 256 ? 1 : 2;  // 16-key tiles a step
  static constexpr int GRAN = kWarps * MT * 16;
  static constexpr int KS = DP / 16;            // 16-wide steps of the first product
  static constexpr int OSTRIDE = DP + 4;
  static constexpr int PER_SM = DP == 64 ? (NT == 1 ? 4 : 3) : DP == 128 ? (NT == 1 ? 3 : 2) : 2;
  static constexpr int PIECE = MT * 16 * DP;    // bytes
  static constexpr int R = DP == 64 ? 5 : 3;
  // shared memory, in 4-byte words
  static constexpr int Q_WORDS = KS * 32 * 2 * NT * TERMS;
  static constexpr int RING_WORDS = kWarps * R * PIECE / 4;
  static constexpr int O_WORDS = kWarps * ROWS * OSTRIDE;
  static constexpr int JOIN_WORDS = 2 * (kJoin<ROWS> + 1) * ROWS;
  static constexpr int BODY = O_WORDS > JOIN_WORDS ? O_WORDS : JOIN_WORDS;  // the warps' results, then a join's factors
  static constexpr int BATCH = 258;  // the batch's arrays, up to 128 sequences
  static constexpr int WORDS = 2 * Q_WORDS + RING_WORDS + BODY + 2 * kWarps * ROWS + 2 * ROWS + 2 * (kThreads + 4) + 16 + 4 + BATCH;
};

// A block goes from segment to segment: a warp that is done with one asks for
// the next one's first pieces and queries before the block's results meet, so
// the memory is busy meanwhile. Per segment two barriers: the queries are
// staged, the results are written.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kThreads, Shape<T, DP, NT>::PER_SM) k_kv_attend_rows(const AttendArgs a, int min_gran) {
  using S = Shape<T, DP, NT>;
  constexpr int ROWS = S::ROWS, MT = S::MT, GRAN = S::GRAN, KS = S::KS, TERMS = S::TERMS, OS = S::OSTRIDE;
  constexpr int KC = DP / 64;        // 16-byte pieces a lane reads of a key row
  constexpr int VW = DP / 32;        // 4-byte words a lane reads of a value row
  constexpr int R = S::R;
  constexpr int QV = (DP + 127) / 128;  // groups of four dimensions a lane stages of a query row
  constexpr int TL = 32 / MT;           // steps of a chunk of pages
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t *const qs0 = smem;                                  // [2][TERMS][NT][KS / 2][32][2][2]
  uint32_t *const rings = smem + 2 * S::Q_WORDS;
  float *const body = reinterpret_cast<float *>(rings + S::RING_WORDS);
  float *const wm = body + S::BODY, *const wl = wm + kWarps * ROWS, *const rs0 = wl + kWarps * ROWS;  // rs0 [2][ROWS]
  long long *const sched = reinterpret_cast<long long *>(rs0 + 2 * ROWS);
  Place *const place = reinterpret_cast<Place *>(sched + kThreads + 4);
  unsigned *const flag = reinterpret_cast<unsigned *>(place) + 16;
  int *const batch = reinterpret_cast<int *>(flag + 4);
  static_assert(sizeof(Place) <= 64, "its room in shared memory");

  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
  const int D = a.pool.head_dim, PT = 1 << a.page_shift;
  Line line;
  BatchArrays ba;
  if (!schedule<ROWS, GRAN, kThreads>(a, min_gran, sched, batch, S::BATCH, ba, line)) return;

  // Rings: a lane's 16 bytes of copy i of a piece are at [i][lane].
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(rings) + warp * (R * S::PIECE) + lane * 16;
  const uint32_t vring = ring - lane * 16 + lane * (VW == 2 ? 8 : 16);
  const int64_t tok = a.pool.token_stride, tok8 = 8 * tok;
  const int64_t klane = g * tok + 16 * c, vlane = 2 * c * tok + (VW == 2 ? 8 : 16) * g;
  const bool wide = D == DP;
  auto copy_k = [&](int slot, int head, int key, int pages, int at) {  // (the caller commits)
    const uint32_t dst = ring + slot * S::PIECE;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      const int pg = __shfl_sync(~0u, pages, at + mt);
      const int8_t *src = a.pool.k + ((int64_t)head * a.pool.head_stride + (int64_t)max(pg, 0) * a.pool.page_stride +
                                      ((key + mt * 16) & (PT - 1)) * tok + klane);
      const int8_t *src8 = src + tok8;
      if (wide && pg >= 0) {
#pragma unroll
        for (int j = 0; j < KC; j++) {
          copy_async<16>(dst + (mt * 2 * KC + j) * 512, src + 64 * j);
          copy_async<16>(dst + ((mt * 2 + 1) * KC + j) * 512, src8 + 64 * j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < KC; j++) {
          const bool ok = pg >= 0 && 64 * j + 16 * c < D;
          copy_async<16>(dst + (mt * 2 * KC + j) * 512, src + 64 * j, ok);
          copy_async<16>(dst + ((mt * 2 + 1) * KC + j) * 512, src8 + 64 * j, ok);
        }
      }
    }
  };
  auto copy_v = [&](int slot, int head, int key, int pages, int at) {
    constexpr int N = VW == 2 ? 8 : 16, VC = VW == 2 ? 1 : VW / 4;
    const uint32_t dst = vring + slot * S::PIECE;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      const int pg = __shfl_sync(~0u, pages, at + mt);
      const int8_t *p[4];
      p[0] = a.pool.v + ((int64_t)head * a.pool.head_stride + (int64_t)max(pg, 0) * a.pool.page_stride +
                         ((key + mt * 16) & (PT - 1)) * tok + vlane);
      p[1] = p[0] + tok;
      p[2] = p[0] + tok8;
      p[3] = p[2] + tok;
      if (wide && pg >= 0) {
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int j = 0; j < VC; j++) copy_async<N>(dst + ((mt * 4 + k) * VC + j) * (32 * N), p[k] + 128 * j);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int j = 0; j < VC; j++)
            copy_async<N>(dst + ((mt * 4 + k) * VC + j) * (32 * N), p[k] + 128 * j, pg >= 0 && 128 * j + N * g < D);
      }
    }
  };
  // Keys of step i of this warp: key0 + i * GRAN + [0, 16 MT).
  auto first_key = [&](const Segment &sg) { return (sg.t.lo / GRAN + sg.off) * GRAN + warp * (MT * 16); };
  // Pages of the coming steps are held across the lanes, 32 tiles of 16 keys (TL
  // steps) at a time; -1: no row of the tile sees a key of it, or there is none.
  auto step_pages = [&](const Segment &sg, int step) -> int {
    step += lane / MT;
    const int key = first_key(sg) + step * GRAN + (lane % MT) * 16;
    if (step >= sg.take || key >= sg.t.hi || key + 16 <= sg.t.lo) return -1;
    const int p = __ldg(a.batch.tables + (int64_t)sg.t.seq * a.batch.table_stride + (key >> a.page_shift));
    return p >= 0 && p < a.pool.pages ? p : -1;
  };
  // A segment's first pieces and its queries. The queries are the first
  // product's right side: step (j, s) of lane (g, c) has row g's dimensions d,
  // d + 2 and d + 1, d + 3, d = 64 j + 16 c + 4 s.
  auto begin = [&](const Segment &sg, int buf) -> int {
    constexpr int RW = ROWS / kWarps;
    const int pages = step_pages(sg, 0), key = first_key(sg);
    T raw[RW][QV][4];  // asked for before the pages are waited for
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const int row = warp + i * kWarps, r = sg.t.row0 + row;
      const T *q = static_cast<const T *>(a.q) + (int64_t)(sg.t.start + r / a.group) * a.q_token +
                   (int64_t)(sg.head * a.group + r % a.group) * a.q_head;
#pragma unroll
      for (int k = 0; k < QV; k++) {
        const int d = 4 * (lane + 32 * k);
#pragma unroll
        for (int j = 0; j < 4; j++) raw[i][k][j] = row < sg.t.rows && d < D ? q[d + j] : (T)0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      if (i / 2 < sg.take) {
        if (i % 2 == 0) copy_k(i, sg.head, key + i / 2 * GRAN, pages, i / 2 * MT);
        else copy_v(i, sg.head, key + i / 2 * GRAN, pages, i / 2 * MT);
      }
      copy_commit();
    }
    uint32_t *const qs = qs0 + buf * S::Q_WORDS;
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const int row = warp + i * kWarps;
      float f[QV][4], m = 0.0f;
#pragma unroll
      for (int k = 0; k < QV; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[k][j] = (float)raw[i][k][j];
          m = fmaxf(m, fabsf(f[k][j]));
        }
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
        // a power of two that brings the row's largest value to [2^13, 2^14)
        int e = 0;
        if (m > 0.0f && m <= 3.402823466e38f) e = max(-126, min(126, 13 - ilogbf(m)));
        const float up = __int_as_float((127 + e) << 23);
        if (lane == 0) rs0[buf * ROWS + row] = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int k = 0; k < QV; k++)
#pragma unroll
          for (int j = 0; j < 4; j++) f[k][j] *= up;
      }
#pragma unroll
      for (int k = 0; k < QV; k++) {
        const int d = 4 * (lane + 32 * k);
        if (d >= DP) break;
        const int ks = (d / 64) * 4 + (d % 16) / 4, l = (row % 8) * 4 + (d % 64) / 16;
        uint32_t *dst = qs + ((row / 8) * KS + ks / 2 * 2) * 64 + l * 4 + ks % 2 * 2;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_half(f[k][0], f[k][2]), pack_half(f[k][1], f[k][3]));
        if constexpr (TERMS == 2) {
          float lo[4];
#pragma unroll
          for (int j = 0; j < 4; j++) lo[j] = f[k][j] - __half2float(__float2half_rn(f[k][j]));
          *reinterpret_cast<uint2 *>(dst + NT * KS * 64) = make_uint2(pack_half(lo[0], lo[2]), pack_half(lo[1], lo[3]));
        }
      }
    }
    return pages;
  };

  seek<ROWS, GRAN, kThreads>(a, ba, line, place);
  __syncthreads();
  Place p = *place;
  Segment sg;
  if (!next_segment<ROWS, GRAN>(a, ba, p, sg)) return;
  int buf = 0, pages = begin(sg, 0);
  for (;;) {
    __syncthreads();
    const uint32_t *const qs = qs0 + buf * S::Q_WORDS;

    // Each lane's two rows (columns 2c, 2c + 1 of the transposed products) of each tile of 8.
    int lo[NT][2], hi[NT][2];
    float col[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = nt * 8 + 2 * c + e;
        const int pos = sg.t.first + (sg.t.row0 + row) / a.group;
        lo[nt][e] = row_lo(a, pos);
        hi[nt][e] = row < sg.t.rows ? row_hi(a, sg.t.keys, pos) : 0;
        col[nt][e] = a.scale_log2;
        if constexpr (TERMS == 2) col[nt][e] *= rs0[buf * ROWS + row];
      }

    float o[NT][VW * 2][4], m[NT][2], l[NT][2], vmax = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < VW * 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[nt][i][j] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
    }
    float ksl = 0.0f, ratio_l = 0.0f;  // of the lane's tile: keys' scale, 2^14 values' scale / vmax
    uint32_t holes = 0;
    int pages_next = -1, slot = 0;  // slot: of the piece that comes next
    const int key0 = first_key(sg);

    for (int i = 0; i < sg.take; i++) {
      const int key = key0 + i * GRAN;
      const int at = (i % TL) * MT;
      if (at == 0) {
        if (i) pages = pages_next;
        pages_next = i + TL < sg.take ? step_pages(sg, i + TL) : -1;
        holes = __ballot_sync(~0u, pages < 0);
        float vs = 0.0f;
        ksl = 0.0f;
        if (pages >= 0) {
          ksl = __ldg(a.pool.k_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pages * a.pool.scale_page_stride));
          vs = __ldg(a.pool.v_scale + ((int64_t)sg.head * a.pool.scale_head_stride + (int64_t)pages * a.pool.scale_page_stride));
        }
        const bool finite = fabsf(vs) <= 3.402823466e38f;
        float top = finite ? fmaxf(vmax, fabsf(vs)) : vmax;
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
        // (a power of two, so that 2^-14 of it is exact where it is no normal number)
        top = top == 0.0f ? 0.0f : fmaxf(__uint_as_float(__float_as_uint(top) & 0x7f800000u), 0x1p-126f);
        if (top != vmax) {
          const float f = __fdiv_rn(vmax, top);
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int w = 0; w < VW * 2; w++)
#pragma unroll
              for (int j = 0; j < 4; j++) o[nt][w][j] *= f;
          vmax = top;
        }
        // a scale that is not finite makes the weights of the keys that are seen NaN
        ratio_l = !finite ? __int_as_float(0x7fc00000) : vmax > 0.0f ? __fdiv_rn(vs, vmax) * 16384.0f : 0.0f;
      }
      const bool hole = (holes >> at & ((1u << MT) - 1)) != 0;
      // S^T: [16 keys][8 rows] a tile. R - 1 pieces were committed after these keys.
      copy_wait<R - 1>();
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[mt][nt][j] = 0.0f;
      // float32's second terms are summed apart: the matrix instructions cut off what
      // falls below a sum's last bit.
      float s2[MT][NT][4] = {};
      uint4 kr[MT][2], b[TERMS][NT];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if (ks % 4 == 0) {
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h2 = 0; h2 < 2; h2++) kr[mt][h2] = lds16(ring + slot * S::PIECE + ((mt * 2 + h2) * KC + ks / 4) * 512);
        }
        if (ks % 2 == 0) {
#pragma unroll
          for (int tm = 0; tm < TERMS; tm++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              b[tm][nt] = *reinterpret_cast<const uint4 *>(qs + ((tm * NT + nt) * KS + ks) * 64 + lane * 4);
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          const uint32_t w0 = (&kr[mt][0].x)[ks % 4] ^ 0x80808080u, w1 = (&kr[mt][1].x)[ks % 4] ^ 0x80808080u;
          const uint32_t af[4] = {half_pair<0x4240>(w0), half_pair<0x4240>(w1), half_pair<0x4341>(w0), half_pair<0x4341>(w1)};
#pragma unroll
          for (int tm = 0; tm < TERMS; tm++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              mma16816(tm == 0 ? s[mt][nt] : s2[mt][nt], af, ks % 2 ? b[tm][nt].z : b[tm][nt].x, ks % 2 ? b[tm][nt].w : b[tm][nt].y);
        }
      }
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[mt][nt][j] += s2[mt][nt][j];
      }
      // The piece R on takes the place of these (none past the segment: its end
      // leaves nothing on the way that could land on the next one's pieces).
      auto refill = [&](int steps, bool keys) {
        if (i + steps < sg.take) {
          const int from = at + steps * MT < 32 ? pages : pages_next, tile = (at + steps * MT) & 31;
          if (keys) copy_k(slot, sg.head, key + steps * GRAN, from, tile);
          else copy_v(slot, sg.head, key + steps * GRAN, from, tile);
        }
        copy_commit();
        slot = slot + 1 == R ? 0 : slot + 1;
      };
      refill(R / 2, R % 2 == 0);

      // scores in units of log2, the unseen at -inf
      float ks_[MT];
#pragma unroll
      for (int mt = 0; mt < MT; mt++) ks_[mt] = __shfl_sync(~0u, ksl, at + mt);
      const bool edge = key < sg.t.lo_all || key + MT * 16 > sg.t.hi_all;
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[mt][nt][j] *= ks_[mt] * col[nt][j & 1];
      uint32_t seen = ~0u;  // bit (mt * NT + nt) * 4 + j
      if (edge || hole) {
        seen = 0;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int kk = key + mt * 16 + g + (j >> 1) * 8;
              const bool y = !(holes >> (at + mt) & 1) && kk >= lo[nt][j & 1] && kk < hi[nt][j & 1];
              if (!y) s[mt][nt][j] = -INFINITY;
              seen |= (y ? 1u : 0u) << ((mt * NT + nt) * 4 + j);
            }
      }
      bool moved = false;
      float mn[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float x = m[nt][e];
#pragma unroll
          for (int mt = 0; mt < MT; mt++) x = fmaxf(x, fmaxf(s[mt][nt][e], s[mt][nt][2 + e]));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
          mn[nt][e] = x;
          moved |= x != m[nt][e];
        }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float f = m[nt][e] == -INFINITY ? 0.0f : ex2(m[nt][e] - mn[nt][e]);
            l[nt][e] *= f;
            m[nt][e] = mn[nt][e];
#pragma unroll
            for (int w = 0; w < VW * 2; w++) {
              o[nt][w][e] *= f;
              o[nt][w][2 + e] *= f;
            }
          }
      }
      float top[NT][2];  // (a row that has seen nothing yet subtracts 0)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) top[nt][e] = m[nt][e] == -INFINITY ? 0.0f : m[nt][e];
      copy_wait<R - 1>();
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        const float ratio = __shfl_sync(~0u, ratio_l, at + mt);
        uint32_t pb[TERMS][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float e = ex2(s[mt][nt][j] - top[nt][j & 1]);
            l[nt][j & 1] += e;
            w[j] = e * ratio;
          }
          if (edge || hole) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              if (!(seen >> ((mt * NT + nt) * 4 + j) & 1)) w[j] = 0.0f;
          }
          const uint32_t p01 = pack_half(w[0], w[1]), p23 = pack_half(w[2], w[3]);
          pb[0][nt][0] = transpose8x8(p01);
          pb[0][nt][1] = transpose8x8(p23);
          if constexpr (TERMS == 2) {
            const float2 h01 = __half22float2(*reinterpret_cast<const __half2 *>(&p01));
            const float2 h23 = __half22float2(*reinterpret_cast<const __half2 *>(&p23));
            pb[1][nt][0] = transpose8x8(pack_half(w[0] - h01.x, w[1] - h01.y));
            pb[1][nt][1] = transpose8x8(pack_half(w[2] - h23.x, w[3] - h23.y));
          }
        }
        // O^T += V^T P^T: word w of a lane holds dimensions 4w .. 4w + 3 of four keys
        uint32_t vr[4][4];
#pragma unroll
        for (int w = 0; w < VW; w++) {
          if (w % 4 == 0) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
              if constexpr (VW == 2) {
                const uint2 r = lds8(vring + slot * S::PIECE + (mt * 4 + k) * 256);
                vr[k][0] = r.x;
                vr[k][1] = r.y;
              } else {
                const uint4 r = lds16(vring + slot * S::PIECE + ((mt * 4 + k) * (VW / 4) + w / 4) * 512);
                vr[k][0] = r.x;
                vr[k][1] = r.y;
                vr[k][2] = r.z;
                vr[k][3] = r.w;
              }
            }
          }
          const uint32_t x0 = vr[0][w % 4] ^ 0x80808080u, x1 = vr[1][w % 4] ^ 0x80808080u;
          const uint32_t x2 = vr[2][w % 4] ^ 0x80808080u, x3 = vr[3][w % 4] ^ 0x80808080u;
          const uint32_t a01 = __byte_perm(x0, x1, 0x5140), b01 = __byte_perm(x0, x1, 0x7362);
          const uint32_t a23 = __byte_perm(x2, x3, 0x5140), b23 = __byte_perm(x2, x3, 0x7362);
          const uint32_t f0[4] = {half_pair<0x4140>(a01), half_pair<0x4342>(a01), half_pair<0x4140>(a23), half_pair<0x4342>(a23)};
          const uint32_t f1[4] = {half_pair<0x4140>(b01), half_pair<0x4342>(b01), half_pair<0x4140>(b23), half_pair<0x4342>(b23)};
          // Over thousands of keys the instructions' cut-off bits would add up (they
          // all point one way): sixteen keys' sums are added to O by rounding adds.
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            float t0[4] = {}, t1[4] = {};
#pragma unroll
            for (int tm = TERMS - 1; tm >= 0; tm--) {
              mma16816(t0, f0, pb[tm][nt][0], pb[tm][nt][1]);
              mma16816(t1, f1, pb[tm][nt][0], pb[tm][nt][1]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
              o[nt][2 * w][j] += t0[j];
              o[nt][2 * w + 1][j] += t1[j];
            }
          }
        }
      }
      refill((R + 1) / 2, R % 2 == 1);
    }

    // The next segment is on its way before this one's results meet in shared memory.
    Segment ns;
    const bool more = next_segment<ROWS, GRAN>(a, ba, p, ns);
    if (more) pages = begin(ns, buf ^ 1);

    const float unscale = vmax * 0x1p-14f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = l[nt][e];
        x += __shfl_xor_sync(~0u, x, 4);
        x += __shfl_xor_sync(~0u, x, 8);
        x += __shfl_xor_sync(~0u, x, 16);
        const int row = nt * 8 + 2 * c + e;
        if (g == 0) {
          wm[warp * ROWS + row] = m[nt][e];
          wl[warp * ROWS + row] = x;
        }
        float *dst = body + (warp * ROWS + row) * OS;
#pragma unroll
        for (int w = 0; w < VW; w++) {
          const int d = VW == 2 ? 8 * g + 4 * w : 128 * (w / 4) + 16 * g + 4 * (w % 4);
          *reinterpret_cast<float4 *>(dst + d) =
              make_float4(o[nt][2 * w][e] * unscale, o[nt][2 * w][2 + e] * unscale, o[nt][2 * w + 1][e] * unscale,
                          o[nt][2 * w + 1][2 + e] * unscale);
        }
      }
    __syncthreads();
    const bool whole = sg.take == sg.units;
    float *part = whole ? nullptr : partial_at<ROWS, DP>(a, blockIdx.x, sg.off == 0);
    for (int i = threadIdx.x; i < ROWS * DP / 4; i += kThreads) {
      const int row = i / (DP / 4), d = (i % (DP / 4)) * 4;
      if (row >= sg.t.rows) break;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) top = fmaxf(top, wm[w * ROWS + row]);
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float f = join_factor(wm[w * ROWS + row], top);
        const float4 v = *reinterpret_cast<const float4 *>(body + (w * ROWS + row) * OS + d);
        sum = __fmaf_rn(f, wl[w * ROWS + row], sum);
        r.x = __fmaf_rn(f, v.x, r.x);
        r.y = __fmaf_rn(f, v.y, r.y);
        r.z = __fmaf_rn(f, v.z, r.z);
        r.w = __fmaf_rn(f, v.w, r.w);
      }
      if (whole) {
        if (d < D) write_out<T>(a, sg.t, sg.head, row, d, r, sum);
        if (d == 0) write_lse(a, sg.t, sg.head, row, top, sum);
      } else {
        *reinterpret_cast<float4 *>(part + row * DP + d) = r;
        if (d == 0) {
          part[ROWS * DP + row] = top;
          part[ROWS * DP + ROWS + row] = sum;
        }
      }
    }
    if (!whole) arrive<T, ROWS, DP, kThreads>(a, sg, line, body, flag);
    if (!more) break;
    sg = ns;
    buf ^= 1;
  }
}

template <typename T, int DP, int NT>
int launch_rows(AttendArgs a, int sms, int device, cudaStream_t st) {
  using S = Shape<T, DP, NT>;
  constexpr size_t smem = S::WORDS * 4;
  static_assert((smem + 1024) * S::PER_SM <= 228 * 1024, "blocks of an SM");
  auto *kern = k_kv_attend_rows<T, DP, NT>;
  static std::atomic<uint64_t> allowed{0};
  SHLO_TRY(allow_smem((const void *)kern, smem, allowed, device));
  a.slots = (int)(((int64_t)a.batch.tokens * a.group) / S::ROWS + a.batch.seqs);
  // No more blocks than granules there can be.
  const int64_t room = ((int64_t)a.batch.table_pages << a.page_shift) / S::GRAN + 1;
  int64_t most = (int64_t)a.slots * a.pool.heads;
  most = most > (1 << 20) ? most : most * room;
  const int64_t full = (int64_t)sms * S::PER_SM;
  int64_t grid = most < full ? most : full;
  if (grid > kAttendMaxBlocks) grid = kAttendMaxBlocks;
  if (grid < 1) grid = 1;
  kern<<<(unsigned)grid, kThreads, smem, st>>>(a, 1);
  return launch_check("kv_attend");
}

template <typename T>
int dispatch_rows(const AttendArgs &a, int nt, int sms, int device, cudaStream_t st) {
  const int D = a.pool.head_dim;
  if (nt == 1 || D > 128) {
    if (D <= 64) return launch_rows<T, 64, 1>(a, sms, device, st);
    if (D <= 128) return launch_rows<T, 128, 1>(a, sms, device, st);
    return launch_rows<T, 256, 1>(a, sms, device, st);
  }
  if (D <= 64) return launch_rows<T, 64, 2>(a, sms, device, st);
  return launch_rows<T, 128, 2>(a, sms, device, st);
}

constexpr size_t kCounterBytes = 2 * kAttendMaxBlocks * sizeof(unsigned);

std::atomic<unsigned> g_give_up{0};

}  // namespace

// Counters, then the partials of the largest variant: two a block.
size_t attend_work_bytes(int sms) {
  size_t most = 0;
  auto of = [&](int rows, int dp, int per_sm) {
    int blocks = sms * per_sm;
    if (blocks > kAttendMaxBlocks) blocks = kAttendMaxBlocks;
    const size_t b = (size_t)blocks * 2 * rows * (dp + 2) * 4;
    if (b > most) most = b;
  };
  of(8, 64, Shape<__half, 64, 1>::PER_SM);
  of(8, 128, Shape<__half, 128, 1>::PER_SM);
  of(8, 256, Shape<__half, 256, 1>::PER_SM);
  of(16, 64, Shape<__half, 64, 2>::PER_SM);
  of(16, 128, Shape<__half, 128, 2>::PER_SM);
  const size_t tiles = attend_tiles_partial_bytes(sms);
  return kCounterBytes + (tiles > most ? tiles : most);
}

int launch_kv_attend(const AttendCall &c, int sms, int device, cudaStream_t st) {
  SHLO_TRY(check_pool(&c.pool, "kv_attend"));
  SHLO_TRY(check_batch(&c.batch, "kv_attend"));
  if (c.dtype != kF16 && c.dtype != kF32) return fail("kv_attend: %s not carried (float16 or float32)", dtype_name(c.dtype));
  if (c.heads < 1 || c.heads % c.pool.heads)
    return fail("kv_attend: %d query heads over %d key/value heads (a multiple)", c.heads, c.pool.heads);
  const int group = c.heads / c.pool.heads;
  if (group > 1024 || (int64_t)group * c.batch.tokens > (1 << 30))
    return fail("kv_attend: %d tokens of %d query heads to a key/value head (at most 1024, 2^30 together)", c.batch.tokens, group);
  if (c.window < 0) return fail("kv_attend: window %d", c.window);
  if (c.batch.seqs == 0 || c.batch.tokens == 0) return 0;
  if (!c.q || !c.out) return fail("kv_attend: null pointer");
  const size_t size = dtype_size(c.dtype);
  if (((uintptr_t)c.q | (uintptr_t)c.out) % size || (uintptr_t)c.lse % 4) return fail("kv_attend: misaligned q, out or lse");
  if (c.work_bytes < attend_work_bytes(sms) || !c.work || (uintptr_t)c.work % 16)
    return fail("kv_attend: a workspace of %zu bytes, aligned to 16, is needed (%zu given)", attend_work_bytes(sms), c.work_bytes);
  AttendArgs a;
  a.pool = c.pool;
  a.batch = c.batch;
  a.q = c.q; a.q_token = c.q_token; a.q_head = c.q_head;
  a.out = c.out; a.out_token = c.out_token; a.out_head = c.out_head;
  a.lse = c.lse;
  a.group = group;
  a.slots = 0;
  a.causal = c.causal; a.window = c.window;
  auto out_by = [&](int v) { return (uintptr_t)c.out % (v * size) == 0 && c.out_token % v == 0 && c.out_head % v == 0; };
  a.out_wide = out_by(8) ? 2 : out_by(4) ? 1 : 0;
  a.scale_log2 = c.scale * 1.44269504088896341f;
  a.page_shift = 31 - __builtin_clz((unsigned)c.pool.page_tokens);
  a.above = 0;
  a.upto = (int64_t)1 << 40;
  a.counters = static_cast<unsigned *>(c.work);
  a.partials = reinterpret_cast<float *>(static_cast<char *>(c.work) + kCounterBytes);
  a.q_wide = (uintptr_t)c.q % 16 == 0 && c.q_token % 8 == 0 && c.q_head % 8 == 0;
  a.err = c.err;
  a.give_up = g_give_up.load(std::memory_order_relaxed);
  // Tiles of 8 rows where the sequences have 8 or fewer on average, else 16. Above
  // 16, float16 sequences of more than 16 rows go to the tiles of 128 (in which a
  // 16-row tile would cost as much as a full one), in a launch of their own.
  // Measured with 32 sequences of 4096 keys and 8 key/value heads, us here and in
  // the tiles: 128 wide, 24 rows 150 and 165, 32 rows 152 and 166, 48 rows 215 and
  // 168, 256 rows 1028 and 265; 64 wide, 32 rows 100 and 142, 48 rows 146 and 142;
  // 256 wide, 20 rows 324 and 260. So 16 is the crossing of the widest heads, and
  // sends rows of 17 to 47 of narrower ones to the tiles 10 to 55 % early. The
  // average hides one prompt among single tokens: 128 tokens (512 rows) among 64 of
  // 2048 keys 200 us, 200 tokens, in the tiles, 180.
  const int64_t rows = (int64_t)c.batch.tokens * group;
  const int nt = rows <= (int64_t)8 * c.batch.seqs ? 1 : 2;
  if (c.dtype == kF16 && rows > (int64_t)16 * c.batch.seqs) {
    AttendArgs big = a;
    if (c.batch.seqs > 1) big.above = 16;  // (one sequence: one launch, whatever rows of q are its own)
    SHLO_TRY(launch_attend_tiles(big, sms, device, st));
    if (c.batch.seqs == 1) return 0;
    a.upto = 16;
  }
  return c.dtype == kF16 ? dispatch_rows<__half>(a, nt, sms, device, st) : dispatch_rows<float>(a, nt, sms, device, st);
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_cuda_device(void) {
  int id;
  return cudaGetDevice(&id) == cudaSuccess ? id : -2;
}

int shlo_kv_attend_workspace(size_t *bytes) {
  if (!bytes) return fail("kv_attend workspace: null pointer");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  *bytes = attend_work_bytes(dev->sm_count);
  return 0;
}

void shlo_test_attend_give_up(int32_t every) { g_give_up.store(every < 0 ? 0u : (unsigned)every); }

int shlo_kv_attend_noalloc(const shlo_kv_pool *pool, const shlo_kv_batch *batch, const void *q, int64_t q_token,
                           int64_t q_head, int32_t heads, uint8_t dtype, float scale, int32_t causal, int32_t window,
                           void *out, int64_t out_token, int64_t out_head, float *lse, void *workspace,
                           size_t workspace_bytes, void *stream) {
  if (!pool || !batch) return fail("kv_attend: null descriptor");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  SHLO_TRY(launch_error(dev, "kv_attend, an earlier call"));
  AttendCall c{*pool, *batch, q, q_token, q_head, out, out_token, out_head, lse, heads, dtype, scale, causal != 0, window,
               workspace, workspace_bytes, dev->pipe_err_dev};
  return launch_kv_attend(c, dev->sm_count, dev->id, (cudaStream_t)stream);
}

}  // extern "C"
