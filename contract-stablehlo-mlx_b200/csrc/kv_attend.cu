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
// Precision. Scores, maxima, sums and outputs are kept in 32 bits. The weights
// are rounded to float16 for the second product, as e^(s - m) (sv / largest sv
// so far) 2^14: at most 2^14 and, since float16 reaches down to 2^-24, exact to
// 2^-38 of the largest weight. For float32 queries q and the weights are split
// into two float16 terms each (22 bits), q after scaling each row by a power of
// two to below 2^14.
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
__device__ __forceinline__ uint4 ld_stream16(const int8_t *p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ld_stream8(const int8_t *p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// DP: the head width rounded up to 64, 128 or 256; NT: row tiles of 8; TERMS: 1
// (float16 queries) or 2 (float32).
template <typename T, int DP, int NT>
struct Shape {
  static constexpr int TERMS = sizeof(T) == 2 ? 1 : 2;
  static constexpr int ROWS = 8 * NT;
  static constexpr int MT = DP == 256 ? 1 : 2;  // 16-key tiles a step
  static constexpr int GRAN = kWarps * MT * 16;
  static constexpr int KS = DP / 16;            // 16-wide steps of the first product
  static constexpr int OSTRIDE = DP + 4;
  // shared memory, in 4-byte words
  static constexpr int Q_WORDS = KS * 32 * 2 * NT * TERMS;
  static constexpr int O_WORDS = kWarps * ROWS * OSTRIDE;
  static constexpr int JOIN_WORDS = (kAttendMaxBlocks / kJoin + 2) * ROWS;
  static constexpr int BODY = O_WORDS > JOIN_WORDS ? O_WORDS : JOIN_WORDS;
  static constexpr int WORDS = Q_WORDS + BODY + 3 * kWarps * ROWS + 2 * (kThreads + 4) + 4;
};

template <typename T, int DP, int NT, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) k_kv_attend_rows(const AttendArgs a, int min_gran) {
  using S = Shape<T, DP, NT>;
  constexpr int ROWS = S::ROWS, MT = S::MT, GRAN = S::GRAN, KS = S::KS, TERMS = S::TERMS, OS = S::OSTRIDE;
  constexpr int KC = DP / 64;        // 16-byte pieces a lane reads of a key row
  constexpr int VW = DP / 32;        // 4-byte words a lane reads of a value row
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t *const qs = smem;                                   // [TERMS][NT][KS][32][2]
  float *const body = reinterpret_cast<float *>(smem + S::Q_WORDS);
  float *const wm = body + S::BODY, *const wl = wm + kWarps * ROWS, *const rs = wl + kWarps * ROWS;
  long long *const sched = reinterpret_cast<long long *>(rs + kWarps * ROWS);
  unsigned *const flag = reinterpret_cast<unsigned *>(sched + kThreads + 4);

  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
  const int D = a.pool.head_dim, PT = 1 << a.page_shift;
  Cursor cur;
  if (!schedule<ROWS, GRAN, kThreads>(a, min_gran, sched, cur)) return;

  while (cur.at < cur.end && cur.head < a.pool.heads) {
    RowTile t;
    const int units = tile_of_slot<ROWS, GRAN>(a, cur.slot, t);
    if (units == 0) {  // a slot without a tile
      cur.slot++;
      if (cur.slot == a.slots) {
        cur.slot = 0;
        cur.head++;
      }
      continue;
    }
    const int take = (int)min((long long)(units - cur.off), cur.end - cur.at);
    const long long u0 = cur.at - cur.off, u1 = u0 + units;
    const int head = cur.head;

    // The rows' queries as the first product's right side: step (j, s) of lane
    // (g, c) has row g's dimensions d, d + 2 and d + 1, d + 3, d = 64 j + 16 c + 4 s.
    if constexpr (TERMS == 2) {
      for (int row = warp; row < ROWS; row += kWarps) {
        float m = 0.0f;
        if (row < t.rows) {
          const int r = t.row0 + row;
          const T *q = static_cast<const T *>(a.q) + (int64_t)(t.start + r / a.group) * a.q_token +
                       (int64_t)(head * a.group + r % a.group) * a.q_head;
          for (int d = lane; d < D; d += 32) m = fmaxf(m, fabsf((float)q[d]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        // a power of two that brings the row's largest value to [2^13, 2^14)
        int e = 0;
        if (m > 0.0f && m <= 3.402823466e38f) e = 13 - ilogbf(m);
        if (lane == 0) rs[row] = (float)max(-126, min(126, e));
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < KS * 32 * NT; i += kThreads) {
      const int l = i % 32, ks = (i / 32) % KS, nt = i / (32 * KS);
      const int row = nt * 8 + l / 4, d = 64 * (ks / 4) + 16 * (l % 4) + 4 * (ks % 4);
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (row < t.rows && d < D) {
        const int r = t.row0 + row;
        const T *q = static_cast<const T *>(a.q) + (int64_t)(t.start + r / a.group) * a.q_token +
                     (int64_t)(head * a.group + r % a.group) * a.q_head + d;
        float sc = 1.0f;
        if constexpr (TERMS == 2) sc = exp2f(rs[row]);
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = (float)q[j] * sc;
      }
      uint32_t *dst = qs + (nt * KS + ks) * 64 + l * 2;
      dst[0] = pack_half(f[0], f[2]);
      dst[1] = pack_half(f[1], f[3]);
      if constexpr (TERMS == 2) {
        float lo[4];
#pragma unroll
        for (int j = 0; j < 4; j++) lo[j] = f[j] - __half2float(__float2half_rn(f[j]));
        dst[NT * KS * 64] = pack_half(lo[0], lo[2]);
        dst[NT * KS * 64 + 1] = pack_half(lo[1], lo[3]);
      }
    }
    __syncthreads();

    // Each lane's two rows (columns 2c, 2c + 1 of the transposed products) of each tile of 8.
    int lo[NT][2], hi[NT][2];
    float col[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = nt * 8 + 2 * c + e;
        const int pos = t.first + (t.row0 + row) / a.group;
        lo[nt][e] = row_lo(a, pos);
        hi[nt][e] = row < t.rows ? row_hi(a, t.keys, pos) : 0;
        col[nt][e] = a.scale_log2;
        if constexpr (TERMS == 2) col[nt][e] *= exp2f(-rs[row]);
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

    const int32_t *table = a.batch.tables + (int64_t)t.seq * a.batch.table_stride;
    const int8_t *kbase = a.pool.k + (int64_t)head * a.pool.head_stride, *vbase = a.pool.v + (int64_t)head * a.pool.head_stride;
    const float *ksc = a.pool.k_scale + (int64_t)head * a.pool.scale_head_stride;
    const float *vsc = a.pool.v_scale + (int64_t)head * a.pool.scale_head_stride;
    // Keys of step i of this warp: key0 + i * GRAN + [0, 16 MT).
    const int key0 = (t.lo / GRAN + cur.off) * GRAN + warp * (MT * 16);
    auto page_of = [&](int key) -> int {  // -1: no such key
      if (key >= t.keys) return -1;
      const int p = __ldg(table + (key >> a.page_shift));
      return p >= 0 && p < a.pool.pages ? p : -1;
    };
    uint4 kr[MT][2][KC];
    uint32_t vr[MT][4][VW];
    float ks_[MT], vs_[MT];
    int page[MT], page_next[MT];
    auto load_k = [&](int key, const int (&pg)[MT]) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        const int8_t *row = kbase + (int64_t)pg[mt] * a.pool.page_stride +
                            (int64_t)((key + mt * 16 + g) & (PT - 1)) * a.pool.token_stride + 16 * c;
        ks_[mt] = pg[mt] >= 0 ? __ldg(ksc + (int64_t)pg[mt] * a.pool.scale_page_stride) : 0.0f;
#pragma unroll
        for (int h2 = 0; h2 < 2; h2++)
#pragma unroll
          for (int j = 0; j < KC; j++) {
            kr[mt][h2][j] = make_uint4(0x0u, 0x0u, 0x0u, 0x0u);
            if (pg[mt] >= 0 && 64 * j + 16 * c < D) kr[mt][h2][j] = ld_stream16(row + h2 * 8 * a.pool.token_stride + 64 * j);
          }
      }
    };
    auto load_v = [&](int key, const int (&pg)[MT]) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        const int8_t *row = vbase + (int64_t)pg[mt] * a.pool.page_stride +
                            (int64_t)((key + mt * 16 + 2 * c) & (PT - 1)) * a.pool.token_stride;
        const float sv = pg[mt] >= 0 ? __ldg(vsc + (int64_t)pg[mt] * a.pool.scale_page_stride) : 0.0f;
        vs_[mt] = fabsf(sv) <= 3.402823466e38f ? sv : __int_as_float(0x7fc00000);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int8_t *p = row + (int64_t)((k & 1) + (k >> 1) * 8) * a.pool.token_stride;
          if constexpr (VW == 2) {
            uint2 r = make_uint2(0u, 0u);
            if (pg[mt] >= 0 && 8 * g < D) r = ld_stream8(p + 8 * g);
            vr[mt][k][0] = r.x;
            vr[mt][k][1] = r.y;
          } else {
#pragma unroll
            for (int j = 0; j < VW / 4; j++) {
              uint4 r = make_uint4(0u, 0u, 0u, 0u);
              if (pg[mt] >= 0 && 128 * j + 16 * g < D) r = ld_stream16(p + 128 * j + 16 * g);
              vr[mt][k][4 * j] = r.x;
              vr[mt][k][4 * j + 1] = r.y;
              vr[mt][k][4 * j + 2] = r.z;
              vr[mt][k][4 * j + 3] = r.w;
            }
          }
        }
      }
    };
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      page[mt] = page_of(key0 + mt * 16);
      page_next[mt] = take > 1 ? page_of(key0 + GRAN + mt * 16) : -1;
    }
    load_k(key0, page);
    load_v(key0, page);

    for (int i = 0; i < take; i++) {
      const int key = key0 + i * GRAN;
      // S^T: [16 keys][8 rows] a tile
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[mt][nt][j] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        uint2 b[TERMS][NT];
#pragma unroll
        for (int tm = 0; tm < TERMS; tm++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
            b[tm][nt] = *reinterpret_cast<const uint2 *>(qs + ((tm * NT + nt) * KS + ks) * 64 + lane * 2);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
          const uint32_t w0 = (&kr[mt][0][ks / 4].x)[ks % 4] ^ 0x80808080u, w1 = (&kr[mt][1][ks / 4].x)[ks % 4] ^ 0x80808080u;
          const uint32_t af[4] = {half_pair<0x4240>(w0), half_pair<0x4240>(w1), half_pair<0x4341>(w0), half_pair<0x4341>(w1)};
#pragma unroll
          for (int tm = 0; tm < TERMS; tm++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma16816(s[mt][nt], af, b[tm][nt].x, b[tm][nt].y);
        }
      }
      // scores in units of log2, the unseen at -inf
      const bool edge = key < t.lo_all || key + MT * 16 > t.hi_all;
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[mt][nt][j] *= ks_[mt] * col[nt][j & 1];
      bool hole = false;
#pragma unroll
      for (int mt = 0; mt < MT; mt++) hole |= page[mt] < 0;
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
              const bool y = page[mt] >= 0 && kk >= lo[nt][j & 1] && kk < hi[nt][j & 1];
              if (!y) s[mt][nt][j] = -INFINITY;
              seen |= (y ? 1u : 0u) << ((mt * NT + nt) * 4 + j);
            }
      }
      // the next step's keys, now that these are used up
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        page[mt] = page_next[mt];
        page_next[mt] = i + 2 < take ? page_of(key + 2 * GRAN + mt * 16) : -1;
      }
      if (i + 1 < take) load_k(key + GRAN, page);

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
      float vtop = vmax;
#pragma unroll
      for (int mt = 0; mt < MT; mt++) vtop = fmaxf(vtop, fabsf(vs_[mt]));
      if (__any_sync(~0u, moved) || vtop != vmax) {
        const float vr_ = vtop != vmax ? __fdiv_rn(vmax, vtop) : 1.0f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float f = m[nt][e] == -INFINITY ? 0.0f : ex2(m[nt][e] - mn[nt][e]);
            l[nt][e] *= f;
            m[nt][e] = mn[nt][e];
            const float fo = f * vr_;
#pragma unroll
            for (int w = 0; w < VW * 2; w++) {
              o[nt][w][e] *= fo;
              o[nt][w][2 + e] *= fo;
            }
          }
        vmax = vtop;
      }
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        // 2^14 sv / largest sv; a scale that is not finite makes the weights of the keys that are seen NaN
        const float ratio = vmax > 0.0f ? __fdiv_rn(vs_[mt], vmax) * 16384.0f : vs_[mt];
        uint32_t pb[TERMS][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float top = m[nt][j & 1] == -INFINITY ? 0.0f : m[nt][j & 1];
            const float e = ex2(s[mt][nt][j] - top);
            l[nt][j & 1] += e;
            p[j] = e * ratio;
          }
          if (edge || hole) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              if (!(seen >> ((mt * NT + nt) * 4 + j) & 1)) p[j] = 0.0f;
          }
          const uint32_t p01 = pack_half(p[0], p[1]), p23 = pack_half(p[2], p[3]);
          pb[0][nt][0] = transpose8x8(p01);
          pb[0][nt][1] = transpose8x8(p23);
          if constexpr (TERMS == 2) {
            const float2 h01 = __half22float2(*reinterpret_cast<const __half2 *>(&p01));
            const float2 h23 = __half22float2(*reinterpret_cast<const __half2 *>(&p23));
            pb[1][nt][0] = transpose8x8(pack_half(p[0] - h01.x, p[1] - h01.y));
            pb[1][nt][1] = transpose8x8(pack_half(p[2] - h23.x, p[3] - h23.y));
          }
        }
        // O^T += V^T P^T: word w of a lane holds dimensions 4w .. 4w + 3 of four keys
#pragma unroll
        for (int w = 0; w < VW; w++) {
          const uint32_t x0 = vr[mt][0][w] ^ 0x80808080u, x1 = vr[mt][1][w] ^ 0x80808080u;
          const uint32_t x2 = vr[mt][2][w] ^ 0x80808080u, x3 = vr[mt][3][w] ^ 0x80808080u;
          const uint32_t a01 = __byte_perm(x0, x1, 0x5140), b01 = __byte_perm(x0, x1, 0x7362);
          const uint32_t a23 = __byte_perm(x2, x3, 0x5140), b23 = __byte_perm(x2, x3, 0x7362);
          const uint32_t f0[4] = {half_pair<0x4140>(a01), half_pair<0x4342>(a01), half_pair<0x4140>(a23), half_pair<0x4342>(a23)};
          const uint32_t f1[4] = {half_pair<0x4140>(b01), half_pair<0x4342>(b01), half_pair<0x4140>(b23), half_pair<0x4342>(b23)};
#pragma unroll
          for (int tm = 0; tm < TERMS; tm++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              mma16816(o[nt][2 * w], f0, pb[tm][nt][0], pb[tm][nt][1]);
              mma16816(o[nt][2 * w + 1], f1, pb[tm][nt][0], pb[tm][nt][1]);
            }
        }
      }
      if (i + 1 < take) load_v(key + GRAN, page);
    }

    // The warps' results meet in shared memory.
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
    const bool whole = take == units;
    float *part = whole ? nullptr : partial_at<ROWS, DP>(a, blockIdx.x, cur.off == 0);
    for (int i = threadIdx.x; i < ROWS * DP / 4; i += kThreads) {
      const int row = i / (DP / 4), d = (i % (DP / 4)) * 4;
      if (row >= t.rows) break;
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
        if (d < D) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          write_out<T>(a, t, head, row, d, sum == 0.0f ? 0.0f : r.x * inv);
          write_out<T>(a, t, head, row, d + 1, sum == 0.0f ? 0.0f : r.y * inv);
          write_out<T>(a, t, head, row, d + 2, sum == 0.0f ? 0.0f : r.z * inv);
          write_out<T>(a, t, head, row, d + 3, sum == 0.0f ? 0.0f : r.w * inv);
        }
        if (d == 0) write_lse(a, t, head, row, top, sum);
      } else {
        *reinterpret_cast<float4 *>(part + row * DP + d) = r;
        if (d == 0) {
          part[ROWS * DP + row] = top;
          part[ROWS * DP + ROWS + row] = sum;
        }
      }
    }
    if (!whole) arrive<T, ROWS, DP, kThreads>(a, t, cur, u0, u1, body, flag);
    __syncthreads();
    cur.at += take;
    cur.off = 0;
    cur.slot++;
    if (cur.slot == a.slots) {
      cur.slot = 0;
      cur.head++;
    }
  }
}

template <typename T, int DP, int NT, int PER_SM>
int launch_rows(AttendArgs a, int sms, cudaStream_t st) {
  using S = Shape<T, DP, NT>;
  constexpr size_t smem = S::WORDS * 4;
  auto *kern = k_kv_attend_rows<T, DP, NT, PER_SM>;
  if (smem > 48 * 1024) SHLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  a.slots = (int)(((int64_t)a.batch.tokens * a.group) / S::ROWS + a.batch.seqs);
  // No more blocks than granules there can be.
  const int64_t room = ((int64_t)a.batch.table_pages << a.page_shift) / S::GRAN + 1;
  int64_t most = (int64_t)a.slots * a.pool.heads;
  most = most > (1 << 20) ? most : most * room;
  const int64_t full = (int64_t)sms * PER_SM;
  int64_t grid = most < full ? most : full;
  if (grid > kAttendMaxBlocks) grid = kAttendMaxBlocks;
  if (grid < 1) grid = 1;
  kern<<<(unsigned)grid, kThreads, smem, st>>>(a, 1);
  return launch_check("kv_attend");
}

template <typename T>
int dispatch_rows(const AttendArgs &a, int nt, int sms, cudaStream_t st) {
  const int D = a.pool.head_dim;
  if (nt == 1) {
    if (D <= 64) return launch_rows<T, 64, 1, 4>(a, sms, st);
    if (D <= 128) return launch_rows<T, 128, 1, 3>(a, sms, st);
    return launch_rows<T, 256, 1, 2>(a, sms, st);
  }
  if (D <= 64) return launch_rows<T, 64, 2, 3>(a, sms, st);
  if (D <= 128) return launch_rows<T, 128, 2, 2>(a, sms, st);
  return launch_rows<T, 256, 2, 2>(a, sms, st);
}

constexpr size_t kCounterBytes = 2 * kAttendMaxBlocks * sizeof(unsigned);

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
  of(8, 64, 4); of(8, 128, 3); of(8, 256, 2); of(16, 64, 3); of(16, 128, 2); of(16, 256, 2);
  return kCounterBytes + most;
}

int launch_kv_attend(const AttendCall &c, int sms, cudaStream_t st) {
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
  a.scale_log2 = c.scale * 1.44269504088896341f;
  a.page_shift = 31 - __builtin_clz((unsigned)c.pool.page_tokens);
  a.above = 0;
  a.upto = (int64_t)1 << 40;
  a.counters = static_cast<unsigned *>(c.work);
  a.partials = reinterpret_cast<float *>(static_cast<char *>(c.work) + kCounterBytes);
  // Tiles of 8 rows where the sequences have 8 or fewer on average, else 16.
  const int nt = (int64_t)c.batch.tokens * group <= (int64_t)8 * c.batch.seqs ? 1 : 2;
  return c.dtype == kF16 ? dispatch_rows<__half>(a, nt, sms, st) : dispatch_rows<float>(a, nt, sms, st);
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_kv_attend_workspace(size_t *bytes) {
  if (!bytes) return fail("kv_attend workspace: null pointer");
  Device *dev;
  SHLO_TRY(current_device(&dev));
  *bytes = attend_work_bytes(dev->sm_count);
  return 0;
}

int shlo_kv_attend_noalloc(const shlo_kv_pool *pool, const shlo_kv_batch *batch, const void *q, int64_t q_token,
                           int64_t q_head, int32_t heads, uint8_t dtype, float scale, int32_t causal, int32_t window,
                           void *out, int64_t out_token, int64_t out_head, float *lse, void *workspace,
                           size_t workspace_bytes, void *stream) {
  if (!pool || !batch) return fail("kv_attend: null descriptor");
  Device *dev;
  SHLO_TRY(current_device(&dev));
  AttendCall c{*pool, *batch, q, q_token, q_head, out, out_token, out_head, lse, heads, dtype, scale, causal != 0, window,
               workspace, workspace_bytes};
  return launch_kv_attend(c, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
