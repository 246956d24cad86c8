// The norm of queries and keys for each head, with the position rotation in the
// same pass, and its gradient. A head x of D values becomes
//   n = x / sqrt(mean(x^2) + eps),   z = n w,   y = turn(z, position),
// where w is the queries' weight for the first q_heads heads and the keys' for
// the others, and turn is rope.cu's (pairs of the first `rot` dimensions, the
// angles' arithmetic too). Of dy:
//   dz = turn(dy, -position),  dw = sum of dz n over tokens and heads,
//   g = dz w,   dx = (g - n mean(g n)) / sqrt(mean(x^2) + eps).
//
// Bound: bytes (each value read once and written once); what keeps it from a copy's rate
// are waits, with the 16 warps an SM that the registers leave (the gradient: 24), whose
// issue slots are 51 % used (63 %): for the loads, of which few are ahead, and for the
// sums over a group, two of them one after the other in the gradient. A group of 1 to 32
// lanes holds a head in registers; it keeps one token and goes over heads, so that its
// pairs' cosines and sines, and the weight, stay in registers too (forward: their
// products); heads to come are asked for ahead, up to four of them forward and one
// backward. Two pairs go through each packed instruction.
// Measured on one B200: 16384 tokens x 40 heads x 128, float16 (336 MB) 63 us, 5.3 TB/s
// (rope.cu alone 55); the gradient of 24001 x 12 x 80 float32, 32 dimensions turned in
// interleaved pairs (277 MB) 70 us, 3.9 TB/s: ten units of eight values a head, on ten
// lanes, three heads a warp (82 us on 16 lanes). Measured and left there, on 16 lanes:
// four blocks an SM (125 us, registers to memory) and two (91 us), no head ahead (88 us).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 16;  // heads of a token that the weights' gradients are summed over in binary32
constexpr int kBackBlocksPerSm = 3;  // the backward pass's, with four pairs a lane or fewer (eight need the registers of two)

struct NormArgs {
  const void *x, *dy;
  void *y;  // dx in the backward pass
  const int32_t *pos;
  const int64_t *phases;
  const void *wq, *wk;
  int64_t xt, xh, gt, gh, yt, yh;  // token and head strides, in values (g: dy's)
  int64_t tokens;
  int heads, q_heads, dim, rot;
  int odd, lanes_log;  // lanes a group: odd << lanes_log
  int nt_log;  // tokens a block (at a time)
  int hb;      // heads a block
  float eps, factor;
  bool w_half, w_wide;  // the weights' type, and whether they allow wide loads
  double *partials;     // backward: [blocks][2][dim], nullptr without the weights' gradients
};

template <int BYTES> struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<2> { using T = uint16_t; };

__device__ __forceinline__ float to_f32(__half h) { return __half2float(h); }
__device__ __forceinline__ float to_f32(float f) { return f; }
__device__ __forceinline__ void of_f32(__half &d, float f) { d = __float2half_rn(f); }
__device__ __forceinline__ void of_f32(float &d, float f) { d = f; }

// A lane's part of a head: NS slots of two vectors of VEC values. The first
// rot / 2 / VEC slots of a head hold pairs (the vectors half the part apart, or
// side by side); the others two vectors of the part that is not turned, the last
// of which may have one only. Side by side, a slot may be turned in part: the pairs
// of the rest of it are turned by nothing, and rot need be no multiple of anything.
template <typename T, int VEC, int NS> struct Part {
  T v[NS][2][VEC];
};
template <int NS> struct Places {
  int o[NS], o2[NS];  // -1: none
  bool pair[NS];
};

template <int VEC, int NS, bool INTER>
__device__ __forceinline__ void places(const NormArgs &a, int L, bool there, int lane, Places<NS> &p) {
  const int half = a.rot / 2, ru = (half + VEC - 1) / VEC, cv = INTER ? 0 : (a.dim - a.rot) / VEC;
#pragma unroll
  for (int s = 0; s < NS; s++) {
    const int u = lane + s * L, c = 2 * (u - ru);
    p.pair[s] = there && u < ru;
    if (INTER) {
      p.o[s] = there && 2 * VEC * u < a.dim ? 2 * VEC * u : -1;
      p.o2[s] = there && 2 * VEC * u + VEC < a.dim ? 2 * VEC * u + VEC : -1;
    } else {
      p.o[s] = !there ? -1 : u < ru ? VEC * u : c < cv ? a.rot + c * VEC : -1;
      p.o2[s] = !there ? -1 : u < ru ? p.o[s] + half : c + 1 < cv ? a.rot + (c + 1) * VEC : -1;
    }
  }
}
template <typename T, int VEC, int NS>
__device__ __forceinline__ void load_part(const T *x, const Places<NS> &p, Part<T, VEC, NS> &r) {
  using R = typename Raw<VEC * sizeof(T)>::T;
#pragma unroll
  for (int s = 0; s < NS; s++) {
    if (p.o[s] >= 0) *reinterpret_cast<R *>(r.v[s][0]) = *reinterpret_cast<const R *>(x + p.o[s]);
    if (p.o2[s] >= 0) *reinterpret_cast<R *>(r.v[s][1]) = *reinterpret_cast<const R *>(x + p.o2[s]);
  }
}
template <typename T, int VEC, int NS>
__device__ __forceinline__ void store_part(T *y, const Places<NS> &p, const Part<T, VEC, NS> &r) {
  using R = typename Raw<VEC * sizeof(T)>::T;
#pragma unroll
  for (int s = 0; s < NS; s++) {
    if (p.o[s] >= 0) *reinterpret_cast<R *>(y + p.o[s]) = *reinterpret_cast<const R *>(r.v[s][0]);
    if (p.o2[s] >= 0) *reinterpret_cast<R *>(y + p.o2[s]) = *reinterpret_cast<const R *>(r.v[s][1]);
  }
}
template <typename T, int VEC, int NS>
__device__ __forceinline__ void clear_part(Part<T, VEC, NS> &r) {
#pragma unroll
  for (int s = 0; s < NS; s++)
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) of_f32(r.v[s][k][j], 0.0f);
}
// The two values of pair j of a slot.
template <int VEC, bool INTER, typename V> __device__ __forceinline__ V &first(V (&v)[2][VEC], int j) { return INTER ? v[(2 * j) / VEC][(2 * j) % VEC] : v[0][j]; }
template <int VEC, bool INTER, typename V> __device__ __forceinline__ V &second(V (&v)[2][VEC], int j) { return INTER ? v[(2 * j + 1) / VEC][(2 * j + 1) % VEC] : v[1][j]; }

// Over a group's lanes, the first of which is `base`: the same sum in each.
template <bool ODD> __device__ __forceinline__ float group_sum(float v, const NormArgs &a, int base) {
  for (int i = 0; i < a.lanes_log; i++) v += __shfl_xor_sync(~0u, v, 1 << i);
  if (ODD) {
    float sum = 0.0f;
    for (int i = 0; i < a.odd; i++) sum += __shfl_sync(~0u, v, base + (i << a.lanes_log));
    v = sum;
  }
  return v;
}

// Squares of 32-bit values can leave the range where the values themselves are
// well inside it: such a head is scaled by a power of two first. Returns the scale.
__device__ __forceinline__ float safe_scale(float ss, float eps) {
  if (!(ss < 0x1p120f)) return 0x1p-80f;
  if (ss < 0x1p-80f && eps < 0x1p-80f) return 0x1p66f;
  return 1.0f;
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg(float2 x) { return make_float2(-x.x, -x.y); }

// A part as pairs (a, b), two of them in a register pair. (Where a slot is not
// turned, its pairs' sine is 0.)
template <typename T, int VEC, int NS, bool INTER>
__device__ __forceinline__ void pairs(Part<T, VEC, NS> &r, float2 (&a)[NS * VEC / 2], float2 (&b)[NS * VEC / 2]) {
#pragma unroll
  for (int i = 0; i < NS * VEC / 2; i++) {
    constexpr int V = VEC;
    const int p = 2 * i, q = 2 * i + 1;
    a[i] = make_float2(to_f32(first<V, INTER>(r.v[p / V], p % V)), to_f32(first<V, INTER>(r.v[q / V], q % V)));
    b[i] = make_float2(to_f32(second<V, INTER>(r.v[p / V], p % V)), to_f32(second<V, INTER>(r.v[q / V], q % V)));
  }
}
template <typename T, int VEC, int NS, bool INTER>
__device__ __forceinline__ void unpairs(const float2 (&a)[NS * VEC / 2], const float2 (&b)[NS * VEC / 2], Part<T, VEC, NS> &r) {
#pragma unroll
  for (int i = 0; i < NS * VEC / 2; i++) {
    constexpr int V = VEC;
    const int p = 2 * i, q = 2 * i + 1;
    of_f32(first<V, INTER>(r.v[p / V], p % V), a[i].x);
    of_f32(first<V, INTER>(r.v[q / V], q % V), a[i].y);
    of_f32(second<V, INTER>(r.v[p / V], p % V), b[i].x);
    of_f32(second<V, INTER>(r.v[q / V], q % V), b[i].y);
  }
}

// BACK: the gradient. A block goes over tiles of 2^nt_log tokens, one in the
// forward pass, for the heads of its part. ODD: a group's lanes are not a power of two;
// a warp's last lanes may have no group. FEW: a group has few heads of a token, and more
// blocks take the place of heads asked for ahead.
constexpr int blocks_per_sm(int values, bool back, bool few) {
  return back ? (values <= 4 ? kBackBlocksPerSm : 2) : values <= 4 ? (few ? 4 : 3) : (few ? 3 : 2);
}
template <typename T, int VEC, int NS, bool INTER, bool BACK, bool ODD, bool FEW>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(NS * VEC, BACK, FEW)) k_norm_rope(const NormArgs a) {
  // Backward: 8 P sums a thread; then the cosines and sines, [token][half] each, and at
  // the end the block's sums, [warp][dim], in their place.
  extern __shared__ double sh[];
  constexpr int P = NS * VEC / 2, AHEAD = BACK ? 1 : P <= 2 ? 2 : FEW ? 1 : 4;  // heads asked for beside the one in hand
  const int half = a.rot / 2, row = (half + VEC - 1) / VEC * VEC, nt = 1 << a.nt_log;  // (row: a token's cosines)
  float *const cs = reinterpret_cast<float *>(sh + (BACK ? 8 * P * kThreads : 0)), *const sn = cs + nt * row;
  const int warp = threadIdx.x / 32, wl = threadIdx.x % 32;
  const int L = ODD ? a.odd << a.lanes_log : 1 << a.lanes_log, in_warp = ODD ? 32 / L : 32 >> a.lanes_log;  // groups
  const int lane = ODD ? wl % L : wl & (L - 1), base = wl - lane, group = ODD ? warp * in_warp + wl / L : (int)threadIdx.x >> a.lanes_log;
  const int groups = kThreads / 32 * in_warp;
  const bool works = !ODD || wl < in_warp * L;
  const int h0 = blockIdx.y * a.hb, h1 = min(h0 + a.hb, a.heads);
  Places<NS> at;
  places<VEC, NS, INTER>(a, L, works, lane, at);
  auto weight = [&](bool keys, float2 (&wa)[P], float2 (&wb)[P]) {
    const void *const wp = keys ? a.wk : a.wq;
    Part<float, VEC, NS> w;
    Part<__half, VEC, NS> wh;
    clear_part(w);
    if (wp && a.w_wide) {
      if (a.w_half) {
        clear_part(wh);
        load_part(static_cast<const __half *>(wp), at, wh);
        pairs<__half, VEC, NS, INTER>(wh, wa, wb);
        return;
      }
      constexpr int V = VEC < 4 ? VEC : 4;
      using R = typename Raw<V * sizeof(float)>::T;
#pragma unroll
      for (int s = 0; s < NS; s++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int o = k ? at.o2[s] : at.o[s];
#pragma unroll
          for (int j = 0; j < VEC; j += V)
            if (o >= 0) *reinterpret_cast<R *>(&w.v[s][k][j]) = *reinterpret_cast<const R *>(static_cast<const float *>(wp) + o + j);
        }
      pairs<float, VEC, NS, INTER>(w, wa, wb);
      return;
    }
#pragma unroll
    for (int s = 0; s < NS; s++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int o = k ? at.o2[s] : at.o[s];
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (o >= 0) w.v[s][k][j] = !wp ? 1.0f : a.w_half ? __half2float(static_cast<const __half *>(wp)[o + j]) : static_cast<const float *>(wp)[o + j];
      }
    pairs<float, VEC, NS, INTER>(w, wa, wb);
  };
  const int t = group & (nt - 1), h_first = h0 + (group >> a.nt_log), h_step = max(groups >> a.nt_log, 1);
  // Of a token's pairs the cosines and sines from shared memory, none where a slot is
  // not turned.
  auto turn = [&](float2 (&c)[P], float2 (&s)[P]) {
    constexpr int V = VEC < 4 ? VEC : 4;
    using R = typename Raw<V * sizeof(float)>::T;
    float cc[2 * P], ss[2 * P];
#pragma unroll
    for (int i = 0; i < 2 * P; i += V) {
      const int slot = i / VEC, p = t * row + (lane + slot * L) * VEC + i % VEC;
#pragma unroll
      for (int j = 0; j < V; j++) cc[i + j] = 1.0f, ss[i + j] = 0.0f;
      if (at.pair[slot]) {
        *reinterpret_cast<R *>(cc + i) = *reinterpret_cast<const R *>(cs + p);
        *reinterpret_cast<R *>(ss + i) = *reinterpret_cast<const R *>(sn + p);
      }
    }
#pragma unroll
    for (int i = 0; i < P; i++) {
      c[i] = make_float2(cc[2 * i], cc[2 * i + 1]);
      s[i] = make_float2(ss[2 * i], ss[2 * i + 1]);
    }
  };
  // Backward: a weight, and the sums of its gradient over kRun heads of a token at most;
  // then they go to the thread's sums in 64 bits, [weight][4 P], in shared memory, also
  // where the next heads are of the same kind (us, sums of the same kind kept over all
  // tokens and not: 16384 x 32 x 128 float16 98 and 100, 55000 x 1 x 64 21.1 and 22.4;
  // kept over up to 16 heads of several tokens 24001 x 12 x 80 float32 would take 77
  // instead of 69.5).
  float2 dwa[BACK ? P : 1], dwb[BACK ? P : 1], wa[BACK ? P : 1], wb[BACK ? P : 1];
  double *const sums = reinterpret_cast<double *>(sh) + threadIdx.x;
  int has = -1;  // whose weight is in registers: 0 the queries', 1 the keys'
  if constexpr (BACK) {
#pragma unroll
    for (int i = 0; i < P; i++) dwa[i] = dwb[i] = both(0.0f);
#pragma unroll
    for (int i = 0; i < 8 * P; i++) sums[i * kThreads] = 0.0;
  }
  auto flush = [&]() {
    if constexpr (BACK) {
      double *const to = sums + has * 4 * P * kThreads;
#pragma unroll
      for (int i = 0; i < P; i++) {
        to[(4 * i) * kThreads] += (double)dwa[i].x;
        to[(4 * i + 1) * kThreads] += (double)dwa[i].y;
        to[(4 * i + 2) * kThreads] += (double)dwb[i].x;
        to[(4 * i + 3) * kThreads] += (double)dwb[i].y;
        dwa[i] = dwb[i] = both(0.0f);
      }
    }
  };
  // (pair and token of this thread's angles, kThreads apart)
  const int tt_first = row ? (int)threadIdx.x / row : 0, p_first = (int)threadIdx.x - tt_first * row;
  const int dt = row ? kThreads / row : 0, dp = kThreads - dt * row;
  const float inv_dim = 1.0f / a.dim;
  const int64_t tiles = (a.tokens + nt - 1) >> a.nt_log;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t t0 = tile << a.nt_log;
    const bool mine = works && t0 + t < a.tokens;
    const T *x = static_cast<const T *>(a.x) + (t0 + t) * a.xt + h_first * a.xh;
    const T *g = BACK ? static_cast<const T *>(a.dy) + (t0 + t) * a.gt + h_first * a.gh : nullptr;
    T *y = static_cast<T *>(a.y) + (t0 + t) * a.yt + h_first * a.yh;
    const int64_t x_step = h_step * a.xh, g_step = h_step * a.gh, y_step = h_step * a.yh;
    // (the loads need nothing of the angles: they go out first)
    Part<T, VEC, NS> next[AHEAD], next_g[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
      clear_part(next[i]);
      if (BACK) clear_part(next_g[i]);
      if (mine && h_first + i * h_step < h1) {
        load_part(x + i * x_step, at, next[i]);
        if (BACK) load_part(g + i * g_step, at, next_g[i]);
      }
    }
    if (BACK && tile != (int64_t)blockIdx.x) __syncthreads();
    for (int i = threadIdx.x, p = p_first, tt = tt_first; i < nt * row; i += kThreads) {
      if (t0 + tt < a.tokens) {
        float s = 0.0f, c = 1.0f;
        if (!INTER || p < half) {
          const int64_t turns = (int64_t)((uint64_t)(int64_t)a.pos[t0 + tt] * (uint64_t)a.phases[p]) >> 32;
          sincospif((float)turns * 0x1p-31f, &s, &c);
          c *= a.factor;
          s *= a.factor;
        }
        cs[i] = c;
        sn[i] = s;
      }
      p += dp;
      tt += dt;
      if (p >= row) p -= row, tt++;
    }
    __syncthreads();
    // Forward: what a pair's two results take of its two values, weight and turn in
    // one: (a, b) -> (a ca + b sb, b cb + a sa). Backward: the turn, its sine negated too.
    float2 ca[P], sa[P], cb[BACK ? 1 : P], sb[P];
    if constexpr (BACK) {
      turn(ca, sa);
#pragma unroll
      for (int i = 0; i < P; i++) sb[i] = neg(sa[i]);
    } else {
      has = -1;
    }
    // (a warp's groups take the same number of turns: its shuffles name all lanes)
    for (int h = h0, stop = BACK ? h0 : h1; h < h1;) {
      if (BACK) stop = min(stop + kRun * h_step, h1);
      for (; h < stop; h += AHEAD * h_step) {
#pragma unroll
        for (int ahead = 0; ahead < AHEAD; ahead++) {
          if (AHEAD > 1 && h + ahead * h_step >= h1) break;
          const int hh = h + ahead * h_step + (group >> a.nt_log);
          const bool there = mine && hh < h1;
          if (has != (int)(hh >= a.q_heads)) {
            if (BACK && has >= 0) flush();
            has = hh >= a.q_heads;
            if constexpr (BACK) {
              weight(has, wa, wb);
            } else {
              float2 c[P], s[P], u[P], v[P];
              turn(c, s);
              weight(has, u, v);
#pragma unroll
              for (int i = 0; i < P; i++) {
                ca[i] = __fmul2_rn(u[i], c[i]);
                sa[i] = __fmul2_rn(u[i], s[i]);
                cb[i] = __fmul2_rn(v[i], c[i]);
                sb[i] = __fmul2_rn(v[i], neg(s[i]));
              }
            }
          }
          float2 xa[P], xb[P], sum = both(0.0f);
          pairs<T, VEC, NS, INTER>(next[ahead], xa, xb);
          Part<T, VEC, NS> in_g;
          if (BACK) in_g = next_g[ahead];
          if (mine && hh + AHEAD * h_step < h1) {
            load_part(x + AHEAD * x_step, at, next[ahead]);
            if (BACK) load_part(g + AHEAD * g_step, at, next_g[ahead]);
          }
#pragma unroll
          for (int i = 0; i < P; i++) sum = __ffma2_rn(xb[i], xb[i], __ffma2_rn(xa[i], xa[i], sum));
          float ss = group_sum<ODD>(sum.x + sum.y, a, base), scale = 1.0f, eps = a.eps;
          if (sizeof(T) == 4) {
            scale = safe_scale(ss, eps);
            if (__any_sync(~0u, scale != 1.0f)) {
              eps = eps * scale * scale;  // (scale^2 itself has no place in 32 bits)
              sum = both(0.0f);
#pragma unroll
              for (int i = 0; i < P; i++) {
                xa[i] = __fmul2_rn(xa[i], both(scale));
                xb[i] = __fmul2_rn(xb[i], both(scale));
                sum = __ffma2_rn(xb[i], xb[i], __ffma2_rn(xa[i], xa[i], sum));
              }
              ss = group_sum<ODD>(sum.x + sum.y, a, base);
            }
          }
          // (2^-22 is enough where the result has 11 bits)
          const float inv = sizeof(T) == 2 ? rsqrtf(__fmaf_rn(ss, inv_dim, eps)) : __frsqrt_rn(__fmaf_rn(ss, inv_dim, eps));
          float2 ya[P], yb[P];
          if constexpr (!BACK) {
#pragma unroll
            for (int i = 0; i < P; i++) {
              const float2 p = __fmul2_rn(xa[i], both(inv)), q = __fmul2_rn(xb[i], both(inv));
              ya[i] = __ffma2_rn(q, sb[i], __fmul2_rn(p, ca[i]));
              yb[i] = __ffma2_rn(q, cb[i], __fmul2_rn(p, sa[i]));
            }
          } else {
            float2 ga[P], gb[P], dot = both(0.0f);
            pairs<T, VEC, NS, INTER>(in_g, ga, gb);
#pragma unroll
            for (int i = 0; i < P; i++) {
              xa[i] = __fmul2_rn(xa[i], both(inv));
              xb[i] = __fmul2_rn(xb[i], both(inv));
              // turned back
              const float2 p = __ffma2_rn(ga[i], ca[i], __fmul2_rn(gb[i], sa[i]));
              const float2 q = __ffma2_rn(ga[i], sb[i], __fmul2_rn(gb[i], ca[i]));
              if (there) {
                dwa[i] = __ffma2_rn(p, xa[i], dwa[i]);
                dwb[i] = __ffma2_rn(q, xb[i], dwb[i]);
              }
              ga[i] = __fmul2_rn(p, wa[i]);
              gb[i] = __fmul2_rn(q, wb[i]);
              dot = __ffma2_rn(gb[i], xb[i], __ffma2_rn(ga[i], xa[i], dot));
            }
            const float gn = -(group_sum<ODD>(dot.x + dot.y, a, base) * inv_dim);
#pragma unroll
            for (int i = 0; i < P; i++) {
              ya[i] = __fmul2_rn(__ffma2_rn(xa[i], both(gn), ga[i]), both(inv));
              yb[i] = __fmul2_rn(__ffma2_rn(xb[i], both(gn), gb[i]), both(inv));
              if (sizeof(T) == 4) {
                ya[i] = __fmul2_rn(ya[i], both(scale));
                yb[i] = __fmul2_rn(yb[i], both(scale));
              }
            }
          }
          Part<T, VEC, NS> out;
          unpairs<T, VEC, NS, INTER>(ya, yb, out);
          if (there) store_part(y, at, out);
          x += x_step;
          y += y_step;
          if (BACK) g += g_step;
        }
      }
      if (BACK) flush(), has = -1;
    }
  }
  if constexpr (BACK) {
    if (!a.partials) return;
    // The block's sums, of one weight and then of the other: a warp's groups, then the
    // warps one after the other.
    double *const rows = reinterpret_cast<double *>(cs);
    for (int k0 = 0; k0 < 2; k0++) {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < 2 * P; p++)
#pragma unroll
        for (int q = 0; q < 2; q++) {  // pair p's first and second value
          constexpr int V = VEC;
          const int s = p / V, j = p % V, k = INTER ? (2 * j + q) / V : q, at_j = INTER ? (2 * j + q) % V : j;
          const int o = k ? at.o2[s] : at.o[s];
          double v = sums[(k0 * 4 * P + p / 2 * 4 + 2 * q + p % 2) * kThreads];
          if (!ODD) {
            for (int i = L; i < 32; i *= 2) v += __shfl_xor_sync(~0u, v, i);
          } else {
            const double mine = v;
            for (int i = 1; i < in_warp; i++) v += __shfl_sync(~0u, mine, (wl + i * L) % 32);
          }
          if (wl < L && o >= 0) rows[warp * a.dim + o + at_j] = v;
        }
      __syncthreads();
      double *const to = a.partials + (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + k0) * a.dim;
      for (int i = threadIdx.x; i < a.dim; i += kThreads) {
        double sum = 0.0;
        for (int k = 0; k < kThreads / 32; k++) sum += rows[k * a.dim + i];
        to[i] = sum;
      }
    }
  }
}

// The blocks' sums of a weight's gradient, added in one order: blockIdx.y 0 the
// queries', 1 the keys'. 32 dimensions a block.
__global__ void __launch_bounds__(1024) k_norm_rope_dw(const double *partials, int blocks, int dim, float *dq, float *dk) {
  __shared__ double sums[32][33];
  const int c = threadIdx.x % 32, r = threadIdx.x / 32, i = blockIdx.x * 32 + c;
  float *const to = blockIdx.y ? dk : dq;
  if (!to) return;
  cudaGridDependencySynchronize();  // (it may begin before the sums are there)
  double sum = 0.0;
  if (i < dim)
    for (int k = r; k < blocks; k += 32) sum += partials[((int64_t)k * 2 + blockIdx.y) * dim + i];
  sums[r][c] = sum;
  __syncthreads();
  if (r == 0 && i < dim) {
    sum = 0.0;
    for (int k = 0; k < 32; k++) sum += sums[k][c];
    to[i] = (float)sum;
  }
}

template <typename T, int VEC, int NS, bool ODD>
int launch(const NormArgs &a, bool inter, bool back, bool few, dim3 grid, size_t smem, cudaStream_t st) {
  const auto kernel = back ? inter ? k_norm_rope<T, VEC, NS, true, true, ODD, false> : k_norm_rope<T, VEC, NS, false, true, ODD, false>
                      : few ? inter ? k_norm_rope<T, VEC, NS, true, false, ODD, true> : k_norm_rope<T, VEC, NS, false, false, ODD, true>
                            : inter ? k_norm_rope<T, VEC, NS, true, false, ODD, false> : k_norm_rope<T, VEC, NS, false, false, ODD, false>;
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> set[2]{};
    int device;
    SHLO_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !(set[inter].load(std::memory_order_relaxed) >> device & 1)) {
      SHLO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024));
      if (device < 64) set[inter].fetch_or(1ull << device);
    }
  }
  kernel<<<grid, kThreads, smem, st>>>(a);
  return launch_check(back ? "norm_rope_grad" : "norm_rope");
}

// Blocks of the backward pass: their sums go to the workspace.
int back_blocks(int sms) { return sms * kBackBlocksPerSm; }

}  // namespace

size_t norm_rope_work_bytes(int sms) { return (size_t)back_blocks(sms) * 2 * 512 * sizeof(double); }

int launch_norm_rope(const NormRopeCall &c, bool back, int sms, cudaStream_t st) {
  const char *const what = back ? "norm_rope_grad" : "norm_rope";
  if (c.dtype != kF16 && c.dtype != kF32) return fail("%s: %s not carried (float16 or float32)", what, dtype_name(c.dtype));
  if (c.weight_dtype != kF16 && c.weight_dtype != kF32) return fail("%s: weights of %s not carried (float16 or float32)", what, dtype_name(c.weight_dtype));
  // (the kernel counts heads in 32 bits, up to a block's turns beyond the last)
  if (c.tokens < 0 || c.heads < 1 || c.heads > (1 << 30) || c.dim < 1 || c.dim > 512)
    return fail("%s: %lld tokens, %d heads (1 to 2^30) of %d (1 to 512)", what, (long long)c.tokens, c.heads, c.dim);
  if (c.q_heads < 0 || c.q_heads > c.heads) return fail("%s: %d query heads of %d", what, c.q_heads, c.heads);
  if (c.rot < 0 || c.rot > c.dim || c.rot % 2) return fail("%s: %d of %d dimensions turned (an even number)", what, c.rot, c.dim);
  if (c.flags & ~1u) return fail("%s: flags 0x%x", what, c.flags);
  if (!(c.eps > 0.0f) || !std::isfinite(c.eps)) return fail("%s: eps %g (finite, above 0)", what, c.eps);
  if (c.tokens > 0x7fffffff) return fail("%s: %lld tokens, at most 2^31 - 1", what, (long long)c.tokens);
  const size_t size = dtype_size(c.dtype), wsize = dtype_size(c.weight_dtype);
  const bool sums = back && (c.dq_weight || c.dk_weight);
  if ((uintptr_t)c.dq_weight % 4 || (uintptr_t)c.dk_weight % 4 || (sums && (uintptr_t)c.workspace % 8)) return fail("%s: misaligned gradient or workspace", what);
  if (sums && (!c.workspace || c.workspace_bytes < norm_rope_work_bytes(sms)))
    return fail("%s: a workspace of %zu bytes, %zu needed", what, c.workspace ? c.workspace_bytes : 0, norm_rope_work_bytes(sms));
  if (sums && meet(c.dq_weight, c.dim * 4, c.dk_weight, c.dim * 4)) return fail("%s: the two weights' gradients share memory", what);
  // What is written beside the rows, against what is read, and the rows against that.
  const int64_t w_bytes = c.dim * (int64_t)wsize, work = sums ? (int64_t)norm_rope_work_bytes(sms) : 0;
  const struct { const void *p; int64_t bytes; } small[4] = {
      {c.q_weight, w_bytes}, {c.k_weight, w_bytes}, {c.rot ? c.positions : nullptr, 4 * c.tokens}, {c.rot ? c.phases : nullptr, 4 * (int64_t)c.rot}};
  auto in_rows = [&](const void *p, int64_t bytes) {
    auto rows = [&](const void *x, int64_t token, int64_t head) {
      return meet(x, c.tokens, token * (int64_t)size, c.heads, head * (int64_t)size, c.dim * (int64_t)size, p, bytes);
    };
    return rows(c.x, c.x_token, c.x_head) || rows(c.y, c.y_token, c.y_head) || (back && rows(c.dy, c.dy_token, c.dy_head));
  };
  const struct { const void *p; int64_t bytes; } made[3] = {{back ? c.dq_weight : nullptr, 4 * (int64_t)c.dim}, {back ? c.dk_weight : nullptr, 4 * (int64_t)c.dim}, {sums ? c.workspace : nullptr, work}};
  for (const auto &m : made) {
    bool used = in_rows(m.p, m.bytes);
    for (const auto &i : small) used = used || meet(m.p, m.bytes, i.p, i.bytes);
    if (used) return fail("%s: a weight's gradient or the workspace shares memory with an operand or dx", what);
  }
  if (sums && (meet(c.workspace, work, c.dq_weight, 4 * (int64_t)c.dim) || meet(c.workspace, work, c.dk_weight, 4 * (int64_t)c.dim)))
    return fail("%s: a weight's gradient shares memory with the workspace", what);
  for (const auto &i : small)
    if (meet(c.y, c.tokens, c.y_token * (int64_t)size, c.heads, c.y_head * (int64_t)size, c.dim * (int64_t)size, i.p, i.bytes))
      return fail("%s: %s shares memory with a weight, positions or phases", what, back ? "dx" : "y");
  if (c.tokens == 0) {
    if (c.dq_weight) SHLO_CUDA(cudaMemsetAsync(c.dq_weight, 0, c.dim * sizeof(float), st));
    if (c.dk_weight) SHLO_CUDA(cudaMemsetAsync(c.dk_weight, 0, c.dim * sizeof(float), st));
    return 0;
  }
  if (!c.x || !c.y || (back && !c.dy) || (c.rot && (!c.positions || !c.phases))) return fail("%s: null pointer", what);
  if ((c.tokens > 1 && llabs(c.y_token) < c.dim) || (c.heads > 1 && llabs(c.y_head) < c.dim))
    return fail("%s: rows of %s overlap", what, back ? "dx" : "y");
  if (((uintptr_t)c.x | (uintptr_t)c.y | (back ? (uintptr_t)c.dy : 0)) % size) return fail("%s: an operand is not aligned to its type", what);
  if (((uintptr_t)c.q_weight | (uintptr_t)c.k_weight) % wsize) return fail("%s: a weight is not aligned to its type", what);
  if ((uintptr_t)c.positions % 4 || (uintptr_t)c.phases % 8) return fail("%s: misaligned positions or phases", what);
  SHLO_TRY(check_in_place(c.x, c.x_token, c.x_head, c.y, c.y_token, c.y_head, c.tokens, c.heads, c.dim, size, what, "x", back ? "dx" : "y"));
  if (back)
    SHLO_TRY(check_in_place(c.dy, c.dy_token, c.dy_head, c.y, c.y_token, c.y_head, c.tokens, c.heads, c.dim, size, what, "dy", "dx"));
  // The widest vector (16 bytes at most) that every offset is a multiple of. (16384 tokens
  // of 40 heads of 72, 18 turned, float16, pairs side by side: 48 us with eight values,
  // which needs no half of them to be whole vectors, 144 with one; the gradient 92 and 260.
  // Half the turned part apart they are 144 and 293: one value at a time.)
  const int half = c.rot / 2, rest = c.dim - c.rot;
  const bool inter = (c.flags & 1) != 0;
  int vec = (int)(16 / size);
  const bool strided_h = c.heads > 1, strided_t = c.tokens > 1;
  auto fits = [&](int v) {
    auto row = [&](const void *p, int64_t token, int64_t head) {
      return (uintptr_t)p % (v * size) == 0 && (!strided_t || token % v == 0) && (!strided_h || head % v == 0);
    };
    return (inter ? c.dim % v == 0 : half % v == 0 && rest % v == 0) && row(c.x, c.x_token, c.x_head) && row(c.y, c.y_token, c.y_head) && (!back || row(c.dy, c.dy_token, c.dy_head));
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  // A lane's slots: 8 / vec of them (as many as its registers are made for) where
  // narrow vectors would leave it few values of a head, and there are heads enough for
  // all lanes; else as few as hold the head in 32 lanes. (750000 tokens' heads of 72, 36
  // turned, float16: 45 us with four slots and 84 with one; 55000 tokens of one such
  // head: 57 and 42.)
  const int units = inter ? (c.dim / vec + 1) / 2 : half / vec + (rest / vec + 1) / 2;
  const bool narrow = c.dtype == kF16 ? vec <= 4 : vec <= 2;
  const int slots = vec == 8 ? 1 : units > 32 || (narrow && c.heads >= 4) ? 8 / vec : vec == 1 ? 2 : 1;
  NormArgs a;
  a.x = c.x; a.dy = c.dy; a.y = c.y; a.pos = c.positions; a.phases = c.phases; a.wq = c.q_weight; a.wk = c.k_weight;
  a.xt = c.x_token; a.xh = c.x_head; a.gt = c.dy_token; a.gh = c.dy_head; a.yt = c.y_token; a.yh = c.y_head;
  a.tokens = c.tokens; a.heads = c.heads; a.q_heads = c.q_heads; a.dim = c.dim; a.rot = c.rot;
  a.eps = c.eps; a.factor = c.factor; a.w_half = c.weight_dtype == kF16;
  a.partials = sums ? (double *)c.workspace : nullptr;
  a.lanes_log = 0, a.odd = 1;
  while (a.lanes_log < 5 && (slots << a.lanes_log) < units) a.lanes_log++;
  // A block's tokens, as long as every SM gets blocks: eight, or more where their heads
  // are fewer than its groups; then its heads are shared among blocks while there are
  // fewer than two a SM.
  int step = 1, groups = 0;
  auto tokens_log = [&](int lanes) {
    int n = 0;
    groups = kThreads / 32 * (32 / lanes);
    while (groups % (2 << n) == 0 && (n < 3 || (groups >> n) > c.heads) && (c.tokens >> (n + 1)) >= 4 * sms) n++;
    step = groups >> n;
    return n;
  };
  a.nt_log = tokens_log(1 << a.lanes_log);
  // Five, six or ten lanes a group, where a block then takes fewer turns over its heads
  // for as many tokens. (80 dimensions, 32 turned, float32, the gradient of 24001 x 12: ten
  // lanes 69 us, sixteen 82.5; 16384 tokens of 40 heads of 72, 18 turned, side by side,
  // float16: 48 and 53.6, all turned, the gradient: 93.6 and 110. Of vectors of two values,
  // which are apart in memory, 8192 x 40 x 80 float32, 36 turned, would take 81 instead of
  // 72, and the gradient 98 instead of 118.)
  if (vec >= 4)
    for (const int lanes : {5, 6, 10})
      if (lanes < 1 << a.lanes_log && slots * lanes >= units) {
        const int turns = (c.heads + step - 1) / step, n = tokens_log(lanes);
        if (n == a.nt_log && (c.heads + step - 1) / step < turns) {
          a.odd = lanes % 2 ? lanes : lanes / 2, a.lanes_log = lanes % 2 ? 0 : 1;
          break;
        }
        tokens_log(1 << a.lanes_log);
      }
  const int64_t tiles = (c.tokens + (1 << a.nt_log) - 1) >> a.nt_log;
  int parts = 1;
  while (tiles * parts < 2 * sms && parts < (c.heads + step - 1) / step) parts++;
  a.hb = (c.heads + parts - 1) / parts;
  // (us, with four heads ahead and two blocks on an SM, and with one and three; tokens x
  // heads x dimensions, float16: 16384 x 40 x 128, ten turns, 62.7 and 68.5; 32768 x 40 x 64,
  // five, 68.4 and 72.9; 16384 x 7 x 256, four, 32.8 and 31.1; 436000 x 3 x 64, two, 182 and
  // 146. Four values a lane, two heads ahead, three blocks and four, float32: 8192 x 40 x
  // 80, 14 turns, 45.9 and 43.3; of 128 dimensions, 20 turns, it goes by the
  // tokens of 40 heads: 6100 45.3 and 50.7, 8192 62.6 and 60.4, 16384 112 and 114.)
  const bool few = (a.hb + step - 1) / step <= (slots * vec > 4 ? 4 : 14);
  dim3 grid((unsigned)tiles, (unsigned)((c.heads + a.hb - 1) / a.hb));
  // The backward pass has as many blocks as run at once, each with a row of sums.
  if (back) grid.x = (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles, (slots * vec > 4 ? 2 * sms : back_blocks(sms)) / grid.y));
  size_t smem = (size_t)(1 << a.nt_log) * ((half + vec - 1) / vec * vec) * 2 * sizeof(float);
  if (back) smem = std::max(smem, (size_t)(kThreads / 32) * c.dim * sizeof(double)) + (size_t)slots * vec * 4 * kThreads * sizeof(double);
  a.w_wide = true;
  for (const void *w : {c.q_weight, c.k_weight})
    if ((uintptr_t)w % (vec * wsize > 16 ? 16 : vec * wsize)) a.w_wide = false;
  auto go = [&](auto v, auto n) {
    constexpr int V = decltype(v)::value, N = decltype(n)::value;
    if constexpr (V >= 4)
      if (a.odd > 1 && c.dtype == kF16) return launch<__half, V, N, true>(a, inter, back, few, grid, smem, st);
    if constexpr (V == 4)
      if (a.odd > 1) return launch<float, V, N, true>(a, inter, back, few, grid, smem, st);
    if constexpr (V <= 4)
      if (c.dtype == kF32) return launch<float, V, N, false>(a, inter, back, few, grid, smem, st);
    return launch<__half, V, N, false>(a, inter, back, few, grid, smem, st);
  };
#define SHLO_INT(n) std::integral_constant<int, n>()
  switch (vec) {
    case 8: SHLO_TRY(go(SHLO_INT(8), SHLO_INT(1))); break;
    case 4: SHLO_TRY(slots == 1 ? go(SHLO_INT(4), SHLO_INT(1)) : go(SHLO_INT(4), SHLO_INT(2))); break;
    case 2: SHLO_TRY(slots == 1 ? go(SHLO_INT(2), SHLO_INT(1)) : go(SHLO_INT(2), SHLO_INT(4))); break;
    default: SHLO_TRY(slots == 2 ? go(SHLO_INT(1), SHLO_INT(2)) : go(SHLO_INT(1), SHLO_INT(8))); break;
  }
#undef SHLO_INT
  if (!sums) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((c.dim + 31) / 32, 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  SHLO_CUDA(cudaLaunchKernelEx(&cfg, k_norm_rope_dw, (const double *)a.partials, (int)(grid.x * grid.y), c.dim, c.dq_weight, c.dk_weight));
  return launch_check("norm_rope_grad");
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_norm_rope_noalloc(const shlo_norm_rope_args *args, void *stream) {
  if (!args) return fail("norm_rope: null arguments");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_norm_rope(*args, false, dev->sm_count, (cudaStream_t)stream);
}

int shlo_norm_rope_workspace(size_t *bytes) {
  if (!bytes) return fail("norm_rope_workspace: null pointer");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  *bytes = norm_rope_work_bytes(dev->sm_count);
  return 0;
}

int shlo_norm_rope_grad_noalloc(const shlo_norm_rope_args *args, void *stream) {
  if (!args) return fail("norm_rope_grad: null arguments");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_norm_rope(*args, true, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
