// Beam search's selection: of every sequence's beams, each with a row of logits
// over the vocabulary, the `keep` best continuations by
//   score[beam] + logit - log(sum over the vocabulary of e^logit),
// in descending order, of equal ones the lowest beam first, then the lowest token.
//
// Two kernels. The first gives a block a segment of a row, which it reads once
// into registers: the segment's largest logit, the sum of e^(logit - largest), and
// its `keep` largest logits, in order. The second joins a sequence's segments: a
// row's sum, then its segments' lists merged one continuation at a time.
//
// Two beams' continuations may lie closer together than binary32 tells apart, and
// the order between them is part of the result: the exponentials are a polynomial
// that is right to 2^-25 at each term and unbiased, eight of them are added in
// binary32 and all else in 64 bits. A row's logarithm is then off by 2^-23 at most
// and, where several logits matter, by 10^-8.
//
// Bound: bytes (each logit read once); the first kernel's 10 instructions a logit
// are next.
#include <algorithm>
#include <cmath>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 64, kMaxBeams = 64;
constexpr int kRoom = 256;  // candidates that a segment ranks at once
constexpr int kJoin = 256;  // the second kernel's threads
constexpr int kPicked = 512;  // candidates that it ranks at once

struct BeamArgs {
  const void *z;
  int64_t row;
  const float *scores;
  const int32_t *ended;
  float *next;
  int32_t *parents, *tokens;
  uint64_t *best;  // [rows][segs][keep]: ordered logit above, ~token below; 0: none
  double *sum;     // [rows][segs]
  float *top;      // [rows][segs]: NaN: a value that is not a number, or infinity
  int vocab, beams, keep, segs, seg, end_token;
  int group;  // lanes: 256 / group is at least keep
};

// Floats in the order of unsigned integers (-0 and 0 alike); -infinity's is above 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_ordered(uint32_t u) {
  return __uint_as_float(u ^ ((int32_t)u < 0 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kNegInf = 0x007fffffu;  // ordered(-infinity)

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// e^d for -87 <= d <= 0: d = i ln 2 + r (ln 2 in two parts, the first of 15 bits, so
// that its products are exact), e^r = 1 + r + r^2 g(r), g of degree 4 fitted to the
// smallest largest relative error (2^-28, 3 10^-10 on average).
__device__ __forceinline__ float2 exp_below(float2 d) {
  const float2 m = __ffma2_rn(d, both(0x1.715476p+0f), both(12582912.0f));
  const float2 i = __fadd2_rn(m, both(-12582912.0f));
  float2 r = __ffma2_rn(i, both(-0x1.62e4p-1f), d);
  r = __ffma2_rn(i, both(-0x1.7f7d1cp-20f), r);
  float2 g = both(0x1.6a23d0p-10f);
  g = __ffma2_rn(g, r, both(0x1.123a20p-7f));
  g = __ffma2_rn(g, r, both(0x1.5558f2p-5f));
  g = __ffma2_rn(g, r, both(0x1.555492p-3f));
  g = __ffma2_rn(g, r, both(0x1.fffffcp-2f));
  g = __ffma2_rn(g, r, both(1.0f));
  g = __ffma2_rn(g, r, both(1.0f));
  g.x = __uint_as_float(__float_as_uint(g.x) + (__float_as_uint(m.x) << 23));
  g.y = __uint_as_float(__float_as_uint(g.y) + (__float_as_uint(m.y) << 23));
  return g;
}

// What a type's vectors of 16 bytes need: the largest of their values (NaN where
// one is), their values less the largest of all, the values themselves.
template <typename T> struct Vec;
template <> struct Vec<__half> {
  static constexpr int W = 8;
  static __device__ __forceinline__ float top(const uint4 &v) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  // (what is more than 80 below adds 10^-35: it is kept there, for e^d's range)
  static __device__ __forceinline__ float2 below(const uint4 &v, int pair, float top) {
    const __half2 h = reinterpret_cast<const __half2 *>(&v)[pair];
    float2 d;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d.x) : "h"(__half_as_ushort(__low2half(h))), "f"(-top));
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d.y) : "h"(__half_as_ushort(__high2half(h))), "f"(-top));
    return make_float2(fmaxf(d.x, -80.0f), fmaxf(d.y, -80.0f));
  }
  static __device__ __forceinline__ float value(const uint4 &v, int i) { return __half2float(reinterpret_cast<const __half *>(&v)[i]); }
  static __device__ __half neg_inf() { return __ushort_as_half(0xfc00); }
};
template <> struct Vec<float> {
  static constexpr int W = 4;
  static __device__ __forceinline__ float top(const uint4 &v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ float2 below(const uint4 &v, int pair, float top) {
    const float *f = reinterpret_cast<const float *>(&v) + 2 * pair;
    const float2 d = __fadd2_rn(make_float2(f[0], f[1]), both(-top));
    return make_float2(fmaxf(d.x, -80.0f), fmaxf(d.y, -80.0f));
  }
  static __device__ __forceinline__ float value(const uint4 &v, int i) { return reinterpret_cast<const float *>(&v)[i]; }
  static __device__ float neg_inf() { return -INFINITY; }
};

// (four blocks on an SM: the waits for the logits and between the warps of one
// are the others' work)
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads, 4) k_beam_segments(const BeamArgs a) {
  using V = Vec<T>;
  constexpr int W = V::W;  // values a vector
  __shared__ float tops[kWarps], lows[kWarps];
  __shared__ double sums[kWarps];
  __shared__ uint64_t found[kRoom];
  __shared__ int count;
  const int row = blockIdx.y, s = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (a.ended && a.ended[row]) return;  // it goes on with one token, whatever its logits
  const T *const z = static_cast<const T *>(a.z) + row * a.row;
  const int lo = s * a.seg;
  // Vector i of this thread. Which logits it has does not depend on where the row
  // lies, so that equal rows have equal sums; where it begins between two 16-byte
  // boundaries it is cut from two of memory's vectors.
  const int past = (int)((uintptr_t)z & 15);
  auto load = [&](int i) -> uint4 {
    const int at = lo + (i * kThreads + threadIdx.x) * W, off = past / (int)sizeof(T);
    if (past == 0 && at + W <= a.vocab) return __ldg(reinterpret_cast<const uint4 *>(z + at));
    if (past && at >= off && at - off + 2 * W <= a.vocab) {
      const uint4 p = __ldg(reinterpret_cast<const uint4 *>(z + (at - off))), q = __ldg(reinterpret_cast<const uint4 *>(z + (at - off) + W));
      const int sh = past % 4 * 8;
      auto cut = [&](uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t c4) {
        return make_uint4(__funnelshift_r(c0, c1, sh), __funnelshift_r(c1, c2, sh), __funnelshift_r(c2, c3, sh), __funnelshift_r(c3, c4, sh));
      };
      switch (past / 4) {
        case 0: return cut(p.x, p.y, p.z, p.w, q.x);
        case 1: return cut(p.y, p.z, p.w, q.x, q.y);
        case 2: return cut(p.z, p.w, q.x, q.y, q.z);
        default: return cut(p.w, q.x, q.y, q.z, q.w);
      }
    }
    T e[W];
#pragma unroll
    for (int j = 0; j < W; j++) e[j] = at + j < a.vocab ? z[at + j] : V::neg_inf();
    uint4 r;
    memcpy(&r, e, 16);
    return r;
  };
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) v[i] = load(i);
  if (threadIdx.x == 0) count = 0;
  auto token = [&](int i, int j) { return lo + (i * kThreads + (int)threadIdx.x) * W + j; };

  // The largest logit, and the smallest of the largest of `group` lanes each: as many
  // groups as are kept, so that at least so many threads' largest reach it.
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; i++) mine = max_nan(mine, V::top(v[i]));
  float top = mine, low = mine;
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    top = max_nan(top, __shfl_xor_sync(~0u, top, i));
    const float o = __shfl_xor_sync(~0u, low, i);
    low = i < a.group ? fmaxf(low, o) : fminf(low, o);
  }
  if (lane == 0) tops[warp] = top, lows[warp] = low;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; i++) {
    top = max_nan(top, tops[i]);
    low = fminf(low, lows[i]);
  }
  const int64_t place = (int64_t)row * a.segs + s;
  uint64_t *const best = a.best + place * a.keep;
  if (!(top < INFINITY) || top == -INFINITY) {  // nothing to choose from
    if (threadIdx.x == 0) {
      a.top[place] = top == -INFINITY ? top : __uint_as_float(0x7fc00000u);
      a.sum[place] = 0.0;
    }
    for (int i = threadIdx.x; i < a.keep; i += kThreads) best[i] = 0;
    return;
  }

  // A border that at least `keep` threads' largest logits reach, and few more: found
  // by halving between two borders. (Where fewer threads than `keep` have any logit
  // above -infinity, all of them are candidates, or the exact border below is found.)
  uint32_t under = low > -INFINITY ? ordered(low) : kNegInf + 1, over = ordered(top) + 1;
  const uint32_t key = ordered(mine);
  int have = __syncthreads_count(key >= under);
  if (have >= a.keep)
    while (have > 2 * a.keep && over - under > 1) {
      const uint32_t mid = under + (over - under) / 2;
      const int n = __syncthreads_count(key >= mid);
      if (n >= a.keep) under = mid, have = n;
      else over = mid;
    }

  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float2 e[W / 2];
#pragma unroll
    for (int j = 0; j < W / 2; j++) e[j] = exp_below(V::below(v[i], j, top));
#pragma unroll
    for (int j = W / 4; j; j /= 2)
#pragma unroll
      for (int l = 0; l < j; l++) e[l] = __fadd2_rn(e[l], e[l + j]);
    sum += (double)(e[0].x + e[0].y);
  }
#pragma unroll
  for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
  if (lane == 0) sums[warp] = sum;
  if (key >= under) {
    const float border = of_ordered(under);
    unsigned which = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) which |= (V::top(v[i]) >= border) << i;
    for (; which; which &= which - 1) {  // (read again, from L2: few threads have any)
      const int i = __ffs(which) - 1;
      const uint4 w = load(i);
#pragma unroll
      for (int j = 0; j < W; j++)
        if (V::value(w, j) >= border) {
          const int n = atomicAdd(&count, 1);
          if (n < kRoom) found[n] = (uint64_t)ordered(V::value(w, j)) << 32 | (uint32_t)~token(i, j);
        }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) all += sums[i];
    a.sum[place] = all;
    a.top[place] = top;
  }
  int n = count;
  if (n > kRoom) {
    // More of them than there is room for (many equal ones, or few threads that
    // hold most): the exact border, and which of those that equal it.
    auto counted = [&](uint32_t t, uint32_t last) {  // logits above t, and those at t whose ~token is at least last
      int c = 0;
#pragma unroll 1
      for (int i = 0; i < NV; i++) {
        const uint4 w = load(i);
#pragma unroll
        for (int j = 0; j < W; j++) {
          const uint32_t u = ordered(V::value(w, j));
          if (u > t || (u == t && (uint32_t)~token(i, j) >= last)) c++;
        }
      }
      c = __reduce_add_sync(~0u, c);
      __syncthreads();
      if (lane == 0) tops[warp] = __int_as_float(c);
      __syncthreads();
      c = 0;
#pragma unroll
      for (int i = 0; i < kWarps; i++) c += __float_as_int(tops[i]);
      return c;
    };
    uint32_t t0 = under, t1 = ordered(top) + 1;  // enough reach t0; t1 is above all
    while (t1 - t0 > 1) {
      const uint32_t mid = t0 + (t1 - t0) / 2;
      if (counted(mid, 0) >= a.keep) t0 = mid;
      else t1 = mid;
    }
    uint32_t l0 = 0, l1 = 0xffffffffu;  // enough at or above l0
    while (l1 - l0 > 1) {
      const uint32_t mid = l0 + (l1 - l0) / 2;
      if (counted(t0, mid) >= a.keep) l0 = mid;
      else l1 = mid;
    }
    __syncthreads();
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < NV; i++) {
      const uint4 w = load(i);
#pragma unroll
      for (int j = 0; j < W; j++) {
        const uint32_t u = ordered(V::value(w, j)), last = ~token(i, j);
        if (u > t0 || (u == t0 && last >= l0)) found[atomicAdd(&count, 1)] = (uint64_t)u << 32 | last;
      }
    }
    __syncthreads();
    n = count;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t k = found[i];
    int above = 0;
    for (int j = 0; j < n; j++) above += found[j] > k;
    if (above < a.keep) best[above] = k;
  }
  for (int i = n + threadIdx.x; i < a.keep; i += kThreads) best[i] = 0;
}

// A sequence a block. A list is a segment's of one beam, in descending order; a
// thread has lists threadIdx.x, + kJoin, ... Of the threads' best heads the
// keep-th best is a border: what reaches it is a handful of each list's entries,
// which are ranked against each other. Where they are too many (or too few lists
// have a head), the best of all heads is taken `keep` times instead.
__global__ void __launch_bounds__(kJoin) k_beam_join(const BeamArgs a) {
  extern __shared__ unsigned char at_list[];  // of a list: how many of its entries are taken
  // Of a beam: its score less the logarithm of its row's sum (NaN: none to choose
  // from), and its row's largest logit, from which the others are counted: they may
  // be far from 0.
  __shared__ double base[kMaxBeams];
  __shared__ float top_of[kMaxBeams];
  __shared__ bool ended[kMaxBeams];
  __shared__ double total_of[kPicked];
  __shared__ uint64_t key_of[kPicked];
  __shared__ int list_of[kPicked];
  __shared__ int picked;
  __shared__ double border;
  const int seq = blockIdx.x, lists = a.beams * a.segs, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const double none = -INFINITY;
  cudaGridDependencySynchronize();  // (it may begin before the segments are done)
  for (int b = warp; b < a.beams; b += kJoin / 32) {
    const int64_t row = (int64_t)seq * a.beams + b;
    const double score = (double)a.scores[row];
    const bool end = a.ended && a.ended[row];
    float top = -INFINITY;
    double sum = 0.0;
    if (!end) {
      for (int s = lane; s < a.segs; s += 32) top = max_nan(top, a.top[row * a.segs + s]);
      for (int i = 16; i; i /= 2) top = max_nan(top, __shfl_xor_sync(~0u, top, i));
      if (top > -INFINITY)
        for (int s = lane; s < a.segs; s += 32) {
          const float t = a.top[row * a.segs + s];
          if (t > -INFINITY) sum += a.sum[row * a.segs + s] * exp((double)t - (double)top);
        }
      for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
    }
    if (lane == 0) {
      base[b] = end ? score : top > -INFINITY ? score - log(sum) : __longlong_as_double(0x7ff8000000000000ll);
      top_of[b] = top;
      ended[b] = end;
    }
  }
  for (int i = threadIdx.x; i < lists; i += kJoin) at_list[i] = 0;
  if (threadIdx.x == 0) picked = 0, border = none;
  __syncthreads();
  // Entry `at` of list l: its key, 0 behind the last, and its total.
  auto entry = [&](int l, int at, double &t) -> uint64_t {
    const int b = l / a.segs, s = l - b * a.segs;
    t = base[b];
    if (ended[b]) return s == 0 && at == 0 && t > none ? ~0ull : 0;
    if (at >= a.keep || !(t > none)) return 0;
    const uint64_t k = a.best[(((int64_t)seq * a.beams + b) * a.segs + s) * a.keep + at];
    t += (double)of_ordered((uint32_t)(k >> 32)) - (double)top_of[b];
    return t > none ? k : 0;
  };
  // Whether the second goes before the first; a list below 0: none.
  auto better = [&](double t, uint64_t k, int l, double t2, uint64_t k2, int l2) {
    if (l2 < 0) return false;
    if (l < 0) return true;
    if (t != t2) return t2 > t;
    const int b = l / a.segs, b2 = l2 / a.segs;
    return b != b2 ? b2 < b : k2 > k;
  };
  auto write = [&](int i, double t, uint64_t k, int l) {
    const int64_t to = (int64_t)seq * a.keep + i;
    a.next[to] = l < 0 ? -INFINITY : (float)t;
    a.parents[to] = l < 0 ? -1 : seq * a.beams + l / a.segs;
    a.tokens[to] = l < 0 ? -1 : k == ~0ull ? a.end_token : (int32_t)~(uint32_t)k;
  };
  // The best of this thread's heads.
  double total;
  uint64_t key;
  int list;
  auto offer = [&]() {
    list = -1;
    total = none;
    key = 0;
    for (int l = threadIdx.x; l < lists; l += kJoin) {
      double t;
      const uint64_t k = entry(l, at_list[l], t);
      if (k && better(total, key, list, t, k, l)) total = t, key = k, list = l;
    }
  };
  offer();

  total_of[threadIdx.x] = total;
  __syncthreads();
  int above = 0;
  for (int i = 0; i < kJoin; i++) above += total_of[i] > total || (total_of[i] == total && i < (int)threadIdx.x);
  if (above == a.keep - 1) border = total;  // (-infinity where fewer threads have a head)
  __syncthreads();
  const double least = border;
  if (list >= 0)
    for (int l = threadIdx.x; l < lists; l += kJoin)
      for (int at = 0;; at += 4) {
        double t[4];
        uint64_t k[4];
#pragma unroll
        for (int j = 0; j < 4; j++) k[j] = entry(l, at + j, t[j]);
        bool on = true;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          on = on && k[j] && t[j] >= least;
          if (on) {
            const int n = atomicAdd(&picked, 1);
            if (n < kPicked) total_of[n] = t[j], key_of[n] = k[j], list_of[n] = l;
            else on = false;
          }
        }
        if (!on) break;
      }
  __syncthreads();
  const int n = picked;
  if (n <= kPicked) {
    for (int i = threadIdx.x; i < n; i += kJoin) {
      const double t = total_of[i];
      const uint64_t k = key_of[i];
      const int l = list_of[i];
      int before = 0;
      for (int j = 0; j < n; j++) {
        const double t2 = total_of[j];
        if (t2 >= t) before += j != i && better(t, k, l, t2, key_of[j], list_of[j]);
      }
      if (before < a.keep) write(before, t, k, l);
    }
    for (int i = n + threadIdx.x; i < a.keep; i += kJoin) write(i, none, 0, -1);
    return;
  }

  for (int i = 0; i < a.keep; i++) {
    double t = total;
    uint64_t k = key;
    int l = list;
    for (int j = 16; j; j /= 2) {
      const double t2 = __shfl_xor_sync(~0u, t, j);
      const uint64_t k2 = __shfl_xor_sync(~0u, k, j);
      const int l2 = __shfl_xor_sync(~0u, l, j);
      if (better(t, k, l, t2, k2, l2)) t = t2, k = k2, l = l2;
    }
    __syncthreads();
    if (lane == 0) total_of[warp] = t, key_of[warp] = k, list_of[warp] = l;
    __syncthreads();
    for (int j = 0; j < kJoin / 32; j++)
      if (better(t, k, l, total_of[j], key_of[j], list_of[j])) t = total_of[j], k = key_of[j], l = list_of[j];
    if (threadIdx.x == 0) write(i, t, k, l);
    if (l >= 0 && l % kJoin == (int)threadIdx.x) {
      at_list[l]++;
      offer();
    }
  }
}

// The segments of a row: a block's registers hold `nv` vectors a thread, fewer where
// the segments would leave SMs without work.
int segments(int vocab, size_t size, int nv) {
  const int seg = nv * kThreads * (16 / (int)size);
  return (vocab + seg - 1) / seg;
}
int vectors(int64_t rows, int vocab, size_t size, int sms) {
  int nv = size == 2 ? 4 : 8;
  while (nv > 1 && rows * segments(vocab, size, nv) < 2 * sms) nv /= 2;
  return nv;
}

}  // namespace

// The room for both types: float32's segments are the shorter ones.
size_t beam_work_bytes(int64_t rows, int32_t keep, int32_t vocab) {
  const int64_t segs = segments(vocab, 4, 1);
  return (size_t)(rows * segs * (8 * (int64_t)keep + 12) + 16);
}

int launch_beam_select(const BeamCall &c, int sms, cudaStream_t st) {
  if (c.dtype != kF16 && c.dtype != kF32) return fail("beam_select: %s not carried (float16 or float32)", dtype_name(c.dtype));
  if (c.seqs < 0 || c.beams < 1 || c.beams > kMaxBeams || c.keep < 1 || c.keep > kMaxKeep)
    return fail("beam_select: %d sequences of %d beams (1 to %d), %d kept (1 to %d)", c.seqs, c.beams, kMaxBeams, c.keep, kMaxKeep);
  if (c.vocab < 1 || c.vocab > (1 << 20)) return fail("beam_select: a vocabulary of %d (1 to 2^20)", c.vocab);
  const int64_t rows = (int64_t)c.seqs * c.beams;
  if (rows > 65535) return fail("beam_select: %lld rows of logits (at most 65535)", (long long)rows);
  if (c.seqs == 0) return 0;
  if (!c.logits || !c.scores || !c.next || !c.parents || !c.tokens) return fail("beam_select: null pointer");
  const size_t size = dtype_size(c.dtype);
  if ((uintptr_t)c.logits % size || ((uintptr_t)c.scores | (uintptr_t)c.ended | (uintptr_t)c.next | (uintptr_t)c.parents | (uintptr_t)c.tokens) % 4)
    return fail("beam_select: an operand is not aligned to its type");
  const size_t need = beam_work_bytes(rows, c.keep, c.vocab);
  if (!c.work || c.work_bytes < need) return fail("beam_select: a workspace of %zu bytes, %zu needed", c.work ? c.work_bytes : 0, need);
  if ((uintptr_t)c.work % 8) return fail("beam_select: misaligned workspace");
  const int nv = vectors(rows, c.vocab, size, sms);
  BeamArgs a;
  a.z = c.logits; a.row = c.row; a.scores = c.scores; a.ended = c.ended; a.next = c.next; a.parents = c.parents; a.tokens = c.tokens;
  a.vocab = c.vocab; a.beams = c.beams; a.keep = c.keep; a.end_token = c.end_token;
  a.group = 32;
  while (a.group > 1 && kThreads / a.group < c.keep) a.group /= 2;
  a.seg = nv * kThreads * (16 / (int)size);
  a.segs = segments(c.vocab, size, nv);
  a.best = (uint64_t *)c.work;
  a.sum = (double *)(a.best + rows * a.segs * c.keep);
  a.top = (float *)(a.sum + rows * a.segs);
  const dim3 grid((unsigned)a.segs, (unsigned)rows);
  if (c.dtype == kF16) {
    if (nv == 4) k_beam_segments<__half, 4><<<grid, kThreads, 0, st>>>(a);
    else if (nv == 2) k_beam_segments<__half, 2><<<grid, kThreads, 0, st>>>(a);
    else k_beam_segments<__half, 1><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (nv == 8) k_beam_segments<float, 8><<<grid, kThreads, 0, st>>>(a);
    else if (nv == 4) k_beam_segments<float, 4><<<grid, kThreads, 0, st>>>(a);
    else if (nv == 2) k_beam_segments<float, 2><<<grid, kThreads, 0, st>>>(a);
    else k_beam_segments<float, 1><<<grid, kThreads, 0, st>>>(a);
  }
  SHLO_TRY(launch_check("beam_select"));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c.seqs);
  cfg.blockDim = dim3(kJoin);
  cfg.dynamicSmemBytes = (size_t)c.beams * a.segs;
  cfg.stream = st;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  SHLO_CUDA(cudaLaunchKernelEx(&cfg, k_beam_join, a));
  return launch_check("beam_select");
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_beam_workspace(int32_t seqs, int32_t beams, int32_t keep, int32_t vocab, size_t *bytes) {
  if (!bytes) return fail("beam_workspace: null pointer");
  if (seqs < 0 || beams < 1 || beams > kMaxBeams || keep < 1 || keep > kMaxKeep || vocab < 1 || vocab > (1 << 20) || (int64_t)seqs * beams > 65535)
    return fail("beam_workspace: %d sequences of %d beams, %d kept, a vocabulary of %d", seqs, beams, keep, vocab);
  *bytes = beam_work_bytes((int64_t)seqs * beams, keep, vocab);
  return 0;
}

int shlo_beam_select_noalloc(const void *logits, int64_t row, const float *scores, const int32_t *ended, int32_t end_token,
                             int32_t seqs, int32_t beams, int32_t keep, int32_t vocab, uint8_t dtype, float *next,
                             int32_t *parents, int32_t *tokens, void *workspace, size_t workspace_bytes, void *stream) {
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  BeamCall c{logits, row, scores, ended, end_token, seqs, beams, keep, vocab, dtype, next, parents, tokens, workspace, workspace_bytes};
  return launch_beam_select(c, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
