// Beam search's selection: of every sequence's beams, each with a row of logits
// over the vocabulary, the `keep` best continuations by
//   score[beam] + logit - log(sum over the vocabulary of e^logit),
// in descending order, of equal ones the lowest beam first, then the lowest token.
//
// Two kernels. The first gives a block a part of a row, which it reads once, a stretch
// of registers at a time: each thread's sum of e^(logit - largest), the largest of the
// first stretch or of what the thread has seen since, and the part's `keep` largest
// logits, of which the first stretch gives a border that few of the later ones pass. The
// second joins a sequence's parts: a row's sum, then its parts' lists.
//
// Two beams' continuations may lie closer together than binary32 tells apart, and
// the order between them is part of the result. A term of the sum is ex2.approx's, off
// by 2.1 10^-7 of it at most where it lies up to 2 above or below what is counted from
// (farther down by more, but of less), eight of them are added in binary32 and the rest
// in 64 bits; the terms of the candidates, which are most of a peaked row's sum, are
// replaced by a polynomial's, off by 7 10^-8. What is left is that share of the light
// terms, which averages out where they are many and not equal. (A thread counts from a
// logit of its own where that is more than 2 above the first stretch's largest: a plateau
// 57 above that would move the logarithm by 3 10^-6. Of 512 rows of 128256 normal logits,
// us: from the first stretch's alone 47.3, from beyond 2 above it 47.9, from any above it
// 49.4.)
//
// Bound: bytes (each logit read once); what keeps the first kernel from their rate are its
// ten instructions a logit and their waits: issue slots 57 % used, DRAM 38 %, 14 warps on
// an SM on average. Measured on one B200: 64 sequences of 8 beams over 128256 float16
// logits (125 MB) 47 us, 37 of them the first kernel, at 512 blocks on 592 places; 5 of 32
// over 50257 float32 logits, 64 kept 28 us; one of 4 over 32001 10 us. Measured and left: the
// polynomial for every term (64 us on the first case: the heavy half of the FMA pipe), a
// part of one stretch each (73 us: every one searches for its border), borders by
// halving over lists in memory (67 us for the second case's join alone).
#include <algorithm>
#include <climits>
#include <cmath>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 64, kMaxBeams = 64;
constexpr int kRoom = 512;  // candidates of a part at a time
constexpr int kGroup = 4;   // stretches whose candidates are looked at together: 1, 1, 2, 4, 4, ...
constexpr int kJoin = 256;  // the second kernel's threads
constexpr int kPicked = 512;  // candidates that it ranks
constexpr int kScan = 2048;   // entries of a sequence's lists that are all looked at
constexpr int kSteps = 7;     // entries 2^j - 1 < kMaxKeep of a list
static_assert(1 << (kSteps - 1) <= kMaxKeep, "entries of a list");

struct BeamArgs {
  const void *z;
  int64_t row;
  const float *scores;
  const int32_t *ended;
  float *next;
  int32_t *parents, *tokens;
  uint64_t *best;  // [rows][parts][keep]: entries; 0: none
  double *sum;     // [rows][parts]
  float *top;      // [rows][parts]: what the sum counts from; NaN: a value that is not a number, or infinity
  int vocab, beams, keep, parts, part, end_token;  // part: logits a part
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
constexpr uint32_t kInf = 0xff800000u;     // ordered(infinity): above it is NaN alone

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits(__half x) { return __half_as_ushort(x); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// e^d for -87 <= d <= 87: d = i ln 2 + r (ln 2 rounded: 2.7 10^-9 of d), e^r = 1 + r +
// r^2 g(r), g of degree 4 fitted to the smallest largest relative error (2^-28,
// 3 10^-10 on average). With its roundings, over all d: 3 10^-8 up to |d| = 0.06, 6.8
// 10^-8 up to 2, 1.1 10^-7 up to 16, 2.8 10^-7 up to 80.
__device__ __forceinline__ float2 exp_near(float2 d) {
  const float2 m = __ffma2_rn(d, both(0x1.715476p+0f), both(12582912.0f));
  const float2 i = __fadd2_rn(m, both(-12582912.0f));
  const float2 r = __ffma2_rn(i, both(-0x1.62e430p-1f), d);
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

// The same for d <= kRise, 1 for 0 and 0 for -infinity: 2^(d log2(e)), the product in two
// parts. What its roundings lose grows with d: over all d 1.8 10^-7 up to |d| = 1, 2.1
// 10^-7 up to 2, 2.7 10^-7 up to 4, 4.9 10^-7 up to 8, 9.3 10^-7 up to 16. (A factor for what
// is lost would hold it at 2 10^-7, and costs 2 us of 47 for 512 rows of 128256.)
__device__ __forceinline__ float2 exp_fast(float2 d) {
  const float2 t = __ffma2_rn(d, both(0x1.4ae0c0p-26f), __fmul2_rn(d, both(0x1.715476p+0f)));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  return e;
}
constexpr float kRise = 2.0f;

// What a candidate's term is more by the polynomial than by the other.
__device__ __forceinline__ double replaced(float d) {
  const float2 near = make_float2(fmaxf(d, -80.0f), 0.0f);
  return (double)exp_near(near).x - (double)exp_fast(near).x;
}

// A sum counted from `from`, counted from `to` above it. (This and the next are rare:
// their code is not the loop's, whose registers it would take.)
__device__ __noinline__ double recounted(double sum, float from, float to) {
  return from > -INFINITY ? sum * exp((double)from - (double)to) : 0.0;
}
__device__ __noinline__ double replaced_apart(float d) { return d < 0.0f ? replaced(d) : 0.0; }

// A candidate: in the order of the logits, of equal ones the lowest token first; the
// lowest bit is no part of the order (tokens are below 2^20), and says that its term is
// the polynomial's already. 0 is below all.
__device__ __forceinline__ uint64_t entry_of(float logit, int token, bool done) {
  return (uint64_t)ordered(logit) << 32 | (uint32_t)~token << 1 | (uint32_t)done;
}
__device__ __forceinline__ int token_of(uint64_t e) { return (int)(~(uint32_t)e >> 1); }

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
  static __device__ __forceinline__ float2 below(const uint4 &v, int pair, float top) {
    const __half2 h = reinterpret_cast<const __half2 *>(&v)[pair];
    float2 d;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d.x) : "h"(__half_as_ushort(__low2half(h))), "f"(-top));
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d.y) : "h"(__half_as_ushort(__high2half(h))), "f"(-top));
    return d;
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
    return __fadd2_rn(make_float2(f[0], f[1]), both(-top));
  }
  static __device__ __forceinline__ float value(const uint4 &v, int i) { return reinterpret_cast<const float *>(&v)[i]; }
  static __device__ float neg_inf() { return -INFINITY; }
};

// (four blocks on an SM: the waits for the logits and between the warps of one
// are the others' work)
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads, 4) k_beam_parts(const BeamArgs a) {
  using V = Vec<T>;
  constexpr int W = V::W;                    // values a vector
  constexpr int STRETCH = NV * kThreads * W;
  __shared__ float tops[kWarps], lows[kWarps];
  __shared__ double sums[kWarps];
  __shared__ uint64_t found[kRoom];
  __shared__ int count;
  __shared__ uint32_t least_shared;
  __shared__ float first_top;
  const int row = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (a.ended && a.ended[row]) return;  // it goes on with one token, whatever its logits
  const T *const z = static_cast<const T *>(a.z) + row * a.row;
  const int begin = blockIdx.x * a.part, end = min(begin + a.part, a.vocab);
  // Vector i of this thread in the stretch from lo on. Which logits it has does not
  // depend on where the row lies, so that equal rows have equal sums; where it begins
  // between two 16-byte boundaries it is cut from two of memory's vectors.
  const int past = (int)((uintptr_t)z & 15);
  auto load = [&](int lo, int i) -> uint4 {
    const int at = lo + (i * kThreads + threadIdx.x) * W, off = past / (int)sizeof(T);
    if (past == 0 && at + W <= a.vocab) return __ldg(reinterpret_cast<const uint4 *>(z + at));
    if (sizeof(T) == 4 && at + W <= a.vocab) return make_uint4(bits(z[at]), bits(z[at + 1]), bits(z[at + 2]), bits(z[at + 3]));
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
  auto token = [&](int lo, int i, int j) { return lo + (i * kThreads + (int)threadIdx.x) * W + j; };

  // (every logit -infinity where `from` is)
  auto exps = [&](const uint4 (&v)[NV], float from) {
    const float zero = from > -INFINITY ? from : 0.0f;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float2 e[W / 2];
#pragma unroll
      for (int j = 0; j < W / 2; j++) e[j] = exp_fast(V::below(v[i], j, zero));
#pragma unroll
      for (int j = W / 4; j; j /= 2)
#pragma unroll
        for (int l = 0; l < j; l++) e[l] = __fadd2_rn(e[l], e[l + j]);
      sum += (double)(e[0].x + e[0].y);
    }
    return sum;
  };
  // Candidates threadIdx.x / per (and, above kThreads of them, threadIdx.x + kThreads),
  // and how many are above them (none of a thread's: kRoom); `per` lanes count for one.
  auto rank = [&](int n, uint64_t (&k)[2]) {
    const int per = n <= kThreads / 4 ? 4 : n <= kThreads / 2 ? 2 : 1, at = (int)threadIdx.x / per, off = (int)threadIdx.x % per;
    int2 above = make_int2(0, 0);
    k[0] = at < n ? found[at] : 0;
    k[1] = at + kThreads < n ? found[at + kThreads] : 0;
    if (n <= kThreads) {
#pragma unroll 8
      for (int j = off; j < n; j += per) above.x += found[j] > k[0];
    } else {
#pragma unroll 8
      for (int j = 0; j < n; j++) {
        const uint64_t o = found[j];
        above.x += o > k[0];
        above.y += o > k[1];
      }
    }
    for (int i = 1; i < per; i *= 2) above.x += __shfl_xor_sync(~0u, above.x, i);
    if (at >= n || off) above.x = kRoom;
    if (at + kThreads >= n || per > 1) above.y = kRoom;
    return above;
  };
  // The next stretch is on its way to shared memory while one is worked on; a thread
  // reads there what it asked for itself.
  __shared__ uint4 ahead[NV * kThreads];
  int asked = -1;
  double sum = 0.0;        // the sum of e^(logit - from) over this thread's logits,
  float from = -INFINITY;  // the first stretch's largest, or one of the thread's own more than kRise above it
  bool odd = false;        // whether one is not a number, or infinity
  int risen = INT_MAX;     // the stretch that has the first such of its own
  uint32_t least = 0;     // candidates are the logits that reach this, in order
  int n = 0;              // candidates so far
  if (threadIdx.x == 0) count = 0;
  for (int lo = begin; lo < end;) {
    const bool first = lo == begin;
    const int group = lo, group_end = min(end, lo + (first ? 1 : min((lo - begin) / STRETCH, kGroup)) * STRETCH);
    bool some = false;
    for (; lo < group_end; lo += STRETCH) {
      uint4 v[NV];
      if (lo == asked) {
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = ahead[i * kThreads + threadIdx.x];
      } else {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = load(lo, i);
      }
      if (past == 0 && lo + STRETCH < end && lo + 2 * STRETCH <= a.vocab) {
        asked = lo + STRETCH;
        const uint4 *const p = reinterpret_cast<const uint4 *>(z + asked) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < NV; i++)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(ahead + i * kThreads + threadIdx.x)), "l"(p + i * kThreads) : "memory");
      }
      float tops_of[NV], mine = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        tops_of[i] = V::top(v[i]);
        mine = max_nan(mine, tops_of[i]);
      }
      odd = odd || !(mine < INFINITY);
      const uint32_t key = ordered(mine);
      if (first) {
        // A border that at least `keep` threads' largest logits reach, and few more: from
        // the smallest of the largest of `group` lanes each, as many groups as are kept,
        // by halving between two borders. (Where fewer threads have any logit above
        // -infinity, all of those are candidates.)
        float top = mine, low = mine;
#pragma unroll
        for (int i = 1; i < 32; i *= 2) {
          top = fmaxf(top, __shfl_xor_sync(~0u, top, i));
          const float o = __shfl_xor_sync(~0u, low, i);
          low = i < a.group ? fmaxf(low, o) : fminf(low, o);
        }
        if (lane == 0) tops[warp] = top, lows[warp] = low;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWarps; i++) {
          top = fmaxf(top, tops[i]);
          low = fminf(low, lows[i]);
        }
        from = top;
        if (threadIdx.x == 0) first_top = top;
        uint32_t over = ordered(top) + 1;
        least = low > -INFINITY ? ordered(low) : kNegInf + 1;
        int have = __syncthreads_count(key >= least);
        if (have >= a.keep)
          for (int i = 0; i < 16 && have > a.keep + 8 && over - least > 1 && over > least; i++) {
            const uint32_t mid = least + (over - least) / 2;
            const int m = __syncthreads_count(key >= mid);
            if (m >= a.keep) least = mid, have = m;
            else over = mid;
          }
      }

      if (mine > from + kRise) {
        sum = recounted(sum, from, mine);
        from = mine;
        risen = min(risen, lo);
      }
      sum += exps(v, from);

      if (key >= least) {
        some = true;
        const float border = of_ordered(least);
        unsigned which = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) which |= (tops_of[i] >= border) << i;
        for (; which; which &= which - 1) {
          const int i = __ffs(which) - 1;
          uint4 w = v[0];
#pragma unroll
          for (int j = 1; j < NV; j++)
            if (i == j) w = v[j];
#pragma unroll
          for (int j = 0; j < W; j++)
            if (V::value(w, j) >= border) {
              const int k = atomicAdd(&count, 1);
              if (k < kRoom) found[k] = entry_of(V::value(w, j), token(lo, i, j), risen <= lo);
              if (risen <= lo) sum += replaced_apart(V::value(w, j) - from);
            }
        }
      }
    }
    if (!__syncthreads_or(some)) continue;
    const int before = n;
    n = count;
    __syncthreads();
    if (n > kRoom) {
      // More of them than there is room for (many equal ones, or rows that rise): the
      // exact border of these stretches, and which of the logits that equal it. (What is
      // not a number was no candidate and is none here: all of them would have no room.)
      auto counted = [&](uint32_t t, uint32_t last) {  // logits above t, and those at t whose ~token is at least last
        int c = 0;
        for (int at = group; at < group_end; at += STRETCH)
#pragma unroll 1
          for (int i = 0; i < NV; i++) {
            const uint4 w = load(at, i);
#pragma unroll
            for (int j = 0; j < W; j++) {
              const uint32_t u = ordered(V::value(w, j));
              if ((u > t && u <= kInf) || (u == t && (uint32_t)~token(at, i, j) >= last)) c++;
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
      uint32_t t0 = least, t1 = kInf + 1;  // enough reach t0; t1 is above all numbers
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
      if (threadIdx.x == 0) count = before;
      __syncthreads();
      for (int at = group; at < group_end; at += STRETCH)
#pragma unroll 1
        for (int i = 0; i < NV; i++) {
          const uint4 w = load(at, i);
#pragma unroll
          for (int j = 0; j < W; j++) {
            const uint32_t u = ordered(V::value(w, j)), last = ~token(at, i, j);
            if ((u > t0 && u <= kInf) || (u == t0 && last >= l0)) {
              const int k = atomicAdd(&count, 1);
              if (k < kRoom) found[k] = entry_of(V::value(w, j), token(at, i, j), risen <= at);
            }
          }
        }
      __syncthreads();
      n = min(count, kRoom);
      __syncthreads();
    }
    // The best of them, in order; later stretches' candidates are above the last (of
    // equal ones the earlier is better).
    if (n >= a.keep) {
      uint64_t k[2];
      const int2 above = rank(n, k);
      __syncthreads();
      if (above.x < a.keep) found[above.x] = k[0];
      if (above.y < a.keep) found[above.y] = k[1];
      if (above.x == a.keep - 1) least_shared = (uint32_t)(k[0] >> 32) + 1, count = a.keep;
      if (above.y == a.keep - 1) least_shared = (uint32_t)(k[1] >> 32) + 1, count = a.keep;
      __syncthreads();
      least = least_shared;
      n = a.keep;
    }
  }

  if (n < a.keep) {  // (else in order already; the order is the sum's below too, and not that of the atomics)
    uint64_t k[2];
    const int above = rank(n, k).x;  // (fewer than keep: one a thread)
    __syncthreads();
    if (above < n) found[above] = k[0];
    __syncthreads();
  }
  // The candidates' terms by the polynomial. A thread's own sum is the first stretch's
  // with it, a risen thread's candidates are done.
  double more = 0.0;
  if ((int)threadIdx.x < n && !(found[threadIdx.x] & 1)) more = replaced(of_ordered((uint32_t)(found[threadIdx.x] >> 32)) - first_top);
  // All from the part's largest logit, if a thread has risen to it: it is a candidate.
  const float largest = n ? of_ordered((uint32_t)(found[0] >> 32)) : first_top, most = largest > first_top + kRise ? largest : first_top;
  if (from < most) sum = recounted(sum, from, most);
  if (first_top < most && more != 0.0) more = recounted(more, first_top, most);
  sum += more;
  const int64_t place = (int64_t)row * a.parts + blockIdx.x;
  uint64_t *const best = a.best + place * a.keep;
  if ((int)threadIdx.x < n) best[threadIdx.x] = found[threadIdx.x];
  for (int i = n + threadIdx.x; i < a.keep; i += kThreads) best[i] = 0;
#pragma unroll
  for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
  if (lane == 0) sums[warp] = sum;
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) all += sums[i];
    a.sum[place] = all;
    a.top[place] = odd ? __uint_as_float(0x7fc00000u) : most;
  }
}

// A sequence a block. A list is a part's of one beam, in descending order; a
// thread has lists threadIdx.x, + kJoin, ... From entries 0, 1, 3, 7, ... of each list
// follows a border that at least `keep` entries reach, and few more; those are ranked
// against each other. Where too many are equal, the best of all heads is taken `keep`
// times instead.
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
  const int seq = blockIdx.x, lists = a.beams * a.parts, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const double none = -INFINITY;
  cudaGridDependencySynchronize();  // (it may begin before the parts are done)
  // (entries 0, 1, 3, 7, ... of a thread's first list are on their way meanwhile)
  uint64_t some[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; j++)
    some[j] = (int)threadIdx.x < lists && (1 << j) <= a.keep ? a.best[((int64_t)seq * lists + threadIdx.x) * a.keep + (1 << j) - 1] : 0;
  // A few lanes a beam: all beams at once.
  int lanes = 32;
  while (lanes * a.beams > kJoin) lanes /= 2;
  {
    const int b = threadIdx.x / lanes;
    const int64_t row = (int64_t)seq * a.beams + b;
    const bool there = b < a.beams, end = there && a.ended && a.ended[row];
    const double score = there ? (double)a.scores[row] : 0.0;
    float top = -INFINITY;
    double sum = 0.0;
    if (there && !end)
      for (int s = threadIdx.x % lanes; s < a.parts; s += lanes) {
        const float t = a.top[row * a.parts + s];
        const double part = a.sum[row * a.parts + s];
        const float m = max_nan(top, t);
        if (m > -INFINITY) sum = (top > -INFINITY ? sum * exp((double)top - (double)m) : 0.0) + (t > -INFINITY ? part * exp((double)t - (double)m) : 0.0);
        top = m;
      }
    float m = top;
    for (int i = 1; i < lanes; i *= 2) m = max_nan(m, __shfl_xor_sync(~0u, m, i));
    sum = top > -INFINITY ? sum * exp((double)top - (double)m) : 0.0;
    for (int i = 1; i < lanes; i *= 2) sum += __shfl_xor_sync(~0u, sum, i);
    if (there && threadIdx.x % lanes == 0) {
      base[b] = end ? score : m > -INFINITY ? score - log(sum) : __longlong_as_double(0x7ff8000000000000ll);
      top_of[b] = m;
      ended[b] = end;
    }
  }
  for (int i = threadIdx.x; i < lists; i += kJoin) at_list[i] = 0;
  if (threadIdx.x == 0) picked = 0;
  __syncthreads();
  // A list is named by its beam (the upper half) and its number. Entry `at` of it: its
  // key, 0 behind the last, and its total.
  auto named = [&](int l) { return l / a.parts << 16 | l; };
  auto entry = [&](int l, int at, double &t) -> uint64_t {
    const int b = l >> 16;
    l &= 0xffff;
    t = base[b];
    if (ended[b]) return l == b * a.parts && at == 0 && t > none ? ~0ull : 0;
    if (at >= a.keep || !(t > none)) return 0;
    const uint64_t k = a.best[((int64_t)seq * lists + l) * a.keep + at];
    t += (double)of_ordered((uint32_t)(k >> 32)) - (double)top_of[b];
    return t > none ? k : 0;
  };
  // Whether the second goes before the first; a list below 0: none.
  auto better = [&](double t, uint64_t k, int l, double t2, uint64_t k2, int l2) {
    if (l2 < 0) return false;
    if (l < 0) return true;
    if (t != t2) return t2 > t;
    return l >> 16 != l2 >> 16 ? l2 >> 16 < l >> 16 : k2 > k;
  };
  auto write = [&](int i, double t, uint64_t k, int l) {
    const int64_t to = (int64_t)seq * a.keep + i;
    a.next[to] = l < 0 ? -INFINITY : (float)t;
    a.parents[to] = l < 0 ? -1 : seq * a.beams + (l >> 16);
    a.tokens[to] = l < 0 ? -1 : k == ~0ull ? a.end_token : token_of(k);
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
      const int name = named(l);
      const uint64_t k = entry(name, at_list[l], t);
      if (k && better(total, key, list, t, k, name)) total = t, key = k, list = name;
    }
  };
  // The totals of those entries; none: -infinity.
  double reached[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; j++) {
    const int b = min((int)threadIdx.x / a.parts, a.beams - 1);
    if (ended[b]) reached[j] = j == 0 && (int)threadIdx.x < lists && threadIdx.x % a.parts == 0 ? base[b] : none;
    else reached[j] = some[j] ? base[b] + ((double)of_ordered((uint32_t)(some[j] >> 32)) - (double)top_of[b]) : none;
    if (!(reached[j] > none)) reached[j] = none;
  }
  // How many entries reach each of eight borders at least: of a list whose entry
  // 2^j - 1 does, 2^j; so that less than twice as many do (and as many lists more).
  // Returns the last border that `keep` reach (and how many do), 8 for none; borders
  // descend.
  auto first_enough = [&](const double (&t)[8], int &c) {
    int m[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      m[i] = 0;
#pragma unroll
      for (int j = 0; j < kSteps; j++) m[i] += reached[j] >= t[i] ? (1 << j) - (1 << j >> 1) : 0;
    }
    for (int l = threadIdx.x + kJoin; l < lists; l += kJoin) {
      const int name = named(l);
      for (int j = 0; j < kSteps && 1 << j <= a.keep; j++) {
        double u;
        if (!entry(name, (1 << j) - 1, u)) break;
        for (int i = 0; i < 8; i++) m[i] += u >= t[i] ? (1 << j) - (1 << j >> 1) : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      m[i] = __reduce_add_sync(~0u, m[i]);
      if (lane == i) list_of[warp * 8 + i] = m[i];
    }
    __syncthreads();
    int got = 0;
    if (lane < 8)
      for (int i = 0; i < kJoin / 32; i++) got += list_of[i * 8 + lane];
    const unsigned enough = __ballot_sync(~0u, lane < 8 && got >= a.keep);
    const int at = enough ? __ffs(enough) - 1 : 8;
    if (at < 8) c = __shfl_sync(~0u, got, at);
    __syncthreads();
    return at;
  };
  // A border that `keep` entries reach, and few more: some way below the best, then
  // by eighths of what is left.
  double best = reached[0];
  for (int l = threadIdx.x + kJoin; l < lists; l += kJoin) {
    double t;
    if (entry(named(l), 0, t)) best = fmax(best, t);
  }
  for (int i = 16; i; i /= 2) best = fmax(best, __shfl_xor_sync(~0u, best, i));
  if (lane == 0) total_of[warp] = best;
  __syncthreads();
  for (int i = 0; i < kJoin / 32; i++) best = fmax(best, total_of[i]);
  double near = best, far = none;  // (too few reach `near`, enough reach `far`)
  if (best > none) {
    int c = 0;
    double t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = best - (double)(1 << (i < 6 ? i : 2 * i - 5));  // 1, 2, 4, ... 32, 128, 512
    const int at = first_enough(t, c);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i == at) far = t[i];
      if (i < at) near = t[i];
    }
    for (int k = 0; k < 4 && far > none && c > a.keep + a.keep / 2 + 8; k++) {
      const double by = (far - near) / 9.0;
#pragma unroll
      for (int i = 0; i < 8; i++) t[i] = near + by * (i + 1);
      const int at = first_enough(t, c);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (i == at) far = t[i];
        if (i < at) near = t[i];
      }
    }
  }
  const double least = far;  // (-infinity: all there are)
  auto pick = [&](double t, uint64_t k, int name) {
    const int i = atomicAdd(&picked, 1);
    if (i < kPicked) total_of[i] = t, key_of[i] = k, list_of[i] = name;
  };
  if (lists * a.keep <= kScan) {  // (all entries at once: their loads wait for nothing)
    for (int i0 = threadIdx.x; i0 < lists * a.keep; i0 += 8 * kJoin) {
      uint64_t k[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int i = i0 + j * kJoin;
        k[j] = i < lists * a.keep ? a.best[(int64_t)seq * lists * a.keep + i] : 0;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int i = i0 + j * kJoin, l = i / a.keep;
        if (i >= lists * a.keep) break;
        const int b = l / a.parts;
        double t = base[b];
        if (ended[b]) k[j] = l == b * a.parts && i == l * a.keep ? ~0ull : 0;
        else t += (double)of_ordered((uint32_t)(k[j] >> 32)) - (double)top_of[b];
        if (k[j] && t >= least && t > none) pick(t, k[j], b << 16 | l);
      }
    }
  } else {
    for (int l = threadIdx.x; l < lists; l += kJoin) {
      const int name = named(l);
      for (int at = 0;; at += 4) {
        double t[4];
        uint64_t k[4];
#pragma unroll
        for (int j = 0; j < 4; j++) k[j] = entry(name, at + j, t[j]);
        bool on = true;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          on = on && k[j] && t[j] >= least;
          if (on) pick(t[j], k[j], name);
        }
        if (!on || picked > kPicked) break;
      }
    }
  }
  __syncthreads();
  const int n = picked;
  if (n <= kPicked) {
    // (`per` lanes count for one; equal totals, which are rare, are told apart after)
    const int per = n <= kJoin / 4 ? 4 : n <= kJoin / 2 ? 2 : 1, off = (int)threadIdx.x % per;
    for (int i0 = 0; i0 < n; i0 += kJoin / per) {
      const int i = i0 + (int)threadIdx.x / per;
      const double t = i < n ? total_of[i] : none;
      int before = 0, same = 0;
#pragma unroll 8
      for (int j = off; j < n; j += per) {
        const double t2 = total_of[j];
        before += t2 > t;
        same += t2 == t;
      }
      for (int j = 1; j < per; j *= 2) {
        before += __shfl_xor_sync(~0u, before, j);
        same += __shfl_xor_sync(~0u, same, j);
      }
      if (i < n && off == 0) {
        const uint64_t k = key_of[i];
        const int l = list_of[i];
        if (same > 1)
          for (int j = 0; j < n; j++) before += j != i && total_of[j] == t && better(t, k, l, t, key_of[j], list_of[j]);
        if (before < a.keep) write(before, t, k, l);
      }
    }
    for (int i = n + threadIdx.x; i < a.keep; i += kJoin) write(i, none, 0, -1);
    return;
  }

  offer();
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
    if (l >= 0 && (l & 0xffff) % kJoin == (int)threadIdx.x) {
      at_list[l & 0xffff]++;
      offer();
    }
  }
}

// How a row is cut: stretches of `nv` vectors a thread, `turns` of them a part.
struct Cut {
  int nv, stretch, turns, parts;
};
Cut cut(int64_t rows, int vocab, size_t size, int sms) {
  Cut c;
  auto stretches = [&](int nv) {
    c.stretch = nv * kThreads * (16 / (int)size);
    return (vocab + c.stretch - 1) / c.stretch;
  };
  // Shorter stretches where they would leave SMs without work, or be half empty.
  c.nv = size == 2 ? 4 : 8;
  while (c.nv > 1 && (rows * stretches(c.nv) < 2 * sms || stretches(c.nv / 2) == 1)) c.nv /= 2;
  const int n = stretches(c.nv);
  // Turns of blocks, four an SM, by the stretches of each, the first of which costs
  // two: its border has to be found. (512 rows of 128256: 47 us at 8 and 16 stretches a
  // part, 53 at 4, 73 at 1; 160 rows of 50257: with a join of 19 us, 38 at 1, 47 at 2,
  // 60 at 7.)
  const int64_t slots = 4 * (int64_t)sms;
  int64_t least = INT64_MAX;
  c.turns = 1;
  for (int t = 1; t <= n; t++) {
    const int64_t cost = (rows * ((n + t - 1) / t) + slots - 1) / slots * (t + 1);
    if (cost < least) least = cost, c.turns = t;
  }
  c.parts = (n + c.turns - 1) / c.turns;
  return c;
}

}  // namespace

// (float32's shortest stretches are the most parts that a row can have)
size_t beam_work_bytes(int64_t rows, int32_t keep, int32_t vocab) {
  const int64_t parts = (vocab + 4 * kThreads - 1) / (4 * kThreads);
  return (size_t)(rows * parts * (8 * (int64_t)keep + 12) + 16);
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
  // (a sequence's scores are read before its results are written, by the same block)
  const int64_t out = 4 * (int64_t)c.seqs * c.keep;
  const bool in_place = (const void *)c.next == c.scores && c.keep == c.beams;
  for (const void *p : {(const void *)c.next, (const void *)c.parents, (const void *)c.tokens})
    if ((!(in_place && p == c.next) && meet(p, out, c.scores, 4 * rows)) || meet(p, out, c.ended, 4 * rows) ||
        meet(p, 1, 0, out, c.logits, rows, c.row * (int64_t)size, c.vocab * (int64_t)size))
      return fail("beam_select: a result shares memory with an operand (the next scores may be the scores, where as many are kept as there are beams)");
  if (meet(c.next, out, c.parents, out) || meet(c.next, out, c.tokens, out) || meet(c.parents, out, c.tokens, out))
    return fail("beam_select: two results share memory");
  const size_t need = beam_work_bytes(rows, c.keep, c.vocab);
  if (!c.workspace || c.workspace_bytes < need) return fail("beam_select: a workspace of %zu bytes, %zu needed", c.workspace ? c.workspace_bytes : 0, need);
  if ((uintptr_t)c.workspace % 8) return fail("beam_select: misaligned workspace");
  bool used = meet(c.workspace, 1, 0, (int64_t)need, c.logits, rows, c.row * (int64_t)size, c.vocab * (int64_t)size) ||
              meet(c.workspace, (int64_t)need, c.scores, 4 * rows) || meet(c.workspace, (int64_t)need, c.ended, 4 * rows);
  for (const void *p : {(const void *)c.next, (const void *)c.parents, (const void *)c.tokens}) used = used || meet(c.workspace, (int64_t)need, p, out);
  if (used) return fail("beam_select: the workspace shares memory with an operand or a result");
  const Cut how = cut(rows, c.vocab, size, sms);
  BeamArgs a;
  a.z = c.logits; a.row = c.row; a.scores = c.scores; a.ended = c.ended; a.next = c.next; a.parents = c.parents; a.tokens = c.tokens;
  a.vocab = c.vocab; a.beams = c.beams; a.keep = c.keep; a.end_token = c.end_token;
  a.group = 32;
  while (a.group > 1 && kThreads / a.group < c.keep) a.group /= 2;
  a.part = how.stretch * how.turns;
  a.parts = how.parts;
  a.best = (uint64_t *)c.workspace;
  a.sum = (double *)(a.best + rows * a.parts * c.keep);
  a.top = (float *)(a.sum + rows * a.parts);
  const dim3 grid((unsigned)a.parts, (unsigned)rows);
  if (c.dtype == kF16) {
    if (how.nv == 4) k_beam_parts<__half, 4><<<grid, kThreads, 0, st>>>(a);
    else if (how.nv == 2) k_beam_parts<__half, 2><<<grid, kThreads, 0, st>>>(a);
    else k_beam_parts<__half, 1><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (how.nv == 8) k_beam_parts<float, 8><<<grid, kThreads, 0, st>>>(a);
    else if (how.nv == 4) k_beam_parts<float, 4><<<grid, kThreads, 0, st>>>(a);
    else if (how.nv == 2) k_beam_parts<float, 2><<<grid, kThreads, 0, st>>>(a);
    else k_beam_parts<float, 1><<<grid, kThreads, 0, st>>>(a);
  }
  SHLO_TRY(launch_check("beam_select"));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c.seqs);
  cfg.blockDim = dim3(kJoin);
  cfg.dynamicSmemBytes = (size_t)c.beams * a.parts;
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

int shlo_beam_select_noalloc(const shlo_beam_args *args, void *stream) {
  if (!args) return fail("beam_select: null arguments");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_beam_select(*args, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
