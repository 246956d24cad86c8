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
// of a degree that is right to 2^-25 at each term and unbiased, sums are split into
// multiples of 2^-20 (exact) and rests, and the join is in 64 bits. A row's
// logarithm is then good to 10^-8 and mostly better.
//
// Bound: bytes (each logit read once); the first kernel's 15 instructions a logit
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

// 2^f = 1 + f q(f) for |f| <= 1/2, q of degree 5 fitted to the smallest largest
// relative error (2^-28; with the coefficients' rounding 2^-26, 1.5e-9 on average).
__device__ __forceinline__ float2 exp_below(float2 x, float2 top) {
  float2 d = __fadd2_rn(x, make_float2(-top.x, -top.y));
  d.x = fmaxf(d.x, -87.0f);  // (what lies below adds 10^-38)
  d.y = fmaxf(d.y, -87.0f);
  // d log2(e) as a sum of two
  const float2 t = __fmul2_rn(d, both(0x1.715476p+0f));
  float2 r = __ffma2_rn(d, both(0x1.715476p+0f), make_float2(-t.x, -t.y));
  r = __ffma2_rn(d, both(0x1.4ae0cp-26f), r);
  const float2 m = __fadd2_rn(t, both(12582912.0f));
  const float2 i = __fadd2_rn(m, both(-12582912.0f));
  const float2 f = __fadd2_rn(__fadd2_rn(t, make_float2(-i.x, -i.y)), r);
  float2 q = both(0x1.41fbaep-13f);
  q = __ffma2_rn(q, f, both(0x1.5f3e6ap-10f));
  q = __ffma2_rn(q, f, both(0x1.3b2d4ep-7f));
  q = __ffma2_rn(q, f, both(0x1.c6aee8p-5f));
  q = __ffma2_rn(q, f, both(0x1.ebfbdcp-3f));
  q = __ffma2_rn(q, f, both(0x1.62e430p-1f));
  q = __ffma2_rn(q, f, both(1.0f));
  q.x = __uint_as_float(__float_as_uint(q.x) + (__float_as_uint(m.x) << 23));
  q.y = __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(m.y) << 23));
  return q;
}

// A vector of 16 bytes as floats.
__device__ __forceinline__ void floats(const uint4 &v, float (&f)[8]) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 p = __half22float2(h[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void floats(const uint4 &v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
template <typename T> struct NegInf;
template <> struct NegInf<__half> { static __device__ __half v() { return __ushort_as_half(0xfc00); } };
template <> struct NegInf<float> { static __device__ float v() { return -INFINITY; } };

template <typename T, int NV>
__global__ void __launch_bounds__(kThreads) k_beam_segments(const BeamArgs a) {
  constexpr int W = 16 / sizeof(T);  // values a vector
  __shared__ float tops[kWarps];
  __shared__ double sums[kWarps];
  __shared__ uint64_t found[kRoom];
  __shared__ int count;
  const int row = blockIdx.y, s = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (a.ended && a.ended[row]) return;  // it goes on with one token, whatever its logits
  // Vectors begin on 16-byte boundaries of memory: segment 0 a few values before the row.
  const T *const z = static_cast<const T *>(a.z) + row * a.row;
  const int before = (int)(((uintptr_t)z & 15) / sizeof(T));
  const int lo = s * a.seg - before;
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int at = lo + (i * kThreads + threadIdx.x) * W;
    if (at >= 0 && at + W <= a.vocab) {
      v[i] = __ldg(reinterpret_cast<const uint4 *>(z + at));
    } else {
      T e[W];
#pragma unroll
      for (int j = 0; j < W; j++) e[j] = at + j >= 0 && at + j < a.vocab ? z[at + j] : NegInf<T>::v();
      memcpy(&v[i], e, 16);
    }
  }
  if (threadIdx.x == 0) count = 0;
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float f[W];
    floats(v[i], f);
#pragma unroll
    for (int j = 0; j < W; j++) mine = max_nan(mine, f[j]);
  }
  float top = mine;
#pragma unroll
  for (int i = 16; i; i /= 2) top = max_nan(top, __shfl_xor_sync(~0u, top, i));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  float low = INFINITY;  // the smallest of the warps' largest: eight logits at least are not below it
#pragma unroll
  for (int i = 0; i < kWarps; i++) {
    top = max_nan(top, tops[i]);
    low = fminf(low, tops[i]);
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

  // A border that at least `keep` threads' largest logits reach (or all that are
  // above -infinity), and few more: found by halving between two borders.
  uint32_t under = kNegInf + 1, over = ordered(top) + 1;  // count(under) is enough, count(over) is not
  const uint32_t key = ordered(mine);
  int have = kThreads;
  if (a.keep <= kWarps && low > -INFINITY) under = ordered(low);
  const int live = __syncthreads_count(key >= under);
  have = live;
  if (live >= a.keep) {
    for (int i = 0; i < 32 && have > 2 * a.keep && over - under > 1; i++) {
      const uint32_t mid = under + (over - under) / 2;
      const int n = __syncthreads_count(key >= mid);
      if (n >= a.keep) under = mid, have = n;
      else over = mid;
    }
  } else {
    under = kNegInf + 1;  // fewer threads than `keep` have any: all of it, or the exact border below
  }

  float2 high = both(0.0f), rest = both(0.0f);
  const float2 tt = both(top);
  const float border = of_ordered(under);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float f[W];
    floats(v[i], f);
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float2 e = exp_below(make_float2(f[j], f[j + 1]), tt);
      // (sums of multiples of 2^-20 up to 16 are exact: each half has 16 terms of at most 1)
      const float2 h = __fadd2_rn(__fadd2_rn(e, both(12.0f)), both(-12.0f));
      high = __fadd2_rn(high, h);
      rest = __fadd2_rn(rest, __fadd2_rn(e, make_float2(-h.x, -h.y)));
    }
  }
  double sum = ((double)high.x + (double)high.y) + ((double)rest.x + (double)rest.y);
#pragma unroll
  for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
  if (lane == 0) sums[warp] = sum;
  if (key >= under) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float f[W];
      floats(v[i], f);
#pragma unroll
      for (int j = 0; j < W; j++)
        if (f[j] >= border) {
          const int n = atomicAdd(&count, 1);
          if (n < kRoom) found[n] = (uint64_t)ordered(f[j]) << 32 | (uint32_t)~(lo + (i * kThreads + threadIdx.x) * W + j);
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
#pragma unroll
      for (int i = 0; i < NV; i++) {
        float f[W];
        floats(v[i], f);
#pragma unroll
        for (int j = 0; j < W; j++) {
          const uint32_t u = ordered(f[j]);
          if (u > t || (u == t && (uint32_t)~(lo + (i * kThreads + threadIdx.x) * W + j) >= last)) c++;
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
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float f[W];
      floats(v[i], f);
#pragma unroll
      for (int j = 0; j < W; j++) {
        const uint32_t u = ordered(f[j]), last = ~(lo + (i * kThreads + threadIdx.x) * W + j);
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
// thread has lists threadIdx.x, + kJoin, ..., and offers the best of their heads.
__global__ void __launch_bounds__(kJoin) k_beam_join(const BeamArgs a) {
  extern __shared__ unsigned char at_list[];  // of a list: how many of its entries are taken
  // Of a beam: its score less the logarithm of its row's sum (NaN: none to choose
  // from), and its row's largest logit, from which the others are counted: they may
  // be far from 0.
  __shared__ double base[kMaxBeams];
  __shared__ float top_of[kMaxBeams];
  __shared__ double won_total[kJoin / 32];
  __shared__ uint64_t won_key[kJoin / 32];
  __shared__ int won_list[kJoin / 32];
  const int seq = blockIdx.x, lists = a.beams * a.segs, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const double none = -INFINITY;
  for (int b = warp; b < a.beams; b += kJoin / 32) {
    const int64_t row = (int64_t)seq * a.beams + b;
    const double score = (double)a.scores[row];
    if (a.ended && a.ended[row]) {
      if (lane == 0) base[b] = score;
      continue;
    }
    float top = -INFINITY;
    for (int s = lane; s < a.segs; s += 32) top = max_nan(top, a.top[row * a.segs + s]);
    for (int i = 16; i; i /= 2) top = max_nan(top, __shfl_xor_sync(~0u, top, i));
    double sum = 0.0;
    if (top > -INFINITY)
      for (int s = lane; s < a.segs; s += 32) {
        const float t = a.top[row * a.segs + s];
        if (t > -INFINITY) sum += a.sum[row * a.segs + s] * exp((double)t - (double)top);
      }
    for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
    if (lane == 0) {
      base[b] = top > -INFINITY ? score - log(sum) : __longlong_as_double(0x7ff8000000000000ll);
      top_of[b] = top;
    }
  }
  for (int i = threadIdx.x; i < lists; i += kJoin) at_list[i] = 0;
  __syncthreads();
  // The best of this thread's heads: its total, its key (a larger one goes first
  // within a beam) and its list; list -1: none.
  double total;
  uint64_t key;
  int list;
  auto better = [&](double t, uint64_t k, int l, double t2, uint64_t k2, int l2) {  // the second is the better one
    if (l2 < 0) return false;
    if (l < 0) return true;
    if (t != t2) return t2 > t;
    const int b = l / a.segs, b2 = l2 / a.segs;
    return b != b2 ? b2 < b : k2 > k;
  };
  auto offer = [&]() {
    list = -1;
    total = none;
    key = 0;
    for (int l = threadIdx.x; l < lists; l += kJoin) {
      const int b = l / a.segs, at = at_list[l];
      const int64_t row = (int64_t)seq * a.beams + b;
      uint64_t k = 0;
      double t = base[b];
      if (a.ended && a.ended[row]) {
        if (l % a.segs == 0 && at == 0) k = ~0ull;
      } else if (at < a.keep) {
        k = a.best[(row * a.segs + l % a.segs) * a.keep + at];
        t += (double)of_ordered((uint32_t)(k >> 32)) - (double)top_of[b];
      }
      if (k == 0 || !(t > none)) continue;
      if (better(total, key, list, t, k, l)) total = t, key = k, list = l;
    }
  };
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
    if (lane == 0) won_total[warp] = t, won_key[warp] = k, won_list[warp] = l;
    __syncthreads();
    for (int j = 0; j < kJoin / 32; j++)
      if (better(t, k, l, won_total[j], won_key[j], won_list[j])) t = won_total[j], k = won_key[j], l = won_list[j];
    if (threadIdx.x == 0) {
      const int64_t to = (int64_t)seq * a.keep + i;
      a.next[to] = l < 0 ? -INFINITY : (float)t;
      a.parents[to] = l < 0 ? -1 : seq * a.beams + l / a.segs;
      a.tokens[to] = l < 0 ? -1 : k == ~0ull ? a.end_token : (int32_t)~(uint32_t)k;
    }
    if (l >= 0 && l % kJoin == (int)threadIdx.x) {
      at_list[l]++;
      offer();
    }
  }
}

// A segment's logits: of a row of 16-byte vectors as many as a block holds, or
// fewer where the segments would leave SMs without work.
int vectors(int64_t rows, int vocab, size_t size, int sms) {
  const int most = size == 2 ? 4 : 8;
  int nv = most;
  auto blocks = [&](int n) { return rows * ((vocab + 16 / (int)size - 1 + n * kThreads * (16 / (int)size) - 1) / (n * kThreads * (16 / (int)size))); };
  while (nv > 1 && blocks(nv) < 2 * sms) nv /= 2;
  return nv;
}
int segments(int vocab, size_t size, int nv) {  // (a row may begin up to a vector's length less one value after a boundary)
  const int w = 16 / (int)size, seg = nv * kThreads * w;
  return (vocab + w - 1 + seg - 1) / seg;
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
  k_beam_join<<<c.seqs, kJoin, (size_t)c.beams * a.segs, st>>>(a);
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
