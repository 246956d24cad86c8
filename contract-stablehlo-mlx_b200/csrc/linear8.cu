// Products of activations and weights in 8-bit integers.
//   rows:    q[i] = the whole number nearest to 127 x[i] / top (of two, the even
//            one), scale = top / 127, where top is the row's largest magnitude;
//            a row of zeros has scale 0, one with a value that is not finite
//            zeros and scale NaN.
//   product: y[r][c] = (sum over i of q[r][i] w[c][i]) scale[r] w_scale[c] + bias[c],
//            the sum in 32-bit integers, exact for up to 131071 terms; then four
//            roundings (to binary32, two products, the bias) and the result's own.
//
// Rows, bound: bytes, and close behind them ten instructions a value. 8192 rows of 4096
// float16 (101 MB) 21 us, 4.8 TB/s; 5893 rows of 5727 float32,
// which start at any multiple of 4 bytes (169 MB) 32 us; 24 rows of 4096 2.4 us, a launch
// and four waits. Measured: the first of these with 256 threads a row and a check of its
// end at every vector 27 us, with 64 threads 25, and no checks 21. The product of linear8
// begins while they are rounded, with its weights.
#include <algorithm>
#include <type_traits>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kQuantThreads = 256;

__device__ __forceinline__ float to_f32(__half h) { return __half2float(h); }
__device__ __forceinline__ float to_f32(float f) { return f; }

template <int BYTES> struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<2> { using T = uint16_t; };
template <> struct Raw<1> { using T = uint8_t; };

// The larger of three magnitudes; NaN if one is. (The first is one already.)
__device__ __forceinline__ float top_of(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest magnitude of what a thread has seen (float16: two of them), and its bits as
// a float's: those of values that are not finite are above all others'.
template <typename T> struct Top;
template <> struct Top<float> {
  float top = 0.0f;
  template <int V> __device__ __forceinline__ void see(const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) top = top_of(top, v[i], v[i + 1]);
  }
  __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(fabsf(top)); }
};
template <> struct Top<__half> {
  __half2 top = __half2half2(__ushort_as_half(0));
  template <int V> __device__ __forceinline__ void see(const __half (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) top = __hmax2_nan(top, __habs2(__halves2half2(v[i], v[i + 1])));
  }
  __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(fabsf(top_of(0.0f, __low2float(top), __high2float(top)))); }
};

// V values as the whole numbers nearest to 127 x / top. x times 127 / top is within
// 2^-23 of that (2^-16 at 127) and mostly decides; it is rounded by an add of 1.5 2^23,
// whose low byte then is the integer's. A value near the middle between two whole
// numbers h and h + 1 is decided by 254 |x| against (2 h + 1) top, both exact: of 18 and
// 19 bits where x has 11, else in 64. Where 127 / top is not a number of 32 bits, a
// quotient of 64 bits decides: x and top have 24, so it is the middle itself or 2^-33 of
// it away.
__device__ __noinline__ int decide(float x, float top) { return (int)rint((double)x * 127.0 / (double)top); }
template <typename T> __device__ __forceinline__ int middle(float x, float top, float r) {
  using W = typename std::conditional<sizeof(T) == 2, float, double>::type;
  const float h = floorf(fabsf(r));
  const W a = (W)254.0f * (W)fabsf(x), b = (W)(2.0f * h + 1.0f) * (W)top;
  const int k = (int)h, up = a > b || (a == b && (k & 1));
  return r < 0.0f ? -(k + up) : k + up;
}
template <typename T, int V>
__device__ __forceinline__ void quantise(const T (&v)[V], float top, float by, uint8_t (&q)[V]) {  // (q on a boundary of four)
  uint32_t m[V];
  float off = 0.0f;  // the farthest from its integer
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const float2 r = __fmul2_rn(make_float2(to_f32(v[j]), to_f32(v[j + 1])), make_float2(by, by));
    const float2 s = __fadd2_rn(r, make_float2(12582912.0f, 12582912.0f));
    const float2 k = __fadd2_rn(s, make_float2(-12582912.0f, -12582912.0f));
    const float2 d = __ffma2_rn(k, make_float2(-1.0f, -1.0f), r);
    off = top_of(off, d.x, d.y);
    m[j] = __float_as_uint(s.x);
    m[j + 1] = __float_as_uint(s.y);
  }
  if (sizeof(T) == 4 && !(by < 0x1p120f)) {
#pragma unroll
    for (int j = 0; j < V; j++) m[j] = (uint32_t)decide(to_f32(v[j]), top);
  } else if (!(off < 0.5f - 0x1p-15f)) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float r = to_f32(v[j]) * by, far = fabsf(r) - floorf(fabsf(r));
      if (fabsf(far - 0.5f) <= 0x1p-15f) m[j] = (uint32_t)middle<T>(to_f32(v[j]), top, r);
    }
  }
#pragma unroll
  for (int j = 0; j < V; j += 4)
    *reinterpret_cast<uint32_t *>(q + j) = __byte_perm(__byte_perm(m[j], m[j + 1], 0x0040), __byte_perm(m[j + 2], m[j + 3], 0x0040), 0x5410);
}

// TPR threads a row, V values of it at a time in loads of PIECE bytes (what x's
// alignment allows); a row of up to KEEP TPR of them stays in registers between the two
// passes, a longer one is read again from L2. `wide`: q allows stores of V bytes.
template <typename T, int V, int PIECE, int TPR, int KEEP>
__global__ void __launch_bounds__(kQuantThreads, KEEP <= 2 ? 6 : KEEP == 4 ? 5 : 4)
k_quantise_rows(const T *x, int64_t x_row, int64_t rows, int n, int8_t *q, int64_t q_row, float *scale, int fill, bool wide) {
  constexpr int ROWS = kQuantThreads / TPR, EACH = PIECE / (int)sizeof(T);
  using R = typename Raw<PIECE>::T;
  __shared__ uint32_t tops[kQuantThreads / 32];
  // (a product that waits for these rows may begin to read its weights)
  cudaTriggerProgrammaticLaunchCompletion();
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool there = row < rows;
  x += (there ? row : 0) * x_row;
  q += (there ? row : 0) * q_row;
  const int full = there ? n / V : 0;  // vectors; what is left of a row, less than one, has a thread
  const bool rest = there && n % V && t == full % TPR;
  auto load = [&](int i, T (&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; j += EACH) *reinterpret_cast<R *>(v + j) = *reinterpret_cast<const R *>(x + (int64_t)i * V + j);
  };
  alignas(16) T v[KEEP][V];
  Top<T> most;
#pragma unroll
  for (int k = 0; k < KEEP; k++) {
#pragma unroll
    for (int j = 0; j < V; j++) v[k][j] = T(0.0f);
    if (t + k * TPR < full) load(t + k * TPR, v[k]);
  }
  alignas(16) T last[V];
#pragma unroll
  for (int j = 0; j < V; j++) last[j] = rest && full * V + j < n ? x[(int64_t)full * V + j] : T(0.0f);
#pragma unroll
  for (int k = 0; k < KEEP; k++) most.see(v[k]);
  most.see(last);
#pragma unroll 2
  for (int i = t + KEEP * TPR; i < full; i += TPR) {
    alignas(16) T w[V];
    load(i, w);
    most.see(w);
  }
  uint32_t bits = __reduce_max_sync(~0u, most.bits());
  if (TPR > 32) {
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TPR / 32; i++) bits = max(bits, tops[threadIdx.x / TPR * (TPR / 32) + i]);
  }
  if (!there) return;
  const float top = __uint_as_float(bits), by = 127.0f / top;
  const bool finite = bits < 0x7f800000u;
  if (t == 0) scale[row] = finite ? top / 127.0f : __uint_as_float(0x7fc00000u);
  if (!finite || bits == 0) {
    for (int i = t; i < max(n, fill); i += TPR) q[i] = 0;
    return;
  }
  auto some = [&](int i, const T (&w)[V], int count) {  // of a vector's results the first few, one by one
    alignas(8) uint8_t b[V];
    quantise(w, top, by, b);
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j < count) q[(int64_t)i * V + j] = (int8_t)b[j];
  };
  auto store = [&](int i, const T (&w)[V]) {
    alignas(8) uint8_t b[V];
    quantise(w, top, by, b);
    *reinterpret_cast<typename Raw<V>::T *>(q + (int64_t)i * V) = *reinterpret_cast<const typename Raw<V>::T *>(b);
  };
  if (rest) some(full, last, n - full * V);
  if (wide) {
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (t + k * TPR < full) store(t + k * TPR, v[k]);
#pragma unroll 2
    for (int i = t + KEEP * TPR; i < full; i += TPR) {
      alignas(16) T w[V];
      load(i, w);
      store(i, w);
    }
  } else {
#pragma unroll 1
    for (int i = t; i < full; i += TPR) {
      alignas(16) T w[V];
      load(i, w);
      some(i, w, V);
    }
  }
  for (int i = n + t; i < fill; i += TPR) q[i] = 0;
}

template <typename T, int V, int PIECE>
void launch_rows(const T *x, int64_t x_row, int64_t rows, int n, int8_t *q, int64_t q_row, float *scale, int fill, cudaStream_t st) {
  const bool wide = (uintptr_t)q % V == 0 && (rows == 1 || q_row % V == 0);
  auto go = [&](auto kernel, int per) { kernel<<<(unsigned)((rows + per - 1) / per), kQuantThreads, 0, st>>>(x, x_row, rows, n, q, q_row, scale, fill, wide); };
  // Threads a row: a warp, or as many as keep the row; where there are rows for all SMs
  // few threads with much of it each, whose shares of the work for a row as a whole
  // are then small.
  const int vecs = (n + V - 1) / V;
  if (vecs <= 64) go(k_quantise_rows<T, V, PIECE, 32, 2>, 8);
  else if (vecs <= 256 && rows > 1024) go(k_quantise_rows<T, V, PIECE, 32, 8>, 8);
  else if (vecs <= 512 && rows > 2048) go(k_quantise_rows<T, V, PIECE, 64, 8>, 4);
  else if (vecs <= 1024 && rows > 4096) go(k_quantise_rows<T, V, PIECE, 128, 8>, 2);
  else if (vecs <= 512) go(k_quantise_rows<T, V, PIECE, 256, 2>, 1);
  else if (vecs <= 1024) go(k_quantise_rows<T, V, PIECE, 256, 4>, 1);
  else go(k_quantise_rows<T, V, PIECE, 256, 8>, 1);
}

// Few rows: a warp a channel, whose bytes go through its lanes 16 at a time, against
// the rows' in shared memory; each block rounds the rows for itself (T float16 or
// float32; int8: they are rounded), so that a step of one sequence is one launch. The
// first bytes of the weights are asked for before that. 1 row of 512 to 768 2.6 us, of
// 4096 to 4096 (16.8 MB from HBM) 6.4, to 12288 11.7 (4.3 TB/s with launch and ramp).
constexpr int kFewThreads = 256, kFewBytes = 64 * 1024;

template <typename T, int R, typename Y>
__global__ void __launch_bounds__(kFewThreads, 4) k_linear8_few(const Mm8Call c, int row_bytes, bool after_rows) {
  constexpr int U = 4, WARPS = kFewThreads / 32;
  constexpr bool ROUNDS = !std::is_same<T, int8_t>::value;
  extern __shared__ uint4 xs[];  // [R][row_bytes]: zeros behind n
  __shared__ uint32_t tops[WARPS];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, units = row_bytes / 16, row_units = row_bytes / 16;
  const int full = c.n / 16;
  auto weights = [&](int ch, int u) -> uint4 {
    const int8_t *const w = c.w + (int64_t)ch * c.w_row + (int64_t)u * 16;
    if (u < full) return __ldg(reinterpret_cast<const uint4 *>(w));
    uint4 v = make_uint4(0, 0, 0, 0);
    if (u == full)
      for (int i = 0; i < c.n % 16; i++) reinterpret_cast<int8_t *>(&v)[i] = w[i];
    return v;
  };
  const int step = gridDim.x * WARPS;
  int ch = blockIdx.x * WARPS + warp;
  uint4 w[U];
#pragma unroll
  for (int i = 0; i < U; i++)
    if (ch < c.m && i * 32 + lane < units) w[i] = weights(ch, i * 32 + lane);

  // The rows: a part of the threads each, up to KEEP vectors a thread on their way at once.
  float scale = 0.0f;  // lane r: row r's
  if constexpr (ROUNDS) {
    constexpr int V = 16 / sizeof(T), TPR = kFewThreads / R, KEEP = 4;
    const bool wide = (uintptr_t)c.x % 16 == 0 && (c.rows == 1 || c.x_row * (int64_t)sizeof(T) % 16 == 0);
    const int r = threadIdx.x / TPR, t = threadIdx.x % TPR, vecs = r < c.rows ? (c.n + V - 1) / V : 0;
    const T *const x = static_cast<const T *>(c.x) + (r < c.rows ? r : 0) * c.x_row;
    auto load = [&](int i, T (&v)[V]) {
      if (wide && i * V + V <= c.n) {
        *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(x + (int64_t)i * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = i * V + j < c.n ? x[(int64_t)i * V + j] : T(0.0f);
      }
    };
    T v[KEEP][V];
    Top<T> most;
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (t + k * TPR < vecs) load(t + k * TPR, v[k]);
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (t + k * TPR < vecs) most.see(v[k]);
    for (int i = t + KEEP * TPR; i < vecs; i += TPR) {
      T u[V];
      load(i, u);
      most.see(u);
    }
    uint32_t top = __reduce_max_sync(~0u, most.bits());
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    auto row_top = [&](int row) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < WARPS / R; i++) m = max(m, tops[row * (WARPS / R) + i]);
      return m;
    };
    if (lane < R) {
      const uint32_t m = row_top(lane);
      scale = m < 0x7f800000u ? __uint_as_float(m) / 127.0f : __uint_as_float(0x7fc00000u);
    }
    top = row_top(r);
    const float by = 127.0f / __uint_as_float(top);
    const bool any = top > 0 && top < 0x7f800000u;
    auto store = [&](int i, const T (&u)[V]) {
      alignas(8) uint8_t b[V];
#pragma unroll
      for (int j = 0; j < V; j++) b[j] = 0;
      if (any && i < vecs) quantise(u, __uint_as_float(top), by, b);
      *reinterpret_cast<typename Raw<V>::T *>(reinterpret_cast<uint8_t *>(xs) + r * row_bytes + i * V) = *reinterpret_cast<const typename Raw<V>::T *>(b);
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (t + k * TPR < row_bytes / V) store(t + k * TPR, v[k]);
    for (int i = t + KEEP * TPR; i < row_bytes / V; i += TPR) {
      T u[V];
      if (i < vecs) load(i, u);
      store(i, u);
    }
  } else {
    if (after_rows) cudaGridDependencySynchronize();
    if (lane < c.rows) scale = c.x_scale[lane];
    for (int i = threadIdx.x; i < R * units; i += kFewThreads) {
      const int r = i / units, u = i - r * units;
      uint4 v = make_uint4(0, 0, 0, 0);
      const int8_t *const x = static_cast<const int8_t *>(c.x) + r * c.x_row + (int64_t)u * 16;
      if (r < c.rows && u < full) v = *reinterpret_cast<const uint4 *>(x);
      else if (r < c.rows && u == full)
        for (int j = 0; j < c.n % 16; j++) reinterpret_cast<int8_t *>(&v)[j] = x[j];
      xs[i] = v;
    }
  }
  __syncthreads();

  for (; ch < c.m; ch += step) {
    int sum[R];
#pragma unroll
    for (int r = 0; r < R; r++) sum[r] = 0;
    for (int u0 = 0; u0 < units; u0 += 32 * U) {
      uint4 v[U];
#pragma unroll
      for (int i = 0; i < U; i++) v[i] = w[i];
      // the bytes that follow: of this channel, or of the next
      const bool more = u0 + 32 * U < units;
      const int ch2 = more ? ch : ch + step, u2 = more ? u0 + 32 * U : 0;
#pragma unroll
      for (int i = 0; i < U; i++)
        if (ch2 < c.m && u2 + i * 32 + lane < units) w[i] = weights(ch2, u2 + i * 32 + lane);
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int u = u0 + i * 32 + lane;
        if (u < units) {
#pragma unroll
          for (int r = 0; r < R; r++) {
            const uint4 x = xs[r * row_units + u];
            sum[r] = __dp4a((int)x.x, (int)v[i].x, sum[r]);
            sum[r] = __dp4a((int)x.y, (int)v[i].y, sum[r]);
            sum[r] = __dp4a((int)x.z, (int)v[i].z, sum[r]);
            sum[r] = __dp4a((int)x.w, (int)v[i].w, sum[r]);
          }
        }
      }
    }
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int all = __reduce_add_sync(~0u, sum[r]);
      if (lane == r) mine = all;
    }
    if (lane < c.rows) {
      float f = (float)mine * scale * c.w_scale[ch];
      if (c.bias) f += c.bias[ch];
      Y *const y = static_cast<Y *>(c.y) + lane * c.y_row + ch;
      if constexpr (sizeof(Y) == 2) *y = __float2half_rn(f);
      else *y = f;
    }
  }
}

template <typename T, typename Y>
int launch_few(const Mm8Call &c, bool after_rows, int sms, cudaStream_t st) {
  const int row_bytes = (c.n + 15) / 16 * 16, r = c.rows <= 1 ? 1 : c.rows <= 2 ? 2 : 4, bytes = r * row_bytes;
  const auto kernel = r == 1 ? k_linear8_few<T, 1, Y> : r == 2 ? k_linear8_few<T, 2, Y> : k_linear8_few<T, 4, Y>;
  if (bytes > 48 * 1024) {
    static std::atomic<uint64_t> set[5]{};
    int device;
    SHLO_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !(set[r].load(std::memory_order_relaxed) >> device & 1)) {
      SHLO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewBytes));
      if (device < 64) set[r].fetch_or(1ull << device);
    }
  }
  // As many blocks as run at once, or as have a channel a warp.
  const int64_t want = ((int64_t)c.m + kFewThreads / 32 - 1) / (kFewThreads / 32), most = (int64_t)sms * std::min(4, 200 * 1024 / std::max(bytes, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(want, most));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = after_rows ? 1 : 0;
  SHLO_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, row_bytes, after_rows));
  return launch_check(std::is_same<T, int8_t>::value ? "mul_mat8" : "linear8");
}
// Up to four rows, as long as a block's copy of them is small beside the weights that
// it reads. (Products alone, us, this and the tiles: 1 row of 4096 to 4096 channels 5.4
// and 9.0, 4 rows 6.8 and 9.1; 4 of 14336 to 4096 18.8 and 15.2.)
bool few(const Mm8Call &c) {
  const int64_t bytes = ((int64_t)c.n + 15) / 16 * 16;
  return c.rows == 1 ? bytes <= kFewBytes : c.rows <= 4 && (c.rows == 2 ? 2 : 4) * bytes <= 24 * 1024;
}
// Whether each of those blocks also rounds the rows, instead of a launch of its own (us:
// 1 row of 4096 to 4096 6.4 and 7.4, of 40000 46 and 43; 4 rows of 512 to 2048 3.4 and
// 4.2, 2 of 2048 5.5 and 4.7, 4 of 4096 to 4096 12.5 and 9.5).
bool few_round(const Mm8Call &c) { return c.rows == 1 ? c.n <= 16384 : c.rows * c.n <= 2048; }

}  // namespace

int launch_quantise_rows(const void *x, int64_t x_row, uint8_t dtype, int64_t rows, int32_t n, int8_t *q, int64_t q_row, float *scale,
                         bool fill, const char *what, cudaStream_t st) {
  if (dtype != kF16 && dtype != kF32) return fail("%s: %s not carried (float16 or float32)", what, dtype_name(dtype));
  if (rows < 0 || rows > 0x7fffffff || n < 1 || n > (1 << 30)) return fail("%s: %lld rows of %d values (up to 2^30)", what, (long long)rows, n);
  if (rows == 0) return 0;
  if (rows > 1 && q_row < n) return fail("%s: rows of q overlap", what);
  if (!x || !q || !scale) return fail("%s: null pointer", what);
  const size_t size = dtype_size(dtype);
  if ((uintptr_t)x % size || (uintptr_t)scale % 4) return fail("%s: an operand is not aligned to its type", what);
  if (meet(q, rows, q_row, n, x, rows, x_row * (int64_t)size, n * (int64_t)size) || meet(scale, 1, 0, 4 * rows, x, rows, x_row * (int64_t)size, n * (int64_t)size) ||
      meet(scale, 1, 0, 4 * rows, q, rows, q_row, n))
    return fail("%s: q, scale and x share memory", what);
  const uintptr_t at = (uintptr_t)x | (rows > 1 ? (uintptr_t)(x_row * (int64_t)size) : 0);
  const int end = fill ? (n + 15) / 16 * 16 : n;
  if (dtype == kF16) {
    const __half *p = (const __half *)x;
    if (at % 16 == 0) launch_rows<__half, 8, 16>(p, x_row, rows, n, q, q_row, scale, end, st);
    else if (at % 8 == 0) launch_rows<__half, 4, 8>(p, x_row, rows, n, q, q_row, scale, end, st);
    else if (at % 4 == 0) launch_rows<__half, 4, 4>(p, x_row, rows, n, q, q_row, scale, end, st);
    else launch_rows<__half, 4, 2>(p, x_row, rows, n, q, q_row, scale, end, st);
  } else {
    const float *p = (const float *)x;
    if (at % 16 == 0) launch_rows<float, 4, 16>(p, x_row, rows, n, q, q_row, scale, end, st);
    else if (at % 8 == 0) launch_rows<float, 4, 8>(p, x_row, rows, n, q, q_row, scale, end, st);
    else launch_rows<float, 4, 4>(p, x_row, rows, n, q, q_row, scale, end, st);
  }
  return launch_check(what);
}

// The weights, the result and the sizes; x (of `x_size` bytes a value) where the result may not lie.
static int check_mul_mat8(const Mm8Call &c, int64_t x_size, const char *what) {
  if (c.dtype != kF16 && c.dtype != kF32) return fail("%s: a result of %s not carried (float16 or float32)", what, dtype_name(c.dtype));
  // (the kernels count channels in 32 bits, up to a grid's or a tile's beyond the last)
  if (c.rows < 0 || c.rows > (1 << 28) || c.m < 1 || c.m > (1 << 30) || c.n < 1 || c.n > 131071)
    return fail("%s: %lld rows, %d channels (at most 2^30) of %d values (32-bit sums hold 131071)", what, (long long)c.rows, c.m, c.n);
  if (c.rows == 0) return 0;
  if (!c.w || !c.w_scale || !c.y) return fail("%s: null pointer", what);
  if ((uintptr_t)c.w % 16 || (c.m > 1 && (c.w_row % 16 || c.w_row < c.n)))
    return fail("%s: rows of w begin on multiples of 16 bytes and do not overlap (a distance of %lld for %d values)", what, (long long)c.w_row, c.n);
  if (c.rows > 1 && c.y_row < c.m) return fail("%s: rows of the result overlap", what);
  if ((uintptr_t)c.w_scale % 4 || (uintptr_t)c.bias % 4 || (uintptr_t)c.y % dtype_size(c.dtype)) return fail("%s: an operand is not aligned to its type", what);
  const int64_t size = dtype_size(c.dtype);
  auto hits = [&](const void *p, int64_t rows, int64_t step, int64_t bytes) { return meet(c.y, c.rows, c.y_row * size, c.m * size, p, rows, step, bytes); };
  if (hits(c.x, c.rows, c.x_row * x_size, c.n * x_size) || hits(c.w, c.m, c.w_row, c.n) || hits(c.w_scale, 1, 0, 4 * (int64_t)c.m) ||
      hits(c.bias, 1, 0, 4 * (int64_t)c.m))
    return fail("%s: the result shares memory with an operand", what);
  return 0;
}

int launch_mul_mat8(const Mm8Call &c, bool after_rows, int *err, int sms, cudaStream_t st) {
  SHLO_TRY(check_mul_mat8(c, 1, "mul_mat8"));
  if (c.rows == 0) return 0;
  if (!c.x || !c.x_scale) return fail("mul_mat8: null pointer");
  if (meet(c.y, c.rows, c.y_row * (int64_t)dtype_size(c.dtype), c.m * (int64_t)dtype_size(c.dtype), c.x_scale, 1, 0, 4 * c.rows))
    return fail("mul_mat8: the result shares memory with an operand");
  if ((uintptr_t)c.x % 16 || (c.rows > 1 && (c.x_row % 16 || c.x_row < c.n)))
    return fail("mul_mat8: rows of x begin on multiples of 16 bytes and do not overlap (a distance of %lld for %d values)", (long long)c.x_row, c.n);
  if ((uintptr_t)c.x_scale % 4) return fail("mul_mat8: an operand is not aligned to its type");
  if (few(c)) return c.dtype == kF16 ? launch_few<int8_t, __half>(c, after_rows, sms, st) : launch_few<int8_t, float>(c, after_rows, sms, st);
  return launch_mul_mat8_tiles(c, after_rows, err, sms, st);
}

// Rows of int8 at distances of a multiple of 16 bytes, then their scales.
static int64_t quantised_row(int32_t n) { return ((int64_t)n + 15) / 16 * 16; }
size_t linear8_work_bytes(int64_t rows, int32_t n) { return (size_t)rows * (quantised_row(n) + 4) + 16; }

int launch_linear8(const Mm8Call &call, int *err, int sms, cudaStream_t st) {
  Mm8Call c = call;
  if (c.x_dtype != kF16 && c.x_dtype != kF32) return fail("linear8: %s not carried (float16 or float32)", dtype_name(c.x_dtype));
  SHLO_TRY(check_mul_mat8(c, dtype_size(c.x_dtype), "linear8"));
  if (c.rows == 0) return 0;
  int8_t *const q = (int8_t *)c.workspace;
  if (!q || c.workspace_bytes < linear8_work_bytes(c.rows, c.n))
    return fail("linear8: a workspace of %zu bytes, %zu needed", q ? c.workspace_bytes : 0, linear8_work_bytes(c.rows, c.n));
  if ((uintptr_t)q % 16) return fail("linear8: the workspace does not begin on a multiple of 16 bytes");
  if (!c.x) return fail("linear8: null pointer");
  const int64_t need = (int64_t)linear8_work_bytes(c.rows, c.n), x_size = dtype_size(c.x_dtype), y_size = dtype_size(c.dtype);
  auto hits = [&](const void *p, int64_t rows, int64_t step, int64_t bytes) { return meet(q, 1, 0, need, p, rows, step, bytes); };
  if (hits(c.x, c.rows, c.x_row * x_size, c.n * x_size) || hits(c.w, c.m, c.w_row, c.n) || hits(c.w_scale, 1, 0, 4 * (int64_t)c.m) ||
      hits(c.bias, 1, 0, 4 * (int64_t)c.m) || hits(c.y, c.rows, c.y_row * y_size, c.m * y_size))
    return fail("linear8: the workspace shares memory with an operand or the result");
  if ((uintptr_t)c.x % dtype_size(c.x_dtype)) return fail("linear8: an operand is not aligned to its type");
  if (few(c) && few_round(c)) {
    if (c.x_dtype == kF16) return c.dtype == kF16 ? launch_few<__half, __half>(c, false, sms, st) : launch_few<__half, float>(c, false, sms, st);
    return c.dtype == kF16 ? launch_few<float, __half>(c, false, sms, st) : launch_few<float, float>(c, false, sms, st);
  }
  c.x = q;
  c.x_row = quantised_row(c.n);
  c.x_scale = (const float *)(q + c.rows * c.x_row);
  SHLO_TRY(launch_quantise_rows(call.x, call.x_row, c.x_dtype, c.rows, c.n, q, c.x_row, (float *)c.x_scale, false, "linear8", st));
  return launch_mul_mat8(c, true, err, sms, st);
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_quantise_rows_noalloc(const void *x, int64_t x_row, int64_t rows, int32_t n, uint8_t dtype, int8_t *q, int64_t q_row,
                               float *scale, void *stream) {
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_quantise_rows(x, x_row, dtype, rows, n, q, q_row, scale, false, "quantise_rows", (cudaStream_t)stream);
}

int shlo_mul_mat8_noalloc(const shlo_mul_mat8_args *args, void *stream) {
  if (!args) return fail("mul_mat8: null arguments");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  SHLO_TRY(launch_error(dev, "mul_mat8, an earlier call"));
  return launch_mul_mat8(*args, false, dev->pipe_err_dev, dev->sm_count, (cudaStream_t)stream);
}

int shlo_linear8_workspace(int64_t rows, int32_t n, size_t *bytes) {
  if (!bytes) return fail("linear8_workspace: null pointer");
  if (rows < 0 || rows > (1 << 28) || n < 1 || n > 131071) return fail("linear8_workspace: %lld rows of %d values", (long long)rows, n);
  *bytes = linear8_work_bytes(rows, n);
  return 0;
}

int shlo_linear8_noalloc(const shlo_mul_mat8_args *args, void *stream) {
  if (!args) return fail("linear8: null arguments");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  SHLO_TRY(launch_error(dev, "linear8, an earlier call"));
  return launch_linear8(*args, dev->pipe_err_dev, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
