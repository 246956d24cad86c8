// Products of activations and weights in 8-bit integers.
//   rows:    q[i] = the whole number nearest to 127 x[i] / top (of two, the even
//            one), scale = top / 127, where top is the row's largest magnitude;
//            a row of zeros has scale 0, one with a value that is not finite
//            zeros and scale NaN.
//   product: y[r][c] = (sum over i of q[r][i] w[c][i]) scale[r] w_scale[c] + bias[c],
//            the sum in 32-bit integers, exact for up to 131071 terms; then four
//            roundings (to binary32, two products, the bias) and the result's own.
#include <algorithm>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kQuantThreads = 256;

__device__ __forceinline__ float to_f32(__half h) { return __half2float(h); }
__device__ __forceinline__ float to_f32(float f) { return f; }

// 127 x / top rounded: exact in 64 bits (x and top have 24 bits, so the quotient is
// never nearer to half a step than 2^-33 of it without being there), and needed
// there only where 32 bits leave it open. Those are off by less than 2^-15.
__device__ __forceinline__ int quantise(float x, float top, float by) {
  const float t = x * by, k = rintf(t);
  if (fabsf(fabsf(t - k) - 0.5f) > 0x1p-14f) return (int)k;
  return (int)rint((double)x * 127.0 / (double)top);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantThreads) k_quantise_rows(const T *x, int64_t x_row, int n, int8_t *q, int64_t q_row, float *scale, int fill) {
  __shared__ uint32_t tops[kQuantThreads / 32];
  const int64_t row = blockIdx.x;
  x += row * x_row;
  q += row * q_row;
  // (as bits, the magnitudes of values that are not finite are the largest)
  uint32_t top_bits = 0;
  const int vecs = n / VEC;
  for (int i = threadIdx.x; i < vecs; i += kQuantThreads) {
    T v[VEC];
    if (VEC * sizeof(T) == 16) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(x + i * VEC);
    else v[0] = x[i];
#pragma unroll
    for (int j = 0; j < VEC; j++) top_bits = max(top_bits, __float_as_uint(fabsf(to_f32(v[j]))));
  }
  if (VEC > 1)
    for (int i = vecs * VEC + threadIdx.x; i < n; i += kQuantThreads) top_bits = max(top_bits, __float_as_uint(fabsf(to_f32(x[i]))));
  top_bits = __reduce_max_sync(~0u, top_bits);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top_bits;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; i++) top_bits = max(top_bits, tops[i]);
  const float top = __uint_as_float(top_bits);
  const bool finite = top_bits < 0x7f800000u, any = finite && top_bits > 0;
  if (threadIdx.x == 0) scale[row] = finite ? top / 127.0f : __uint_as_float(0x7fc00000u);
  const float by = 127.0f / top;
  for (int i = threadIdx.x; i < n; i += kQuantThreads) q[i] = any ? (int8_t)quantise(to_f32(x[i]), top, by) : 0;
  for (int i = n + threadIdx.x; i < fill; i += kQuantThreads) q[i] = 0;
}

}  // namespace

int launch_quantise_rows(const void *x, int64_t x_row, uint8_t dtype, int64_t rows, int32_t n, int8_t *q, int64_t q_row, float *scale,
                         bool fill, const char *what, cudaStream_t st) {
  if (dtype != kF16 && dtype != kF32) return fail("%s: %s not carried (float16 or float32)", what, dtype_name(dtype));
  if (rows < 0 || rows > 0x7fffffff || n < 1) return fail("%s: %lld rows of %d values", what, (long long)rows, n);
  if (rows == 0) return 0;
  if (!x || !q || !scale) return fail("%s: null pointer", what);
  const size_t size = dtype_size(dtype);
  if ((uintptr_t)x % size || (uintptr_t)scale % 4) return fail("%s: an operand is not aligned to its type", what);
  const bool wide = (uintptr_t)x % 16 == 0 && (rows == 1 || x_row * (int64_t)size % 16 == 0);
  const int end = fill ? (n + 15) / 16 * 16 : n;
  const unsigned grid = (unsigned)rows;
  if (dtype == kF16) {
    const __half *p = (const __half *)x;
    if (wide) k_quantise_rows<__half, 8><<<grid, kQuantThreads, 0, st>>>(p, x_row, n, q, q_row, scale, end);
    else k_quantise_rows<__half, 1><<<grid, kQuantThreads, 0, st>>>(p, x_row, n, q, q_row, scale, end);
  } else {
    const float *p = (const float *)x;
    if (wide) k_quantise_rows<float, 4><<<grid, kQuantThreads, 0, st>>>(p, x_row, n, q, q_row, scale, end);
    else k_quantise_rows<float, 1><<<grid, kQuantThreads, 0, st>>>(p, x_row, n, q, q_row, scale, end);
  }
  return launch_check(what);
}

// What x does not enter into: the weights, the result and the sizes.
static int check_mul_mat8(const Mm8Call &c, const char *what) {
  if (c.dtype != kF16 && c.dtype != kF32) return fail("%s: a result of %s not carried (float16 or float32)", what, dtype_name(c.dtype));
  if (c.rows < 0 || c.rows > (1 << 28) || c.m < 1 || c.n < 1 || c.n > 131071)
    return fail("%s: %lld rows, %d channels of %d values (32-bit sums hold 131071)", what, (long long)c.rows, c.m, c.n);
  if (c.rows == 0) return 0;
  if (!c.w || !c.w_scale || !c.y) return fail("%s: null pointer", what);
  if ((uintptr_t)c.w % 16 || (c.m > 1 && (c.w_row % 16 || c.w_row < c.n)))
    return fail("%s: rows of w begin on multiples of 16 bytes and do not overlap (a distance of %lld for %d values)", what, (long long)c.w_row, c.n);
  if ((uintptr_t)c.w_scale % 4 || (uintptr_t)c.bias % 4 || (uintptr_t)c.y % dtype_size(c.dtype)) return fail("%s: an operand is not aligned to its type", what);
  return 0;
}

int launch_mul_mat8(const Mm8Call &c, int sms, cudaStream_t st) {
  SHLO_TRY(check_mul_mat8(c, "mul_mat8"));
  if (c.rows == 0) return 0;
  if (!c.x || !c.x_scale) return fail("mul_mat8: null pointer");
  if ((uintptr_t)c.x % 16 || (c.rows > 1 && (c.x_row % 16 || c.x_row < c.n)))
    return fail("mul_mat8: rows of x begin on multiples of 16 bytes and do not overlap (a distance of %lld for %d values)", (long long)c.x_row, c.n);
  if ((uintptr_t)c.x_scale % 4) return fail("mul_mat8: an operand is not aligned to its type");
  return launch_mul_mat8_tiles(c, sms, st);
}

// Rows of int8 at distances of a multiple of 16 bytes, then their scales.
static int64_t quantised_row(int32_t n) { return ((int64_t)n + 15) / 16 * 16; }
size_t linear8_work_bytes(int64_t rows, int32_t n) { return (size_t)rows * (quantised_row(n) + 4) + 16; }

int launch_linear8(const Mm8Call &call, const void *x, int64_t x_row, uint8_t x_dtype, void *work, size_t work_bytes, int sms, cudaStream_t st) {
  Mm8Call c = call;
  SHLO_TRY(check_mul_mat8(c, "linear8"));
  if (x_dtype != kF16 && x_dtype != kF32) return fail("linear8: %s not carried (float16 or float32)", dtype_name(x_dtype));
  if (c.rows == 0) return 0;
  if (!work || work_bytes < linear8_work_bytes(c.rows, c.n))
    return fail("linear8: a workspace of %zu bytes, %zu needed", work ? work_bytes : 0, linear8_work_bytes(c.rows, c.n));
  if ((uintptr_t)work % 16) return fail("linear8: the workspace does not begin on a multiple of 16 bytes");
  c.x_row = quantised_row(c.n);
  c.x = (const int8_t *)work;
  c.x_scale = (const float *)((const int8_t *)work + c.rows * c.x_row);
  SHLO_TRY(launch_quantise_rows(x, x_row, x_dtype, c.rows, c.n, (int8_t *)work, c.x_row, (float *)c.x_scale, false, "linear8", st));
  return launch_mul_mat8(c, sms, st);
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

int shlo_mul_mat8_noalloc(const int8_t *x, int64_t x_row, const float *x_scale, const int8_t *w, int64_t w_row, const float *w_scale,
                          const float *bias, void *y, int64_t y_row, int64_t rows, int32_t n, int32_t m, uint8_t dtype, void *stream) {
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  SHLO_TRY(launch_error(dev, "mul_mat8, an earlier call"));
  Mm8Call c{x, x_row, x_scale, w, w_row, w_scale, bias, y, y_row, rows, n, m, dtype, dev->pipe_err_dev};
  return launch_mul_mat8(c, dev->sm_count, (cudaStream_t)stream);
}

int shlo_linear8_workspace(int64_t rows, int32_t n, size_t *bytes) {
  if (!bytes) return fail("linear8_workspace: null pointer");
  if (rows < 0 || rows > (1 << 28) || n < 1 || n > 131071) return fail("linear8_workspace: %lld rows of %d values", (long long)rows, n);
  *bytes = linear8_work_bytes(rows, n);
  return 0;
}

int shlo_linear8_noalloc(const void *x, int64_t x_row, uint8_t x_dtype, const int8_t *w, int64_t w_row, const float *w_scale,
                         const float *bias, void *y, int64_t y_row, int64_t rows, int32_t n, int32_t m, uint8_t y_dtype,
                         void *workspace, size_t workspace_bytes, void *stream) {
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  SHLO_TRY(launch_error(dev, "linear8, an earlier call"));
  Mm8Call c{nullptr, 0, nullptr, w, w_row, w_scale, bias, y, y_row, rows, n, m, y_dtype, dev->pipe_err_dev};
  return launch_linear8(c, x, x_row, x_dtype, workspace, workspace_bytes, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
