// Rotary positions: every pair (a, b) of a head's first `rot` dimensions turned
// by its token's angle,
//   (a, b) -> f (a cos t - b sin t, b cos t + a sin t),   t = position * frequency,
// the other dimensions copied. Pairs lie half a rotated part apart (i, i + rot/2)
// or side by side (2i, 2i + 1). The gradient is the same with -t.
//
// Angles: a frequency is kept as a phase, the turns it makes per position as a
// 64-bit fraction. position * phase wraps at whole turns, exactly, in integers;
// its upper 32 bits are the signed fraction of a turn, which sincospif takes as a
// binary32 number: 2^-26 turns off at most near half a turn, less nearer 0, and
// the phase's own rounding adds position * 2^-65 (2^-34 at 2^31). A 32-bit product
// of position and frequency would be off by 0.06 rad at position 10^6, and no
// 64-bit float is used.
//
// Bound: bytes (each value read once and written once). A block computes the
// cosines and sines of its tokens once, into shared memory, for all heads.
// Measured on one B200: 16384 tokens x 40 heads x 128, float16 (336 MB) 55.3 us,
// 6.07 TB/s (0.93 of a copy's rate); 24001 x 12 x 80 float32, 32 dimensions turned
// in interleaved pairs (184 MB) 34.4 us, 5.36 TB/s; 16 x 40 x 128 4.1 us, a launch.
#include <cmath>

#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kRopeThreads = 256;

template <int BYTES> struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<2> { using T = uint16_t; };

struct RopeArgs {
  const void *x;
  void *y;
  const int32_t *pos;
  const int64_t *phases;
  int64_t xt, xh, yt, yh;  // token and head strides, in values
  int64_t tokens;
  int heads, dim, rot;
  int tb;          // tokens a block
  int hb;          // heads a block (gridDim.y blocks share a token's heads)
  int copy;        // units of the copied part (0 when x and y are the same storage)
  float factor;
  bool inverse;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, T (&v)[VEC]) {
  using R = typename Raw<VEC * sizeof(T)>::T;
  *reinterpret_cast<R *>(v) = *reinterpret_cast<const R *>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const T (&v)[VEC]) {
  using R = typename Raw<VEC * sizeof(T)>::T;
  *reinterpret_cast<R *>(p) = *reinterpret_cast<const R *>(v);
}
__device__ __forceinline__ float to_f32(__half h) { return __half2float(h); }
__device__ __forceinline__ float to_f32(float f) { return f; }
__device__ __forceinline__ void of_f32(__half &d, float f) { d = __float2half_rn(f); }
__device__ __forceinline__ void of_f32(float &d, float f) { d = f; }

// A unit is VEC pairs (two vectors of x), or one vector of the copied part.
// Shared memory: cos and sin, each [token][part][unit][4] with the unit's VEC
// values in VEC/4 parts, so neighbouring units' 16-byte reads do not conflict.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) k_rope(const RopeArgs a) {
  extern __shared__ float sh[];
  constexpr int PART = VEC >= 4 ? 4 : VEC;  // values a part
  const int half = a.rot / 2, ru = half / VEC, units = ru + a.copy;
  float *const cs = sh, *const sn = sh + a.tb * half;
  const int64_t t0 = (int64_t)blockIdx.x * a.tb;
  const int nt = (int)min((int64_t)a.tb, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int t = i / half, p = i - t * half;
    const int64_t turns = (int64_t)((uint64_t)(int64_t)a.pos[t0 + t] * (uint64_t)a.phases[p]) >> 32;
    float s, c;
    sincospif((float)turns * 0x1p-31f, &s, &c);
    const int u = p / VEC, j = p - u * VEC;
    const int at = t * half + (j / PART) * (ru * PART) + u * PART + j % PART;
    cs[at] = c * a.factor;
    sn[at] = (a.inverse ? -s : s) * a.factor;
  }
  __syncthreads();
  const int h0 = blockIdx.y * a.hb, nh = min(a.hb, a.heads - h0);
  // (token, head, unit) of this thread's items, kRopeThreads apart
  const int dh = kRopeThreads / units, du = kRopeThreads - dh * units;
  int h = threadIdx.x / units, u = threadIdx.x - h * units, t = 0;
  // Several items' loads go out before the first is stored: a block's life is a
  // few waits for memory, not one an item.
  constexpr int AT_ONCE = 3;
  while (t < nt) {
    T v[AT_ONCE][2][VEC];
    T *y[AT_ONCE];
    int tab[AT_ONCE];  // where the unit's cosines begin; -1: copied; -2: nothing
    int o2[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) {
      while (h >= nh) {
        h -= nh;
        t++;
      }
      tab[k] = -2;
      if (t < nt) {
        const T *x = static_cast<const T *>(a.x) + (t0 + t) * a.xt + (h0 + h) * a.xh;
        y[k] = static_cast<T *>(a.y) + (t0 + t) * a.yt + (h0 + h) * a.yh;
        const int o = u < ru ? (INTER ? 2 * VEC : VEC) * u : a.rot + (u - ru) * VEC;
        load_vec<T, VEC>(x + o, v[k][0]);
        y[k] += o;
        tab[k] = -1;
        if (u < ru) {
          tab[k] = t * half + u * PART;
          o2[k] = INTER ? VEC : half;
          load_vec<T, VEC>(x + o + o2[k], v[k][1]);
        }
      }
      u += du;
      h += dh;
      if (u >= units) {
        u -= units;
        h++;
      }
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) {
      if (tab[k] == -2) break;
      if (tab[k] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const int at = tab[k] + (j / PART) * (ru * PART) + j % PART;
          const float c = cs[at], s = sn[at];
          T &lo = INTER ? v[k][(2 * j) / VEC][(2 * j) % VEC] : v[k][0][j];
          T &hi = INTER ? v[k][(2 * j + 1) / VEC][(2 * j + 1) % VEC] : v[k][1][j];
          const float p = to_f32(lo), q = to_f32(hi);
          of_f32(lo, __fmaf_rn(p, c, -(q * s)));
          of_f32(hi, __fmaf_rn(q, c, p * s));
        }
        store_vec<T, VEC>(y[k] + o2[k], v[k][1]);
      }
      store_vec<T, VEC>(y[k], v[k][0]);
    }
  }
}

template <typename T, int VEC>
void launch(const RopeArgs &a, bool inter, dim3 grid, size_t smem, cudaStream_t st) {
  if (inter)
    k_rope<T, VEC, true><<<grid, kRopeThreads, smem, st>>>(a);
  else
    k_rope<T, VEC, false><<<grid, kRopeThreads, smem, st>>>(a);
}

// Whether x and y have a value in common, y not being x itself (blocks then read
// what others have written). Where their extents overlap they need the same
// strides to have none: it comes down to one distance between rows.
bool overlap(const void *x, int64_t x_token, int64_t x_head, const void *y, int64_t y_token, int64_t y_head, int64_t T, int64_t H,
             int64_t D, size_t size) {
  const int64_t off = ((intptr_t)y - (intptr_t)x) / (int64_t)size;
  auto low = [](int64_t n, int64_t s) { return s < 0 ? (double)(n - 1) * s : 0.0; };
  auto high = [](int64_t n, int64_t s) { return s > 0 ? (double)(n - 1) * s : 0.0; };
  const double x0 = low(T, x_token) + low(H, x_head), x1 = high(T, x_token) + high(H, x_head) + D;
  const double y0 = off + low(T, y_token) + low(H, y_head), y1 = off + high(T, y_token) + high(H, y_head) + D;
  if (y1 <= x0 || x1 <= y0) return false;
  if ((T > 1 && x_token != y_token) || (H > 1 && x_head != y_head)) return true;
  const bool by_heads = H <= T;  // the shorter axis is gone through, the other solved for
  const int64_t n1 = by_heads ? H : T, s1 = by_heads ? x_head : x_token;
  const int64_t n2 = by_heads ? T : H, s2 = by_heads ? x_token : x_head;
  for (int64_t i = 1 - n1; i < n1; i++) {
    const int64_t r = off - i * s1, j0 = s2 && n2 > 1 ? r / s2 : 0;
    for (int64_t j = j0 - 1; j <= j0 + 1; j++)
      if (j > -n2 && j < n2 && llabs(r - j * s2) < D) return true;
  }
  return false;
}

}  // namespace

int check_in_place(const void *x, int64_t x_token, int64_t x_head, const void *y, int64_t y_token, int64_t y_head, int64_t tokens,
                   int64_t heads, int64_t dim, size_t size, const char *what, const char *x_name, const char *y_name) {
  const bool same = x == y;
  if (same && (x_token != y_token || x_head != y_head)) return fail("%s: %s and %s share storage with different strides", what, x_name, y_name);
  if (!same && overlap(x, x_token, x_head, y, y_token, y_head, tokens, heads, dim, size))
    return fail("%s: %s and %s overlap (%s is %s itself, or shares no value with it)", what, x_name, y_name, y_name, x_name);
  return 0;
}

int launch_rope(const RopeCall &c, int sms, cudaStream_t st) {
  if (c.dtype != kF16 && c.dtype != kF32) return fail("rope: %s not carried (float16 or float32)", dtype_name(c.dtype));
  if (c.tokens < 0 || c.heads < 1 || c.dim < 1) return fail("rope: %lld tokens, %d heads of %d", (long long)c.tokens, c.heads, c.dim);
  if (c.rot < 0 || c.rot > c.dim || c.rot % 2 || c.rot > 2048)
    return fail("rope: %d of %d dimensions turned (an even number, at most 2048)", c.rot, c.dim);
  if (c.flags & ~3u) return fail("rope: flags 0x%x", c.flags);
  if (c.tokens == 0) return 0;
  if (!c.x || !c.y || (c.rot && (!c.positions || !c.phases))) return fail("rope: null pointer");
  if (c.tokens > 0x7fffffff) return fail("rope: %lld tokens, at most 2^31 - 1", (long long)c.tokens);
  const size_t size = dtype_size(c.dtype);
  if (((uintptr_t)c.x | (uintptr_t)c.y) % size) return fail("rope: x or y is not aligned to its type");
  if ((uintptr_t)c.positions % 4 || (uintptr_t)c.phases % 8) return fail("rope: misaligned positions or phases");
  const bool same = c.x == c.y;
  SHLO_TRY(check_in_place(c.x, c.x_token, c.x_head, c.y, c.y_token, c.y_head, c.tokens, c.heads, c.dim, size, "rope", "x", "y"));
  const int half = c.rot / 2, rest = same ? 0 : c.dim - c.rot;
  if (half == 0 && rest == 0) return 0;
  // The widest vector (16 bytes at most) that every offset is a multiple of.
  int vec = (int)(16 / size);
  const bool strided_h = c.heads > 1, strided_t = c.tokens > 1;
  auto fits = [&](int v) {
    return half % v == 0 && rest % v == 0 && (rest == 0 || c.rot % v == 0) && ((uintptr_t)c.x | (uintptr_t)c.y) % (v * size) == 0 &&
           (!strided_t || (c.x_token % v == 0 && c.y_token % v == 0)) && (!strided_h || (c.x_head % v == 0 && c.y_head % v == 0));
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  RopeArgs a;
  a.x = c.x; a.y = c.y; a.pos = c.positions; a.phases = c.phases;
  a.xt = c.x_token; a.xh = c.x_head; a.yt = c.y_token; a.yh = c.y_head;
  a.tokens = c.tokens; a.heads = c.heads; a.dim = c.dim; a.rot = c.rot;
  a.factor = c.factor; a.inverse = (c.flags & 2) != 0;
  a.copy = rest / vec;
  // A block's tokens: enough for one angle a thread, as long as every SM gets
  // blocks; when tokens are few, a token's heads are shared among blocks.
  a.tb = 1;
  while (a.tb < 8 && a.tb * half < kRopeThreads && c.tokens / (2 * a.tb) >= 4 * sms) a.tb *= 2;
  const int64_t gx = (c.tokens + a.tb - 1) / a.tb;
  const int units = half / vec + a.copy;
  int parts = 1;
  while (gx * parts < 2 * sms && parts < c.heads && (int64_t)units * c.heads / parts > kRopeThreads / 2) parts *= 2;
  a.hb = (c.heads + parts - 1) / parts;
  const dim3 grid((unsigned)gx, (unsigned)((c.heads + a.hb - 1) / a.hb));
  const size_t smem = (size_t)a.tb * half * 2 * sizeof(float);
  const bool inter = (c.flags & 1) != 0;
  if (c.dtype == kF16) {
    switch (vec) {
      case 8: launch<__half, 8>(a, inter, grid, smem, st); break;
      case 4: launch<__half, 4>(a, inter, grid, smem, st); break;
      case 2: launch<__half, 2>(a, inter, grid, smem, st); break;
      default: launch<__half, 1>(a, inter, grid, smem, st); break;
    }
  } else {
    switch (vec) {
      case 4: launch<float, 4>(a, inter, grid, smem, st); break;
      case 2: launch<float, 2>(a, inter, grid, smem, st); break;
      default: launch<float, 1>(a, inter, grid, smem, st); break;
    }
  }
  return launch_check("rope");
}

}  // namespace shlo

using namespace shlo;

extern "C" {

// Frequencies base^(-2i/rot), scaled, as phases: turns a position in units of
// 2^-64 (frequency / 2 pi, rounded).
int shlo_rope_phases(int32_t rot, double base, int32_t scaling, double by, double trained, double fast, double slow,
                     int64_t *phases, float *factor) {
  if (rot < 2 || rot % 2 || rot > 2048) return fail("rope phases: %d dimensions (an even number, 2 to 2048)", rot);
  if (!phases || !factor) return fail("rope phases: null pointer");
  if (!(base > 1.0) || !std::isfinite(base)) return fail("rope phases: base %g (finite, above 1)", base);
  if (scaling < 0 || scaling > 4) return fail("rope phases: scaling %d not carried", scaling);
  if (scaling && (!(by >= 1.0) || !std::isfinite(by))) return fail("rope phases: scaled by %g (at least 1)", by);
  if (scaling >= 3 && !(trained > 0 && fast > slow && slow > 0 && std::isfinite(trained) && std::isfinite(fast)))
    return fail("rope phases: %g trained positions, %g fast and %g slow turns", trained, fast, slow);
  const long double two_pi = 6.283185307179586476925286766559005768L;
  long double b = base;
  // The base raised so that the slowest pair turns `by` times slower.
  if (scaling == 2 && rot > 2) b *= powl((long double)by, (long double)rot / (rot - 2));
  for (int i = 0; i < rot / 2; i++) {
    long double f = powl(b, -2.0L * i / rot);
    if (scaling == 1) f /= by;
    if (scaling == 3) {
      // Pairs that turn at least `fast` times over the trained positions keep
      // their frequency, those under `slow` turns are slowed `by` times; a
      // ramp in the pair's index between the two (bounds rounded outward).
      const long double per = rot / (2.0L * logl((long double)base));
      long double lo = floorl(per * logl(trained / (fast * two_pi))), hi = ceill(per * logl(trained / (slow * two_pi)));
      if (lo < 0) lo = 0;
      if (hi > rot - 1) hi = rot - 1;
      long double width = hi - lo;
      if (width < 1e-3L) width = 1e-3L;
      long double ramp = (i - lo) / width;
      ramp = ramp < 0 ? 0 : ramp > 1 ? 1 : ramp;
      f = f / by * ramp + f * (1 - ramp);
    }
    if (scaling == 4) {
      // The same two ends, blended by the turns themselves.
      const long double turns = trained * f / two_pi;
      long double w = (turns - slow) / ((long double)fast - slow);
      w = w < 0 ? 0 : w > 1 ? 1 : w;
      f = f / by * (1 - w) + f * w;
    }
    phases[i] = (int64_t)llrintl(ldexpl(f / two_pi, 64));
  }
  // The logits' temperature that goes with the ramp.
  *factor = scaling == 3 ? (float)(0.1L * logl((long double)by) + 1.0L) : 1.0f;
  return 0;
}

int shlo_rope_noalloc(const void *x, int64_t x_token, int64_t x_head, const int32_t *positions, const int64_t *phases,
                      void *y, int64_t y_token, int64_t y_head, int64_t tokens, int32_t heads, int32_t dim, int32_t rot,
                      uint8_t dtype, uint32_t flags, float factor, void *stream) {
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  RopeCall c{x, x_token, x_head, positions, phases, y, y_token, y_head, tokens, heads, dim, rot, dtype, flags, factor};
  return launch_rope(c, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
