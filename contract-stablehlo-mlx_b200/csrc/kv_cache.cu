// The paged key/value cache in 8 bits: writing new tokens into it and reading
// tokens back.
//
// A value of page p and head h is q * s, q an int8 in [-127, 127] and s the
// page's and head's own scale (keys and values have one each). A call's new
// values of one page and head give
//   s' = max(s, max|x| (1/127))   (s only where older tokens stay in the page)
//   q  = round(x / s')            (ties to even),
// and where s' > s the older tokens' values are rounded again, round(q s / s').
// Every step is one IEEE binary32 operation, so the cache is the same bits on
// every run; a call made again with the same arguments changes nothing, since
// the scale is by then the larger one. A page that takes a value that is not
// finite gets the scale NaN: what is read from it says so.
//
// Bound: bytes (x read once, int8 written once). A block owns the part of one
// page and head that a call writes, so the maximum needs no atomics: its values
// stay in registers between the two passes (256-token pages of wide heads read
// what does not fit again, from L2). Measured on one B200: 12300 tokens x 8 heads
// x 128 of float16 keys and values (76 MB) into 64-token pages 30 us, 2.5 TB/s:
// three waves of blocks, each a chain of waits (the sequence's place, its table,
// the values) and about 15 instructions a value; one token of each of 48
// sequences 6 us, the chain alone. Reading the same tokens back 20 us.
#include "decode.cuh"

namespace shlo {

int check_pool(const shlo_kv_pool *p, const char *what) {
  if (!p) return fail("%s: null cache", what);
  if (p->heads < 1 || p->heads > 65535) return fail("%s: %d key/value heads (1 to 65535)", what, p->heads);
  if (p->head_dim < 16 || p->head_dim > 256 || p->head_dim % 16)
    return fail("%s: head width %d not carried (multiples of 16 up to 256)", what, p->head_dim);
  const int t = p->page_tokens;
  if (t < 16 || t > 256 || (t & (t - 1))) return fail("%s: %d tokens a page not carried (16, 32, 64, 128, 256)", what, t);
  if (p->pages < 0 || p->pages > 0x7fffffff) return fail("%s: %lld pages (at most 2^31 - 1)", what, (long long)p->pages);
  if (p->pages && (!p->k || !p->v || !p->k_scale || !p->v_scale)) return fail("%s: null pointer in the cache", what);
  // Rows are read and written 16 bytes at a time.
  if (((uintptr_t)p->k | (uintptr_t)p->v) % 16 || p->page_stride % 16 || p->head_stride % 16 || p->token_stride % 16)
    return fail("%s: the cache's pointers and strides are multiples of 16 bytes", what);
  if (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) % 4) return fail("%s: misaligned scales", what);
  return 0;
}

int check_batch(const shlo_kv_batch *b, const char *what) {
  if (!b) return fail("%s: null batch", what);
  if (b->seqs < 0 || b->tokens < 0 || b->table_pages < 0)
    return fail("%s: %d sequences, %d tokens, tables of %d pages", what, b->seqs, b->tokens, b->table_pages);
  if (b->seqs > (1 << 20) || b->tokens > (1 << 28)) return fail("%s: %d sequences (at most 2^20), %d tokens (at most 2^28)", what, b->seqs, b->tokens);
  if (b->seqs && (!b->starts || !b->lens || (b->table_pages && !b->tables))) return fail("%s: null pointer in the batch", what);
  if (((uintptr_t)b->starts | (uintptr_t)b->lens | (uintptr_t)b->tables) % 4) return fail("%s: misaligned starts, lens or tables", what);
  if (b->table_pages > (1 << 22)) return fail("%s: tables of %d pages (at most 2^22)", what, b->table_pages);
  return 0;
}

namespace {

constexpr int kAppendThreads = 128;
constexpr int kKeep = 4;  // 16-value pieces a thread keeps between the passes

struct AppendArgs {
  shlo_kv_pool pool;
  shlo_kv_batch batch;
  const void *x[2];
  int64_t xt[2], xh[2];
};

// 16 values of x as they come (WIDE: every offset allows 16-byte loads), kept so
// between the passes: half the registers of floats for float16.
template <typename T>
struct Raw16 {
  uint4 w[sizeof(T)];
};
template <typename T, bool WIDE>
__device__ __forceinline__ void load16(const T *p, Raw16<T> &r) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); i++) r.w[i] = *(reinterpret_cast<const uint4 *>(p) + i);
  } else {
    T v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = p[i];
    memcpy(&r, v, sizeof r);
  }
}
template <typename T>
__device__ __forceinline__ void floats16(const Raw16<T> &r, float (&f)[16]) {
  T v[16];
  memcpy(v, &r, sizeof r);
#pragma unroll
  for (int i = 0; i < 16; i++) f[i] = (float)v[i];
}

// Sixteen values as round(x / s), the quotient rounded to binary32 first. x times
// the reciprocal is within 2^-21 of the quotient relative (2^-14 at 127); away
// from a tie it rounds to the same integer, near one the division decides for
// the piece. Rounding is an add of 1.5 2^23, whose low byte then is the integer's:
// conversions would run at a quarter of the rate.
__device__ __forceinline__ uint4 pack16(const float (&f)[16], float s) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  // s = 0: every value of the page is 0. s NaN: the page reads as NaN.
  if (s > 0.0f) {
    const float inv = __fdiv_rn(1.0f, s);  // (not a normal number for the smallest and largest s: the division decides)
    float off = 0.0f;                      // the farthest from its integer
    uint32_t q[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float r = f[i] * inv, m = r + 12582912.0f;
      off = fmaxf(off, fabsf(r - (m - 12582912.0f)));
      q[i] = __float_as_uint(m);
    }
    if (!(off < 0.5f - 0x1p-12f) || !(s > 0x1p-120f && s < 0x1p120f)) {
#pragma unroll
      for (int i = 0; i < 16; i++) q[i] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(f[i], s)), -127.0f), 127.0f);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest magnitude of a piece's values as bits that order like it: above
// infinity's where one is not a number.
template <typename T>
__device__ __forceinline__ uint32_t top16(const Raw16<T> &r) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = __vmaxu2(m, (&r.w[i / 4].x)[i % 4] & 0x7fff7fffu);
    const uint32_t h = max(m & 0xffffu, m >> 16);
    return h >= 0x7c00u ? 0x7f800000u : __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, (&r.w[i / 4].x)[i % 4] & 0x7fffffffu);
    return m;
  }
}

// One block: the pages that a call writes are numbered in slots (a sequence of
// n new tokens touches at most n / page + 2), blockIdx.y the head, z keys or
// values.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(const AppendArgs a) {
  const shlo_kv_pool &pool = a.pool;
  const int PT = pool.page_tokens, sh = 31 - __clz(PT), slot = blockIdx.x, h = blockIdx.y, z = blockIdx.z;
  const int b = slot_owner(a.batch.starts, a.batch.tokens, a.batch.seqs, 0, slot, 1, sh, 2);
  const SeqSpan sp = seq_span(a.batch.starts, a.batch.lens, a.batch.tokens, b);
  const int slot0 = slot_base(a.batch.starts, a.batch.tokens, b, 1, sh, 2);
  const int first = sp.len - sp.n;  // the first new token's position
  const int from = max(first, 0);
  const int page_of = (from >> sh) + (slot - slot0);
  if (slot < slot0 || page_of >= a.batch.table_pages) return;
  const int p0 = max(page_of * PT, from), p1 = min((page_of + 1) * PT, sp.len);  // its new positions
  if (p0 >= p1) return;
  const int page = __ldg(a.batch.tables + (int64_t)b * a.batch.table_stride + page_of);
  if (page < 0 || page >= pool.pages) return;
  const int pieces = pool.head_dim / 16, items = (p1 - p0) * pieces;
  const T *x = static_cast<const T *>(a.x[z]) + (int64_t)(sp.start + p0 - first) * a.xt[z] + h * a.xh[z];
  int8_t *dst = (z ? pool.v : pool.k) + (int64_t)page * pool.page_stride + (int64_t)h * pool.head_stride;
  float *scale = (z ? pool.v_scale : pool.k_scale) + (int64_t)page * pool.scale_page_stride + (int64_t)h * pool.scale_head_stride;
  const int old_n = p0 - page_of * PT;  // older tokens that stay in the page

  Raw16<T> keep[kKeep];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kKeep; k++) {
    const int i = threadIdx.x + k * kAppendThreads;
    if (i < items) load16<T, WIDE>(x + (int64_t)(i / pieces) * a.xt[z] + (i % pieces) * 16, keep[k]);
  }
#pragma unroll
  for (int k = 0; k < kKeep; k++)
    if ((int)threadIdx.x + k * kAppendThreads < items) top = max(top, top16(keep[k]));
  for (int i = threadIdx.x + kKeep * kAppendThreads; i < items; i += kAppendThreads) {
    Raw16<T> r;
    load16<T, WIDE>(x + (int64_t)(i / pieces) * a.xt[z] + (i % pieces) * 16, r);
    top = max(top, top16(r));
  }
  __shared__ uint32_t red[kAppendThreads / 32];
  const float old_s = old_n ? *scale : 0.0f;
  top = __reduce_max_sync(~0u, top);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = top;
  __syncthreads();  // every thread has read the old scale by now
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; w++) top = max(top, red[w]);
  const bool bad = top >= 0x7f800000u;
  const float most = __uint_as_float(top);
  float s = __fmul_rn(most, 1.0f / 127.0f);
  if (old_n) s = old_s > s || old_s != old_s ? old_s : s;
  if (bad) s = __int_as_float(0x7fc00000);
  if (threadIdx.x == 0) *scale = s;
  if (old_n && s != old_s && s == s) {
    const float ratio = s > 0.0f ? __fdiv_rn(old_s, s) : 0.0f;
    for (int i = threadIdx.x; i < old_n * pieces; i += kAppendThreads) {
      uint4 *p = reinterpret_cast<uint4 *>(dst + (int64_t)(i / pieces) * pool.token_stride + (i % pieces) * 16);
      uint4 r = *p;
      uint32_t *w = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t o = 0;
#pragma unroll
        for (int l = 0; l < 4; l++) {
          const float q = (float)(int8_t)(w[j] >> (8 * l));
          o |= ((uint32_t)(int)rintf(__fmul_rn(q, ratio)) & 0xffu) << (8 * l);
        }
        w[j] = o;
      }
      *p = r;
    }
  }
  auto put = [&](int i, const Raw16<T> &r) {
    float f[16];
    floats16(r, f);
    *reinterpret_cast<uint4 *>(dst + (int64_t)(old_n + i / pieces) * pool.token_stride + (i % pieces) * 16) = pack16(f, s);
  };
#pragma unroll
  for (int k = 0; k < kKeep; k++) {
    const int i = threadIdx.x + k * kAppendThreads;
    if (i < items) put(i, keep[k]);
  }
  for (int i = threadIdx.x + kKeep * kAppendThreads; i < items; i += kAppendThreads) {
    Raw16<T> r;
    load16<T, WIDE>(x + (int64_t)(i / pieces) * a.xt[z] + (i % pieces) * 16, r);
    put(i, r);
  }
}

struct GatherArgs {
  shlo_kv_pool pool;
  const int32_t *tables, *seq, *pos;
  int64_t table_stride;
  int32_t seqs, table_pages;
  int64_t n;
  void *y[2];
  int64_t yt[2], yh[2];
};

// A warp reads one token, keys and values, V values a lane and step (16 bytes of
// output), four steps' loads on their way: the waits for the token's place and
// page come once a token, not once a value.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_kv_gather(const GatherArgs a) {
  const shlo_kv_pool &pool = a.pool;
  const int pieces = pool.head_dim / V, items = 2 * pieces * pool.heads, lane = threadIdx.x % 32;
  for (int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; row < a.n; row += (int64_t)gridDim.x * 8) {
    const int s = __ldg(a.seq + row), at = __ldg(a.pos + row);
    int page = -1;  // (a token that the tables do not hold reads as zeros)
    if (s >= 0 && s < a.seqs && at >= 0 && at / pool.page_tokens < a.table_pages)
      page = __ldg(a.tables + (int64_t)s * a.table_stride + at / pool.page_tokens);
    const bool there = page >= 0 && page < pool.pages;
    const int64_t base = (int64_t)page * pool.page_stride + (int64_t)(at % pool.page_tokens) * pool.token_stride;
    for (int i0 = lane; i0 < items; i0 += 4 * 32) {
      uint2 q[4];
      float sc[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = i0 + k * 32, z = i >= items / 2, j = i - z * (items / 2), h = j / pieces, d = (j - h * pieces) * V;
        q[k] = make_uint2(0u, 0u);
        sc[k] = 0.0f;
        if (there && i < items) {
          const int8_t *p = (z ? pool.v : pool.k) + base + (int64_t)h * pool.head_stride + d;
          if constexpr (V == 8) q[k] = __ldg(reinterpret_cast<const uint2 *>(p));
          else q[k].x = __ldg(reinterpret_cast<const uint32_t *>(p));
          sc[k] = __ldg((z ? pool.v_scale : pool.k_scale) + (int64_t)page * pool.scale_page_stride + (int64_t)h * pool.scale_head_stride);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = i0 + k * 32, z = i >= items / 2, j = i - z * (items / 2), h = j / pieces, d = (j - h * pieces) * V;
        if (i >= items) break;
        T y[V];
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float f = (float)(int8_t)((e < 4 ? q[k].x : q[k].y) >> (8 * (e % 4))) * sc[k];
          if constexpr (sizeof(T) == 2) y[e] = __float2half_rn(f);
          else y[e] = f;
        }
        uint4 w;
        memcpy(&w, y, 16);
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.y[z]) + row * a.yt[z] + (int64_t)h * a.yh[z] + d) = w;
      }
    }
  }
}

}  // namespace

static int check_type(uint8_t dtype, const char *what) {
  if (dtype != kF16 && dtype != kF32) return fail("%s: %s not carried (float16 or float32)", what, dtype_name(dtype));
  return 0;
}

int launch_kv_append(const shlo_kv_pool &p, const shlo_kv_batch &b, const void *k, int64_t k_token, int64_t k_head,
                     const void *v, int64_t v_token, int64_t v_head, uint8_t dtype, cudaStream_t st) {
  SHLO_TRY(check_pool(&p, "kv_append"));
  SHLO_TRY(check_batch(&b, "kv_append"));
  SHLO_TRY(check_type(dtype, "kv_append"));
  if (b.seqs == 0 || b.tokens == 0 || p.pages == 0) return 0;
  if (!k || !v) return fail("kv_append: null pointer");
  const size_t size = dtype_size(dtype);
  if (((uintptr_t)k | (uintptr_t)v) % size) return fail("kv_append: k or v is not aligned to its type");
  AppendArgs a;
  a.pool = p;
  a.batch = b;
  a.x[0] = k; a.xt[0] = k_token; a.xh[0] = k_head;
  a.x[1] = v; a.xt[1] = v_token; a.xh[1] = v_head;
  const int64_t per16 = (int64_t)(16 / size);
  const bool wide = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_token % per16 == 0 && k_head % per16 == 0 &&
                    v_token % per16 == 0 && v_head % per16 == 0;
  const dim3 grid((unsigned)(b.tokens / p.page_tokens + 2 * b.seqs), (unsigned)p.heads, 2);
  if (dtype == kF16) {
    if (wide) k_kv_append<__half, true><<<grid, kAppendThreads, 0, st>>>(a);
    else k_kv_append<__half, false><<<grid, kAppendThreads, 0, st>>>(a);
  } else {
    if (wide) k_kv_append<float, true><<<grid, kAppendThreads, 0, st>>>(a);
    else k_kv_append<float, false><<<grid, kAppendThreads, 0, st>>>(a);
  }
  return launch_check("kv_append");
}

int launch_kv_gather(const shlo_kv_pool &p, const int32_t *tables, int64_t table_stride, int32_t seqs,
                     int32_t table_pages, const int32_t *seq, const int32_t *pos, int64_t n, void *k, int64_t k_token,
                     int64_t k_head, void *v, int64_t v_token, int64_t v_head, uint8_t dtype, int sms, cudaStream_t st) {
  SHLO_TRY(check_pool(&p, "kv_gather"));
  SHLO_TRY(check_type(dtype, "kv_gather"));
  if (n < 0 || seqs < 0 || table_pages < 0) return fail("kv_gather: %lld tokens of %d sequences", (long long)n, seqs);
  if (n == 0) return 0;
  if (!seq || !pos || !k || !v || (seqs && table_pages && !tables)) return fail("kv_gather: null pointer");
  if (((uintptr_t)seq | (uintptr_t)pos | (uintptr_t)tables) % 4) return fail("kv_gather: misaligned tables, seq or pos");
  const int64_t per16 = (int64_t)(16 / dtype_size(dtype));
  if (((uintptr_t)k | (uintptr_t)v) % 16 || k_token % per16 || k_head % per16 || v_token % per16 || v_head % per16)
    return fail("kv_gather: the outputs' pointers and strides are multiples of 16 bytes");
  GatherArgs a;
  a.pool = p;
  a.tables = tables; a.seq = seq; a.pos = pos;
  a.table_stride = table_stride;
  a.seqs = p.pages ? seqs : 0;
  a.table_pages = table_pages;
  a.n = n;
  a.y[0] = k; a.yt[0] = k_token; a.yh[0] = k_head;
  a.y[1] = v; a.yt[1] = v_token; a.yh[1] = v_head;
  const int64_t want = (n + 7) / 8, cap = (int64_t)sms * 8;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (dtype == kF16) k_kv_gather<__half, 8><<<grid, 256, 0, st>>>(a);
  else k_kv_gather<float, 4><<<grid, 256, 0, st>>>(a);
  return launch_check("kv_gather");
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_kv_append_noalloc(const shlo_kv_pool *pool, const shlo_kv_batch *batch, const void *k, int64_t k_token,
                           int64_t k_head, const void *v, int64_t v_token, int64_t v_head, uint8_t dtype, void *stream) {
  if (!pool || !batch) return fail("kv_append: null descriptor");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_kv_append(*pool, *batch, k, k_token, k_head, v, v_token, v_head, dtype, (cudaStream_t)stream);
}

int shlo_kv_gather_noalloc(const shlo_kv_pool *pool, const int32_t *tables, int64_t table_stride, int32_t seqs,
                           int32_t table_pages, const int32_t *seq, const int32_t *pos, int64_t n, void *k,
                           int64_t k_token, int64_t k_head, void *v, int64_t v_token, int64_t v_head, uint8_t dtype,
                           void *stream) {
  if (!pool) return fail("kv_gather: null descriptor");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_kv_gather(*pool, tables, table_stride, seqs, table_pages, seq, pos, n, k, k_token, k_head, v, v_token,
                          v_head, dtype, dev->sm_count, (cudaStream_t)stream);
}

}  // extern "C"
