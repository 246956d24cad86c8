// The decoder operators on arrays: the "shlo_rope" kernel, and caches whose
// storage the library owns. A cache is changed in place, which arrays never
// are: it is a handle of its own, and compiled functions, whose replays work on
// private copies, do not take it.
#include "decode.cuh"

namespace shlo {

// "shlo_rope": x [T][H][D], positions int32 [T], phases int64 [rot / 2],
// p = [T, H, D, rot, flags, factor bits]; the result is of x's type.
int k_rope(Device *dev, Arr *x, Arr *positions, Arr *phases, const uint32_t *p, Arr **out) {
  const int64_t T = p[0], H = p[1], D = p[2], rot = p[3];
  if (positions->dtype != kI32) return fail("shlo_rope: positions of %s, int32 expected", dtype_name(positions->dtype));
  if (phases->dtype != kI64) return fail("shlo_rope: phases of %s, int64 expected", dtype_name(phases->dtype));
  // (products within 64 bits: the words are the caller's)
  if (H < 1 || D < 1 || T > 0x7fffffff || H > 0x7fffffff || D > 0x7fffffff || T * H > ((int64_t)1 << 40) / D)
    return fail("shlo_rope: %lld tokens of %lld heads of %lld", (long long)T, (long long)H, (long long)D);
  if (numel(x) != T * H * D || numel(positions) != T || numel(phases) < rot / 2)
    return fail("shlo_rope: %lld values, %lld positions and %lld phases for [%lld, %lld, %lld] and %lld dimensions turned",
                (long long)numel(x), (long long)numel(positions), (long long)numel(phases), (long long)T, (long long)H,
                (long long)D, (long long)rot);
  const int64_t shape[3] = {T, H, D};
  Arr *o;
  SHLO_TRY(new_array(dev, x->dtype, shape, 3, &o));
  RopeCall c{data_ptr(x), H * D, D, (const int32_t *)data_ptr(positions), (const int64_t *)data_ptr(phases), data_ptr(o), H * D, D,
             T, (int32_t)H, (int32_t)D, (int32_t)rot, x->dtype, p[4], bitsf_host(p[5])};
  if (launch_rope(c, dev->sm_count, dev->stream)) {
    shlo_release(o);
    return 1;
  }
  *out = o;
  return 0;
}

namespace {

// The attention's workspace, one a device: all of a device's work is on its stream.
std::mutex g_work_mu;
Buffer *g_work[64];

int workspace(Device *dev, Buffer **out) {
  std::lock_guard<std::mutex> lk(g_work_mu);
  if (!g_work[dev->id]) {
    Buffer *b;
    const size_t bytes = attend_work_bytes(dev->sm_count);
    SHLO_TRY(buffer_alloc(dev, bytes, &b));
    if (cuda_check(cudaMemsetAsync(b->ptr, 0, bytes, dev->stream), "kv_attend: workspace")) {
      buffer_release(b);
      return 1;
    }
    g_work[dev->id] = b;
  }
  *out = g_work[dev->id];
  return 0;
}

}  // namespace

}  // namespace shlo

using namespace shlo;

struct shlo_kv_s {
  Device *dev = nullptr;
  Buffer *buf[4] = {nullptr, nullptr, nullptr, nullptr};  // k, v, their scales
  shlo_kv_pool pool = {};
  ~shlo_kv_s() {
    for (Buffer *b : buf) buffer_release(b);
  }
};

namespace {

// References that are dropped at the end of a call.
struct Held {
  std::vector<Arr *> arrays;
  ~Held() {
    for (Arr *a : arrays) shlo_release(a);
  }
};

int usable(shlo_kv kv, const char *what) {
  if (!kv) return fail("%s: null cache", what);
  Device *dev;
  SHLO_TRY(device_by_id(kv->dev->id, &dev));
  if (dev->capturing || t_tracer)
    return fail("%s: a cache changes in place and is not carried inside a compiled function", what);
  return 0;
}

int on_device(shlo_kv kv, Arr *a, const char *what, const char *name) {
  if (!a) return fail("%s: %s is null", what, name);
  if (numel(a) && (!a->buf || a->buf->dev != kv->dev)) return fail("%s: %s is not on the cache's device", what, name);
  return 0;
}

// [tokens][heads][dim] activations of float16 or float32, read in place where a
// head's values are contiguous.
int rows_of(shlo_kv kv, Arr *a, const char *what, const char *name, Held &held, Arr **out) {
  SHLO_TRY(on_device(kv, a, what, name));
  if (a->ndim != 3 || a->shape[2] != kv->pool.head_dim)
    return fail("%s: %s is not [tokens, heads, %d]", what, name, kv->pool.head_dim);
  if (a->dtype != kF16 && a->dtype != kF32) return fail("%s: %s of %s not carried (float16 or float32)", what, name, dtype_name(a->dtype));
  if (a->strides[2] == 1) {
    *out = a;
    return 0;
  }
  SHLO_TRY(make_contiguous(a, out));
  held.arrays.push_back(*out);
  return 0;
}

int ints_of(shlo_kv kv, Arr *a, int ndim, const char *what, const char *name, Held &held, Arr **out) {
  SHLO_TRY(on_device(kv, a, what, name));
  if (a->ndim != ndim || a->dtype != kI32)
    return fail("%s: %s is %s of rank %d, int32 of rank %d expected", what, name, dtype_name(a->dtype), a->ndim, ndim);
  SHLO_TRY(make_contiguous(a, out));
  held.arrays.push_back(*out);
  return 0;
}

int batch_of(shlo_kv kv, Arr *starts, Arr *lens, Arr *tables, int64_t tokens, const char *what, Held &held, shlo_kv_batch *b) {
  Arr *s, *l, *t;
  SHLO_TRY(ints_of(kv, starts, 1, what, "starts", held, &s));
  SHLO_TRY(ints_of(kv, lens, 1, what, "lens", held, &l));
  SHLO_TRY(ints_of(kv, tables, 2, what, "tables", held, &t));
  const int64_t n = t->shape[0];
  if (s->shape[0] != n + 1 || l->shape[0] != n)
    return fail("%s: %lld starts and %lld lengths for tables of %lld sequences", what, (long long)s->shape[0], (long long)l->shape[0], (long long)n);
  if (n > (1 << 20) || t->shape[1] > (1 << 22) || tokens > (1 << 28))
    return fail("%s: %lld sequences, tables of %lld pages, %lld tokens", what, (long long)n, (long long)t->shape[1], (long long)tokens);
  b->starts = (const int32_t *)data_ptr(s);
  b->lens = (const int32_t *)data_ptr(l);
  b->tables = (const int32_t *)data_ptr(t);
  b->table_stride = t->shape[1];
  b->seqs = (int32_t)n;
  b->table_pages = (int32_t)t->shape[1];
  b->tokens = (int32_t)tokens;
  return 0;
}

}  // namespace

extern "C" {

int shlo_kv_new(int64_t pages, int32_t heads, int32_t head_dim, int32_t page_tokens, shlo_kv *out) {
  if (!out) return fail("kv_new: null pointer");
  shlo_kv_pool p = {};
  p.heads = heads;
  p.head_dim = head_dim;
  p.page_tokens = page_tokens;
  SHLO_TRY(check_pool(&p, "kv_new"));
  if (pages < 1 || pages > 0x7fffffff) return fail("kv_new: %lld pages (1 to 2^31 - 1)", (long long)pages);
  Device *dev;
  SHLO_TRY(current_device(&dev));
  if (dev->capturing || t_tracer) return fail("kv_new: a cache is not carried inside a compiled function");
  p.pages = pages;
  p.token_stride = head_dim;
  p.head_stride = (int64_t)page_tokens * head_dim;
  p.page_stride = heads * p.head_stride;
  p.scale_page_stride = heads;
  p.scale_head_stride = 1;
  std::unique_ptr<shlo_kv_s> kv(new shlo_kv_s());
  kv->dev = dev;
  for (int i = 0; i < 4; i++) {
    const size_t bytes = i < 2 ? (size_t)pages * p.page_stride : (size_t)pages * heads * sizeof(float);
    SHLO_TRY(buffer_alloc(dev, bytes, &kv->buf[i]));
    SHLO_CUDA(cudaMemsetAsync(kv->buf[i]->ptr, 0, bytes, dev->stream));
  }
  p.k = (int8_t *)kv->buf[0]->ptr;
  p.v = (int8_t *)kv->buf[1]->ptr;
  p.k_scale = (float *)kv->buf[2]->ptr;
  p.v_scale = (float *)kv->buf[3]->ptr;
  kv->pool = p;
  *out = kv.release();
  return 0;
}

void shlo_kv_free(shlo_kv kv) { delete kv; }

int shlo_kv_storage(shlo_kv kv, shlo_kv_pool *pool) {
  if (!kv || !pool) return fail("kv_storage: null pointer");
  *pool = kv->pool;
  return 0;
}

int shlo_kv_append(shlo_kv kv, shlo_arr k, shlo_arr v, shlo_arr starts, shlo_arr lens, shlo_arr tables) {
  SHLO_TRY(usable(kv, "kv_append"));
  Held held;
  Arr *ka, *va;
  SHLO_TRY(rows_of(kv, k, "kv_append", "k", held, &ka));
  SHLO_TRY(rows_of(kv, v, "kv_append", "v", held, &va));
  if (ka->dtype != va->dtype || ka->shape[0] != va->shape[0] || ka->shape[1] != kv->pool.heads || va->shape[1] != kv->pool.heads)
    return fail("kv_append: k and v are not [tokens, %d, %d] of one type", kv->pool.heads, kv->pool.head_dim);
  shlo_kv_batch b;
  SHLO_TRY(batch_of(kv, starts, lens, tables, ka->shape[0], "kv_append", held, &b));
  return launch_kv_append(kv->pool, b, data_ptr(ka), ka->strides[0], ka->strides[1], data_ptr(va), va->strides[0], va->strides[1],
                          ka->dtype, kv->dev->stream);
}

int shlo_kv_gather(shlo_kv kv, shlo_arr tables, shlo_arr seq, shlo_arr pos, uint8_t dtype, shlo_arr *k, shlo_arr *v) {
  SHLO_TRY(usable(kv, "kv_gather"));
  if (!k || !v) return fail("kv_gather: null pointer");
  if (dtype != kF16 && dtype != kF32) return fail("kv_gather: %s not carried (float16 or float32)", dtype_name(dtype));
  Held held;
  Arr *t, *s, *p;
  SHLO_TRY(ints_of(kv, tables, 2, "kv_gather", "tables", held, &t));
  SHLO_TRY(ints_of(kv, seq, 1, "kv_gather", "seq", held, &s));
  SHLO_TRY(ints_of(kv, pos, 1, "kv_gather", "pos", held, &p));
  if (s->shape[0] != p->shape[0]) return fail("kv_gather: %lld sequences for %lld positions", (long long)s->shape[0], (long long)p->shape[0]);
  if (t->shape[0] > (1 << 20) || t->shape[1] > (1 << 22)) return fail("kv_gather: tables of %lld sequences of %lld pages", (long long)t->shape[0], (long long)t->shape[1]);
  const int64_t shape[3] = {s->shape[0], kv->pool.heads, kv->pool.head_dim}, token = (int64_t)kv->pool.heads * kv->pool.head_dim;
  Arr *ko, *vo;
  SHLO_TRY(new_array(kv->dev, dtype, shape, 3, &ko));
  held.arrays.push_back(ko);
  SHLO_TRY(new_array(kv->dev, dtype, shape, 3, &vo));
  held.arrays.push_back(vo);
  SHLO_TRY(launch_kv_gather(kv->pool, (const int32_t *)data_ptr(t), t->shape[1], (int32_t)t->shape[0], (int32_t)t->shape[1],
                            (const int32_t *)data_ptr(s), (const int32_t *)data_ptr(p), shape[0], data_ptr(ko), token,
                            kv->pool.head_dim, data_ptr(vo), token, kv->pool.head_dim, dtype, kv->dev->sm_count, kv->dev->stream));
  shlo_retain(ko);
  shlo_retain(vo);
  *k = ko;
  *v = vo;
  return 0;
}

int shlo_kv_attend(shlo_kv kv, shlo_arr q, shlo_arr starts, shlo_arr lens, shlo_arr tables, float scale, int32_t causal,
                   int32_t window, shlo_arr *out, shlo_arr *lse) {
  SHLO_TRY(usable(kv, "kv_attend"));
  if (!out) return fail("kv_attend: null pointer");
  Held held;
  Arr *qa, *o, *l = nullptr;
  SHLO_TRY(rows_of(kv, q, "kv_attend", "q", held, &qa));
  const int64_t T = qa->shape[0], H = qa->shape[1], D = qa->shape[2];
  if (H < 1 || H > 1 << 20) return fail("kv_attend: %lld query heads", (long long)H);
  AttendCall c = {};
  SHLO_TRY(batch_of(kv, starts, lens, tables, T, "kv_attend", held, &c.batch));
  Buffer *work;
  SHLO_TRY(workspace(kv->dev, &work));
  SHLO_TRY(new_array(kv->dev, qa->dtype, qa->shape, 3, &o));
  held.arrays.push_back(o);
  if (lse) {
    SHLO_TRY(new_array(kv->dev, kF32, qa->shape, 2, &l));
    held.arrays.push_back(l);
  }
  // (rows that no sequence has are not the kernels' to write)
  SHLO_CUDA(cudaMemsetAsync(data_ptr(o), 0, (size_t)numel(o) * dtype_size(o->dtype), kv->dev->stream));
  if (l) SHLO_CUDA(cudaMemsetAsync(data_ptr(l), 0, (size_t)numel(l) * 4, kv->dev->stream));
  c.pool = kv->pool;
  c.q = data_ptr(qa); c.q_token = qa->strides[0]; c.q_head = qa->strides[1];
  c.out = data_ptr(o); c.out_token = H * D; c.out_head = D;
  c.lse = l ? (float *)data_ptr(l) : nullptr;
  c.heads = (int32_t)H;
  c.dtype = qa->dtype;
  c.scale = scale;
  c.causal = causal != 0;
  c.window = window;
  c.work = work->ptr;
  c.work_bytes = work->bytes;
  c.err = kv->dev->pipe_err_dev;
  SHLO_TRY(launch_kv_attend(c, kv->dev->sm_count, kv->dev->id, kv->dev->stream));
  shlo_retain(o);
  *out = o;
  if (l) {
    shlo_retain(l);
    *lse = l;
  }
  return 0;
}

}  // extern "C"
