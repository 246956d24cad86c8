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

// "shlo_norm_rope": x [T][H][D], positions int32 [T], phases int64 [rot / 2], the
// queries' and the keys' weight [D], p = [T, H, D, rot, flags, factor bits, query
// heads, eps bits]; the result is of x's type.
int k_norm_rope(Device *dev, Arr *x, Arr *positions, Arr *phases, Arr *q_weight, Arr *k_weight, const uint32_t *p, Arr **out) {
  NormRopeCall c = {};
  SHLO_TRY(norm_rope_call("shlo_norm_rope", x, positions, phases, q_weight, k_weight, p, &c));
  const int64_t shape[3] = {p[0], p[1], p[2]};
  Arr *o;
  SHLO_TRY(new_array(dev, x->dtype, shape, 3, &o));
  c.y = data_ptr(o);
  c.y_token = c.x_token;
  c.y_head = c.x_head;
  if (launch_norm_rope(c, false, dev->sm_count, dev->stream)) {
    shlo_release(o);
    return 1;
  }
  *out = o;
  return 0;
}

int norm_rope_call(const char *what, Arr *x, Arr *positions, Arr *phases, Arr *q_weight, Arr *k_weight, const uint32_t *p, NormRopeCall *c) {
  const int64_t T = p[0], H = p[1], D = p[2], rot = p[3];
  if (positions->dtype != kI32) return fail("%s: positions of %s, int32 expected", what, dtype_name(positions->dtype));
  if (phases->dtype != kI64) return fail("%s: phases of %s, int64 expected", what, dtype_name(phases->dtype));
  if (H < 1 || D < 1 || T > 0x7fffffff || H > 0x7fffffff || D > 512 || T * H > ((int64_t)1 << 40) / D)
    return fail("%s: %lld tokens of %lld heads of %lld", what, (long long)T, (long long)H, (long long)D);
  if (numel(x) != T * H * D || numel(positions) != T || numel(phases) < rot / 2)
    return fail("%s: %lld values, %lld positions and %lld phases for [%lld, %lld, %lld] and %lld dimensions turned", what,
                (long long)numel(x), (long long)numel(positions), (long long)numel(phases), (long long)T, (long long)H,
                (long long)D, (long long)rot);
  if (numel(q_weight) != D || numel(k_weight) != D || q_weight->dtype != k_weight->dtype)
    return fail("%s: the weights are not of %lld values of one type", what, (long long)D);
  c->x = data_ptr(x);
  c->x_token = H * D;
  c->x_head = D;
  c->positions = (const int32_t *)data_ptr(positions);
  c->phases = (const int64_t *)data_ptr(phases);
  c->q_weight = data_ptr(q_weight);
  c->k_weight = data_ptr(k_weight);
  c->weight_dtype = q_weight->dtype;
  c->q_heads = (int32_t)p[6];
  c->eps = bitsf_host(p[7]);
  c->tokens = T;
  c->heads = (int32_t)H;
  c->dim = (int32_t)D;
  c->rot = (int32_t)rot;
  c->dtype = x->dtype;
  c->flags = p[4];
  c->factor = bitsf_host(p[5]);
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

// The op log's names of what is read here (those of elementwise.cu and runtime.cu are below 30).
enum { OT_NORM_ROPE_GRAD = 30, OT_QUANTISE_ROWS, OT_LINEAR8, OT_BEAM_SELECT };

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

// Row-major copies where they are needed, held to one device.
int whole(Device *dev, Arr *a, const char *what, const char *name, Held &held, Arr **out) {
  if (!a) return fail("%s: %s is null", what, name);
  if (numel(a) && (!a->buf || a->buf->dev != dev)) return fail("%s: %s is on another device", what, name);
  SHLO_TRY(make_contiguous(a, out));
  held.arrays.push_back(*out);
  return 0;
}
int shaped(Arr *a, uint8_t dtype, std::initializer_list<int64_t> shape, const char *what, const char *name) {
  bool same = a->dtype == dtype && a->ndim == (int)shape.size();
  int i = 0;
  for (int64_t n : shape) {
    same = same && a->shape[i] == n;
    i++;
  }
  if (!same) return fail("%s: %s is %s of rank %d, or of another shape", what, name, dtype_name(a->dtype), a->ndim);
  return 0;
}
int made(Device *dev, uint8_t dtype, std::initializer_list<int64_t> shape, Held &held, Arr **out) {
  std::vector<int64_t> n(shape);
  SHLO_TRY(new_array(dev, dtype, n.data(), (int)n.size(), out));
  held.arrays.push_back(*out);
  return 0;
}
void give(Arr *a, shlo_arr *out) {
  shlo_retain(a);
  *out = a;
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

int shlo_kv_fork(shlo_kv kv, shlo_arr tables, shlo_arr lens, shlo_arr parents, shlo_arr fresh, shlo_arr *out_tables, shlo_arr *out_lens) {
  SHLO_TRY(usable(kv, "kv_fork"));
  if (!out_tables || !out_lens) return fail("kv_fork: null pointer");
  Held held;
  Arr *t, *l, *p, *f, *ot, *ol;
  SHLO_TRY(ints_of(kv, tables, 2, "kv_fork", "tables", held, &t));
  SHLO_TRY(ints_of(kv, lens, 1, "kv_fork", "lens", held, &l));
  SHLO_TRY(ints_of(kv, parents, 1, "kv_fork", "parents", held, &p));
  SHLO_TRY(ints_of(kv, fresh, 1, "kv_fork", "fresh", held, &f));
  const int64_t rows = t->shape[0], width = t->shape[1], news = p->shape[0];
  if (l->shape[0] != rows || f->shape[0] != news || rows > 0x7fffffff || news > 65536 || width > (1 << 22))
    return fail("kv_fork: %lld lengths for tables of %lld rows of %lld pages, %lld fresh pages for %lld rows", (long long)l->shape[0],
                (long long)rows, (long long)width, (long long)f->shape[0], (long long)news);
  SHLO_TRY(made(kv->dev, kI32, {news, width}, held, &ot));
  SHLO_TRY(made(kv->dev, kI32, {news}, held, &ol));
  const shlo_kv_fork_args c{(const int32_t *)data_ptr(t), (const int32_t *)data_ptr(l), width, (const int32_t *)data_ptr(p),
                            (const int32_t *)data_ptr(f), (int32_t *)data_ptr(ot), (int32_t *)data_ptr(ol), width, (int32_t)rows,
                            (int32_t)news, (int32_t)width};
  SHLO_TRY(launch_kv_fork(kv->pool, c, kv->dev->stream));
  give(ot, out_tables);
  give(ol, out_lens);
  return 0;
}

int shlo_norm_rope_grad(shlo_arr x, shlo_arr dy, shlo_arr positions, shlo_arr phases, shlo_arr q_weight, shlo_arr k_weight,
                        int32_t q_heads, float eps, uint32_t flags, float factor, shlo_arr *dx, shlo_arr *dq_weight, shlo_arr *dk_weight) {
  const char *const what = "norm_rope_grad";
  if (!x || !dx || !dq_weight || !dk_weight) return fail("%s: null pointer", what);
  Arr *const ins[6] = {x, dy, positions, phases, q_weight, k_weight};
  for (Arr *a : ins)
    if (!a) return fail("%s: null array", what);
  TraceScope ts(TK_OTHER, OT_NORM_ROPE_GRAD, nullptr, 0, ins, 6);
  Device *dev;
  SHLO_TRY(arr_device(x, &dev));
  Held held;
  Arr *a[6];
  static const char *const names[6] = {"x", "dy", "positions", "phases", "q_weight", "k_weight"};
  for (int i = 0; i < 6; i++) SHLO_TRY(whole(dev, ins[i], what, names[i], held, &a[i]));
  if (x->ndim != 3 || phases->ndim != 1) return fail("%s: x is not [tokens, heads, dim], or phases are no vector", what);
  SHLO_TRY(shaped(dy, x->dtype, {x->shape[0], x->shape[1], x->shape[2]}, what, "dy"));
  if (x->shape[0] > 0x7fffffff || x->shape[1] > 0x7fffffff || x->shape[2] > 512) return fail("%s: x is too large", what);
  uint32_t p[8] = {(uint32_t)x->shape[0], (uint32_t)x->shape[1], (uint32_t)x->shape[2], (uint32_t)(2 * phases->shape[0]), flags, 0, (uint32_t)q_heads, 0};
  memcpy(&p[5], &factor, 4);
  memcpy(&p[7], &eps, 4);
  NormRopeCall c = {};
  SHLO_TRY(norm_rope_call(what, a[0], a[2], a[3], a[4], a[5], p, &c));
  Arr *o, *q, *k, *w;
  SHLO_TRY(made(dev, x->dtype, {x->shape[0], x->shape[1], x->shape[2]}, held, &o));
  SHLO_TRY(made(dev, kF32, {c.dim}, held, &q));
  SHLO_TRY(made(dev, kF32, {c.dim}, held, &k));
  const size_t bytes = norm_rope_work_bytes(dev->sm_count);
  SHLO_TRY(made(dev, kU8, {(int64_t)bytes}, held, &w));
  c.dy = data_ptr(a[1]);
  c.dy_token = c.x_token;
  c.dy_head = c.x_head;
  c.y = data_ptr(o);
  c.y_token = c.x_token;
  c.y_head = c.x_head;
  c.dq_weight = (float *)data_ptr(q);
  c.dk_weight = (float *)data_ptr(k);
  c.workspace = data_ptr(w);
  c.workspace_bytes = bytes;
  SHLO_TRY(launch_norm_rope(c, true, dev->sm_count, dev->stream));
  give(o, dx);
  give(q, dq_weight);
  give(k, dk_weight);
  ts.done(nullptr);
  return 0;
}

int shlo_quantise_rows(shlo_arr x, shlo_arr *q, shlo_arr *scale) {
  const char *const what = "quantise_rows";
  if (!x || !q || !scale) return fail("%s: null pointer", what);
  TraceScope ts(TK_OTHER, OT_QUANTISE_ROWS, nullptr, 0, &x, 1);
  Device *dev;
  SHLO_TRY(arr_device(x, &dev));
  Held held;
  Arr *a, *o, *s;
  SHLO_TRY(whole(dev, x, what, "x", held, &a));
  if (x->ndim != 2 || x->shape[1] < 1 || x->shape[1] > 0x7fffff00) return fail("%s: x is not [rows, values]", what);
  const int64_t rows = x->shape[0], n = x->shape[1], row = (n + 15) / 16 * 16;
  SHLO_TRY(made(dev, kI8, {rows, row}, held, &o));
  SHLO_TRY(made(dev, kF32, {rows}, held, &s));
  SHLO_TRY(launch_quantise_rows(data_ptr(a), n, x->dtype, rows, (int32_t)n, (int8_t *)data_ptr(o), row, (float *)data_ptr(s), true, what, dev->stream));
  give(o, q);
  give(s, scale);
  ts.done(nullptr);
  return 0;
}

int shlo_linear8(shlo_arr x, shlo_arr x_scale, shlo_arr w, shlo_arr w_scale, shlo_arr bias, uint8_t dtype, shlo_arr *out) {
  const char *const what = "linear8";
  if (!x || !w || !w_scale || !out) return fail("%s: null pointer", what);
  Arr *ins[5] = {x, w, w_scale, nullptr, nullptr};
  int n_ins = 3;
  if (x_scale) ins[n_ins++] = x_scale;
  if (bias) ins[n_ins++] = bias;
  TraceScope ts(TK_OTHER, OT_LINEAR8, nullptr, 0, ins, n_ins);
  Device *dev;
  SHLO_TRY(arr_device(x, &dev));
  Held held;
  Arr *a, *b, *s, *o, *e = nullptr;
  SHLO_TRY(whole(dev, x, what, "x", held, &a));
  SHLO_TRY(whole(dev, w, what, "w", held, &b));
  SHLO_TRY(whole(dev, w_scale, what, "w_scale", held, &s));
  if (x->ndim != 2 || w->ndim != 2 || w->dtype != kI8) return fail("%s: x is not [rows, values], or w not int8 [channels, values]", what);
  const int64_t rows = x->shape[0], n = x->shape[1], m = w->shape[0], row = (n + 15) / 16 * 16;
  if (n < 1 || n > 131071 || m < 1 || m > (1 << 30) || rows > (1 << 28)) return fail("%s: %lld rows, %lld channels of %lld values", what, (long long)rows, (long long)m, (long long)n);
  if (w->shape[1] != row) return fail("%s: rows of w of %lld values, x's %lld and zeros up to a multiple of 16 expected", what, (long long)w->shape[1], (long long)n);
  SHLO_TRY(shaped(w_scale, kF32, {m}, what, "w_scale"));
  if (bias) {
    SHLO_TRY(whole(dev, bias, what, "bias", held, &e));
    SHLO_TRY(shaped(bias, kF32, {m}, what, "bias"));
  }
  SHLO_TRY(made(dev, dtype, {rows, m}, held, &o));
  Mm8Call c = {};
  c.x = data_ptr(a); c.x_row = n; c.x_dtype = x->dtype;
  c.w = (const int8_t *)data_ptr(b); c.w_row = row; c.w_scale = (const float *)data_ptr(s);
  c.bias = e ? (const float *)data_ptr(e) : nullptr;
  c.y = data_ptr(o); c.y_row = m; c.dtype = dtype;
  c.rows = rows; c.n = (int32_t)n; c.m = (int32_t)m;
  if (x->dtype == kI8) {
    if (!x_scale) return fail("%s: x of int8 without its scales", what);
    if (n != row) return fail("%s: rows of x of %lld values, a multiple of 16 expected", what, (long long)n);
    Arr *t;
    SHLO_TRY(whole(dev, x_scale, what, "x_scale", held, &t));
    SHLO_TRY(shaped(x_scale, kF32, {rows}, what, "x_scale"));
    c.x_scale = (const float *)data_ptr(t);
    SHLO_TRY(launch_mul_mat8(c, false, dev->pipe_err_dev, dev->sm_count, dev->stream));
  } else {
    if (x_scale) return fail("%s: scales of rows that are not int8", what);
    c.workspace_bytes = linear8_work_bytes(rows, (int32_t)n);
    Arr *t;
    SHLO_TRY(made(dev, kU8, {(int64_t)c.workspace_bytes}, held, &t));
    c.workspace = data_ptr(t);
    SHLO_TRY(launch_linear8(c, dev->pipe_err_dev, dev->sm_count, dev->stream));
  }
  give(o, out);
  ts.done(o);
  return 0;
}

int shlo_beam_select(shlo_arr logits, shlo_arr scores, shlo_arr ended, int32_t end_token, int32_t keep, shlo_arr *next, shlo_arr *parents,
                     shlo_arr *tokens) {
  const char *const what = "beam_select";
  if (!logits || !scores || !next || !parents || !tokens) return fail("%s: null pointer", what);
  Arr *ins[3] = {logits, scores, ended};
  TraceScope ts(TK_OTHER, OT_BEAM_SELECT, nullptr, 0, ins, ended ? 3 : 2);
  Device *dev;
  SHLO_TRY(arr_device(logits, &dev));
  Held held;
  Arr *z, *s, *e = nullptr, *o, *p, *t, *w;
  SHLO_TRY(whole(dev, logits, what, "logits", held, &z));
  SHLO_TRY(whole(dev, scores, what, "scores", held, &s));
  if (logits->ndim != 2 || scores->ndim != 2 || scores->dtype != kF32 || scores->shape[0] * scores->shape[1] != logits->shape[0])
    return fail("%s: logits are not [sequences * beams, vocabulary] of scores float32 [sequences, beams]", what);
  const int64_t seqs = scores->shape[0], beams = scores->shape[1], vocab = logits->shape[1];
  if (seqs > 65535 || beams > 65535 || vocab > 0x7fffffff) return fail("%s: %lld sequences of %lld beams over %lld", what, (long long)seqs, (long long)beams, (long long)vocab);
  if (ended) {
    SHLO_TRY(whole(dev, ended, what, "ended", held, &e));
    SHLO_TRY(shaped(ended, kI32, {seqs, beams}, what, "ended"));
  }
  size_t bytes;
  SHLO_TRY(shlo_beam_workspace((int32_t)seqs, (int32_t)beams, keep, (int32_t)vocab, &bytes));
  SHLO_TRY(made(dev, kF32, {seqs, keep}, held, &o));
  SHLO_TRY(made(dev, kI32, {seqs, keep}, held, &p));
  SHLO_TRY(made(dev, kI32, {seqs, keep}, held, &t));
  SHLO_TRY(made(dev, kU8, {(int64_t)bytes}, held, &w));
  BeamCall c = {};
  c.logits = data_ptr(z); c.row = vocab; c.dtype = logits->dtype;
  c.scores = (const float *)data_ptr(s); c.ended = e ? (const int32_t *)data_ptr(e) : nullptr; c.end_token = end_token;
  c.next = (float *)data_ptr(o); c.parents = (int32_t *)data_ptr(p); c.tokens = (int32_t *)data_ptr(t);
  c.workspace = data_ptr(w); c.workspace_bytes = bytes;
  c.seqs = (int32_t)seqs; c.beams = (int32_t)beams; c.keep = keep; c.vocab = (int32_t)vocab;
  SHLO_TRY(launch_beam_select(c, dev->sm_count, dev->stream));
  give(o, next);
  give(p, parents);
  give(t, tokens);
  ts.done(nullptr);
  return 0;
}

}  // extern "C"
