// Rows of a paged cache that go on as other rows: what a beam search's selection
// asks of the cache. New row r continues row parents[r]: it gets that row's length
// and pages. Full pages are shared; a last page that is not full, which the rows
// that share it would all write into, stays with the first row that continues its
// owner, and every later one gets a copy of its tokens (and scales) in a page of
// its own, fresh[r].
//
// Bound: bytes (a copied token read once and written once), and for a few rows a launch
// and four waits. A block has one new row and one head, or the row's table. Measured on
// one B200: 512 rows, 208 of which copy up to 127 tokens of 8 heads of 128 (45 MB, in
// part from L2), and tables of 236 pages 9.2 us; four rows of 8 heads of 64 2.8 us.
#include "decode.cuh"

namespace shlo {

namespace {

constexpr int kForkThreads = 128;

struct ForkCall : shlo_kv_fork_args {
  shlo_kv_pool pool;
};

__global__ void __launch_bounds__(kForkThreads) k_kv_fork(const ForkCall a) {
  const int r = blockIdx.x, parent = __ldg(a.parents + r), PT = a.pool.page_tokens;
  const bool live = parent >= 0 && parent < a.rows;
  const int len = live ? max(__ldg(a.lens + parent), 0) : 0, last = len / PT, tail = len % PT;
  bool shared = false;  // an earlier row continues the same one
  if (tail && last < a.table_pages) {
    for (int i = r - 1 - threadIdx.x; i >= 0; i -= kForkThreads)
      if (__ldg(a.parents + i) == parent) {
        shared = true;
        break;
      }
    shared = __syncthreads_or(shared);
  }
  const int32_t *const from = a.tables + (int64_t)parent * a.table_stride;  // (read where live)
  auto held = [&](int p) { return p >= 0 && p < a.pool.pages; };
  const int fresh = shared ? __ldg(a.fresh + r) : -1;
  if (blockIdx.y == a.pool.heads) {
    int32_t *const to = a.out_tables + (int64_t)r * a.out_stride;
    const int pages = last + (tail > 0);
    for (int i = threadIdx.x; i < a.table_pages; i += kForkThreads) {
      int p = -1;
      if (i < pages) {
        p = __ldg(from + i);
        if (i == last && shared && held(p)) p = held(fresh) ? fresh : -1;
      }
      to[i] = p;
    }
    if (threadIdx.x == 0) a.out_lens[r] = len;
    return;
  }
  if (!shared) return;
  const int old = __ldg(from + last), h = blockIdx.y;
  if (!held(old) || !held(fresh) || old == fresh) return;
  const int64_t src = (int64_t)old * a.pool.page_stride + (int64_t)h * a.pool.head_stride;
  const int64_t dst = (int64_t)fresh * a.pool.page_stride + (int64_t)h * a.pool.head_stride;
  const int pieces = a.pool.head_dim / 16, n = tail * pieces;
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * kForkThreads) {
    uint4 k[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = i0 + j * kForkThreads, t = i / pieces;
      const int64_t o = t * a.pool.token_stride + (i - t * pieces) * 16;
      if (i < n) {
        k[j] = *reinterpret_cast<const uint4 *>(a.pool.k + src + o);
        v[j] = *reinterpret_cast<const uint4 *>(a.pool.v + src + o);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = i0 + j * kForkThreads, t = i / pieces;
      const int64_t o = t * a.pool.token_stride + (i - t * pieces) * 16;
      if (i < n) {
        *reinterpret_cast<uint4 *>(a.pool.k + dst + o) = k[j];
        *reinterpret_cast<uint4 *>(a.pool.v + dst + o) = v[j];
      }
    }
  }
  if (threadIdx.x < 2) {
    float *const s = (threadIdx.x ? a.pool.v_scale : a.pool.k_scale) + (int64_t)h * a.pool.scale_head_stride;
    s[(int64_t)fresh * a.pool.scale_page_stride] = s[(int64_t)old * a.pool.scale_page_stride];
  }
}

}  // namespace

int launch_kv_fork(const shlo_kv_pool &p, const shlo_kv_fork_args &args, cudaStream_t st) {
  ForkCall c;
  static_cast<shlo_kv_fork_args &>(c) = args;
  c.pool = p;
  SHLO_TRY(check_pool(&c.pool, "kv_fork"));
  if (c.rows < 0 || c.news < 0 || c.news > 65536 || c.table_pages < 0 || c.table_pages > (1 << 22))
    return fail("kv_fork: %d rows continued by %d (at most 65536), tables of %d pages (at most 2^22)", c.rows, c.news, c.table_pages);
  if (c.news == 0) return 0;
  if (!c.parents || !c.fresh || !c.out_lens || (c.rows && !c.lens) || (c.table_pages && ((c.rows && !c.tables) || !c.out_tables)))
    return fail("kv_fork: null pointer");
  if (((uintptr_t)c.parents | (uintptr_t)c.fresh | (uintptr_t)c.lens | (uintptr_t)c.tables | (uintptr_t)c.out_tables | (uintptr_t)c.out_lens) % 4)
    return fail("kv_fork: misaligned tables, lens, parents or fresh");
  const int64_t list = 4 * (int64_t)c.news, wide = 4 * (int64_t)c.table_pages, old_step = 4 * c.table_stride, new_step = 4 * c.out_stride;
  auto hits = [&](const void *p, int64_t rows, int64_t step, int64_t bytes) {
    return meet(c.out_tables, c.news, new_step, wide, p, rows, step, bytes) || meet(c.out_lens, 1, 0, list, p, rows, step, bytes);
  };
  if (hits(c.tables, c.rows, old_step, wide) || hits(c.lens, 1, 0, 4 * (int64_t)c.rows) || hits(c.parents, 1, 0, list) || hits(c.fresh, 1, 0, list) ||
      meet(c.out_tables, c.news, new_step, wide, c.out_lens, 1, 0, list))
    return fail("kv_fork: the new tables and lengths are not the old ones' memory, nor parents' or fresh's");
  if (c.pool.heads > 65534) return fail("kv_fork: %d heads", c.pool.heads);
  k_kv_fork<<<dim3((unsigned)c.news, (unsigned)c.pool.heads + 1), kForkThreads, 0, st>>>(c);
  return launch_check("kv_fork");
}

}  // namespace shlo

using namespace shlo;

extern "C" {

int shlo_kv_fork_noalloc(const shlo_kv_pool *pool, const shlo_kv_fork_args *args, void *stream) {
  if (!pool || !args) return fail("kv_fork: null descriptor");
  Device *dev;
  SHLO_TRY(calling_device(&dev));
  return launch_kv_fork(*pool, *args, (cudaStream_t)stream);
}

}  // extern "C"
