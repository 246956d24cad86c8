// What the kernels of the attention over the paged cache share: the arguments,
// the work list and its even split over the blocks, and the joining of partial
// results.
//
// Work. The rows of a sequence and a key/value head are its new tokens times
// the query heads that share the head, r = token * group + head, in tiles of
// kRows. A tile sees the keys [lo, hi) of its rows; a granule is kGran keys from
// a multiple of kGran. A unit is one tile of one key/value head: all its
// granules. The units of all heads lie on one line of W granules, which the N
// blocks cut into equal parts, so ragged lengths and few long sequences load
// every block alike. A block computes the line itself from `starts` and `lens`
// (the host knows neither), by a scan over slots: sequence s has the slots from
// floor(starts[s] * group / kRows) + s on, always enough for its tiles.
//
// Joining. A unit cut between blocks leaves one partial result a block: the sum
// of exp2(score - m) v without the division, m and the sum l, in 32 bits. At
// most two a block: of the unit it starts in the middle of, and of the one it
// leaves unfinished. The block that arrives last joins them, always in the
// order of the keys, so the result does not depend on who is last; more than
// kJoin partials are joined in groups of kJoin first.
#pragma once

#include "decode.cuh"

namespace shlo {

struct AttendArgs {
  shlo_kv_pool pool;
  shlo_kv_batch batch;
  const void *q;
  void *out;
  float *lse;
  int64_t q_token, q_head, out_token, out_head;
  int group;         // query heads a key/value head
  int slots;         // slots of the work list
  int causal, window;
  float scale_log2;  // scale * log2(e)
  int page_shift;
  // Which sequences this launch takes: those with rows (new tokens * group) in
  // (above, upto].
  int64_t above, upto;
  unsigned *counters;  // [2][kAttendMaxBlocks], zero between calls
  float *partials;     // [blocks][2][rows * (dim + 2)]
};

constexpr int kAttendMaxBlocks = 1024;
constexpr int kJoin = 16;

// A tile of rows and what it sees.
struct RowTile {
  int seq, row0, rows;   // the sequence, its first row, how many (1..kRows)
  int start, n, first;   // the sequence's first token in q, new tokens, the first one's position
  int keys;              // the keys that exist: min(length, table)
  int lo, hi;            // keys any row of the tile sees are in [lo, hi)
  int lo_all, hi_all;    // keys in [lo_all, hi_all) are seen by every row of the tile
};

__device__ __forceinline__ int row_hi(const AttendArgs &a, int keys, int pos) {
  return a.causal ? max(0, min(keys, pos + 1)) : keys;
}
__device__ __forceinline__ int row_lo(const AttendArgs &a, int pos) {
  return a.window ? max(0, pos - a.window + 1) : 0;
}

// The tile of a slot; returns its granules (0: the slot has no tile here).
template <int ROWS, int GRAN>
__device__ __forceinline__ int tile_of_slot(const AttendArgs &a, int slot, RowTile &t) {
  constexpr int SH = ROWS == 8 ? 3 : ROWS == 16 ? 4 : ROWS == 64 ? 6 : 7;
  static_assert(1 << SH == ROWS, "rows of a tile");
  const int s = slot_owner(a.batch, slot, a.group, SH, 1);
  const SeqSpan sp = seq_span(a.batch, s);
  const int64_t rows = (int64_t)sp.n * a.group;
  const int64_t row0 = (int64_t)(slot - slot_base(a.batch, s, a.group, SH, 1)) * ROWS;
  if (row0 < 0 || row0 >= rows || rows <= a.above || rows > a.upto) return 0;
  t.seq = s;
  t.row0 = (int)row0;
  t.rows = (int)min((int64_t)ROWS, rows - row0);
  t.start = sp.start;
  t.n = sp.n;
  t.first = sp.len - sp.n;
  t.keys = (int)min((int64_t)sp.len, (int64_t)a.batch.table_pages << a.page_shift);
  const int p0 = t.first + t.row0 / a.group, p1 = t.first + (t.row0 + t.rows - 1) / a.group;
  t.lo = row_lo(a, p0);
  t.hi = row_hi(a, t.keys, p1);
  t.lo_all = row_lo(a, p1);
  t.hi_all = row_hi(a, t.keys, p0);
  if (t.hi <= t.lo) {  // nothing to see: one granule, which writes the empty result
    t.lo = t.hi = 0;
    return 1;
  }
  return (t.hi + GRAN - 1) / GRAN - t.lo / GRAN;
}

// A block's part of the line, and where it stands on it.
struct Cursor {
  long long per_head;    // granules a head
  long long total;       // W
  int blocks;            // blocks with work
  long long at, end;     // this block's part
  int head, slot, off;   // the unit `at` is in, and the granule in it
};

// All threads call it; NT threads, `sh` shared memory of NT + 4 long longs. A
// block without work returns false.
template <int ROWS, int GRAN, int NT>
__device__ bool schedule(const AttendArgs &a, int min_gran, long long *sh, Cursor &c) {
  const int chunk = (a.slots + NT - 1) / NT;
  const int s0 = min((int)threadIdx.x * chunk, a.slots), s1 = min(s0 + chunk, a.slots);
  long long mine = 0;
  RowTile t;
  for (int s = s0; s < s1; s++) mine += tile_of_slot<ROWS, GRAN>(a, s, t);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(~0u, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) sh[warp] = sum;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; w++) {
    const long long v = sh[w];
    if (w < warp) before += v;
    all += v;
  }
  before += sum - mine;
  c.per_head = all;
  c.total = all * a.pool.heads;
  if (c.total == 0) return false;
  const long long fit = c.total / min_gran;
  c.blocks = (int)(fit < 1 ? 1 : fit < (long long)gridDim.x ? fit : (long long)gridDim.x);
  if ((int)blockIdx.x >= c.blocks) return false;
  c.at = c.total * blockIdx.x / c.blocks;
  c.end = c.total * (blockIdx.x + 1) / c.blocks;
  c.head = (int)(c.at / all);
  const long long rem = c.at - c.head * all;
  __syncthreads();
  if (rem >= before && rem < before + mine) {
    long long r = rem - before;
    int s = s0;
    for (; s < s1; s++) {
      const int g = tile_of_slot<ROWS, GRAN>(a, s, t);
      if (r < g) break;
      r -= g;
    }
    sh[0] = s;
    sh[1] = r;
  }
  __syncthreads();
  c.slot = (int)sh[0];
  c.off = (int)sh[1];
  __syncthreads();
  return true;
}

// The block that a granule of the line belongs to.
__device__ __forceinline__ int block_of(const Cursor &c, long long x) {
  return (int)(((x + 1) * c.blocks - 1) / c.total);
}

// Where block `i` keeps its partial: 0 of a unit begun by an earlier block, 1
// of one that it begins.
template <int ROWS, int DP>
__device__ __forceinline__ float *partial_at(const AttendArgs &a, int i, int which) {
  return a.partials + ((int64_t)i * 2 + which) * (ROWS * (DP + 2));
}

template <typename T>
__device__ __forceinline__ void write_out(const AttendArgs &a, const RowTile &t, int head, int row, int d, float v) {
  const int r = t.row0 + row, tok = t.start + r / a.group, h = head * a.group + r % a.group;
  T *o = static_cast<T *>(a.out) + (int64_t)tok * a.out_token + (int64_t)h * a.out_head + d;
  if constexpr (sizeof(T) == 2) *o = __float2half_rn(v);
  else *o = v;
}
__device__ __forceinline__ void write_lse(const AttendArgs &a, const RowTile &t, int head, int row, float m, float l) {
  if (!a.lse) return;
  const int r = t.row0 + row, tok = t.start + r / a.group, h = head * a.group + r % a.group;
  a.lse[(int64_t)tok * (a.group * a.pool.heads) + h] =
      l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

// m and l of a set of partials: what each contributes.
__device__ __forceinline__ float join_factor(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2f(m - top);
}

// Join the partials of blocks i0 .. i0 + n - 1 (the first one's slot is
// `which0`, the others' 0; `step` blocks apart) into `dst` (a partial), or into
// the output when dst is null. NT threads; fac: shared memory of (n + 2) * ROWS floats.
template <typename T, int ROWS, int DP, int NT>
__device__ void join(const AttendArgs &a, const RowTile &t, int head, int i0, int n, int step, int which0, float *dst,
                     float *fac) {
  auto src = [&](int k) -> const float * { return partial_at<ROWS, DP>(a, i0 + k * step, k == 0 ? which0 : 0); };
  for (int i = threadIdx.x; i < n * ROWS; i += NT) {
    const int k = i / ROWS, row = i % ROWS;
    fac[i] = __ldcg(src(k) + ROWS * DP + row);
  }
  __syncthreads();
  float *const top = fac + n * ROWS, *const sum = top + ROWS;
  for (int row = threadIdx.x; row < ROWS; row += NT) {
    float m = -INFINITY;
    for (int k = 0; k < n; k++) m = fmaxf(m, fac[k * ROWS + row]);
    float l = 0.0f;
    for (int k = 0; k < n; k++) {
      const float f = join_factor(fac[k * ROWS + row], m);
      fac[k * ROWS + row] = f;
      l = __fmaf_rn(f, __ldcg(src(k) + ROWS * DP + ROWS + row), l);
    }
    top[row] = m;
    sum[row] = l;
    if (dst) {
      dst[ROWS * DP + row] = m;
      dst[ROWS * DP + ROWS + row] = l;
    } else if (row < t.rows) {
      write_lse(a, t, head, row, m, l);
    }
  }
  __syncthreads();
  // In place where dst is the first partial: each thread reads a value of it before it writes it.
  for (int i = threadIdx.x; i < t.rows * DP / 4; i += NT) {
    const int row = i / (DP / 4), d = (i % (DP / 4)) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < n; k++) {
      const float4 v = __ldcg(reinterpret_cast<const float4 *>(src(k) + row * DP + d));
      const float f = fac[k * ROWS + row];
      o.x = __fmaf_rn(f, v.x, o.x);
      o.y = __fmaf_rn(f, v.y, o.y);
      o.z = __fmaf_rn(f, v.z, o.z);
      o.w = __fmaf_rn(f, v.w, o.w);
    }
    if (dst) {
      *reinterpret_cast<float4 *>(dst + row * DP + d) = o;
    } else if (d < a.pool.head_dim) {
      const float l = sum[row];
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      write_out<T>(a, t, head, row, d, l == 0.0f ? 0.0f : o.x * inv);
      write_out<T>(a, t, head, row, d + 1, l == 0.0f ? 0.0f : o.y * inv);
      write_out<T>(a, t, head, row, d + 2, l == 0.0f ? 0.0f : o.z * inv);
      write_out<T>(a, t, head, row, d + 3, l == 0.0f ? 0.0f : o.w * inv);
    }
  }
  __syncthreads();
}

// Called by all threads of a block after it wrote its partial of a unit of the
// line's granules [u0, u1): joins what is complete. `flag`: shared memory.
template <typename T, int ROWS, int DP, int NT>
__device__ void arrive(const AttendArgs &a, const RowTile &t, const Cursor &c, long long u0, long long u1, float *fac,
                       unsigned *flag) {
  const int i0 = block_of(c, u0), i1 = block_of(c, u1 - 1), n = i1 - i0 + 1;
  auto last = [&](unsigned *ctr, int of) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *flag = atomicInc(ctr, (unsigned)of - 1) == (unsigned)of - 1;  // wraps to 0
    __syncthreads();
    const bool yes = *flag != 0;
    __syncthreads();
    if (yes) __threadfence();
    return yes;
  };
  if (n <= kJoin) {
    if (last(a.counters + i0, n)) join<T, ROWS, DP, NT>(a, t, c.head, i0, n, 1, 1, nullptr, fac);
    return;
  }
  const int k = ((int)blockIdx.x - i0) / kJoin, g0 = i0 + k * kJoin, gn = min(kJoin, i1 - g0 + 1);
  const int groups = (n + kJoin - 1) / kJoin;
  // (a group of one needs no count; its block's counter may be another unit's)
  if (gn > 1) {
    if (!last(a.counters + g0, gn)) return;
    join<T, ROWS, DP, NT>(a, t, c.head, g0, gn, 1, k == 0, partial_at<ROWS, DP>(a, g0, k == 0), fac);
  }
  if (last(a.counters + kAttendMaxBlocks + i0, groups))
    join<T, ROWS, DP, NT>(a, t, c.head, i0, groups, kJoin, 1, nullptr, fac);
}

}  // namespace shlo
