// What the kernels of the attention over the paged cache share: the arguments,
// the work list and its even split over the blocks, and the joining of partial
// results.
//
// Work. The rows of a sequence and a key/value head are its new tokens times
// the query heads that share the head, r = token * group + head, in tiles of
// kRows. A tile sees the keys [lo, hi) of its rows; a granule is kGran keys from
// a multiple of kGran. A unit is one tile of one key/value head: all its
// granules. The units of all heads lie on one line of W granules, which the N
// blocks cut into equal chunks, whatever units they fall in: ragged lengths and
// few long sequences give every block the same number of keys, though not the
// same time, as the beginnings, cuts and joins are not counted (in a batch of 64
// ragged sequences blocks ended after 83 to 121 us). A block computes the line
// itself from `starts` and `lens` (the host knows neither), by a scan over slots:
// sequence s has the slots from floor(starts[s] * group / kRows) + s on, always
// enough for its tiles. (Measured and left: four chunks a block of falling size,
// taken from a counter. 64 x 8192 keys took 246 us instead of 230: every cut
// costs a block about 8 us, more than the unevenness it evens out.)
//
// Joining. A unit cut between chunks leaves one partial result a chunk: the sum
// of exp2(score - m) v without the division, m and the sum l, in 32 bits. At
// most two a chunk: of the unit it starts in the middle of, and of the one it
// leaves unfinished. The block that arrives last joins them, always in the
// order of the keys; more than kJoin partials are joined in groups of kJoin first.
#pragma once

#include <type_traits>

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
  int out_wide;      // out allows stores of four values (1), of eight (2)
  int q_wide;        // q allows 16-byte loads
  float scale_log2;  // scale * log2(e)
  int page_shift;
  // Which sequences this launch takes: those with rows (new tokens * group) in
  // (above, upto].
  int64_t above, upto;
  unsigned *counters;  // [2][kAttendMaxBlocks], zero between calls
  float *partials;     // [chunks][2][rows * (dim + 2)]
  int *err;            // 1: a launch gave up a wait; 2: the batch's starts descend
  unsigned give_up;    // every so many blocks of the tiles give up at once (0: none)
};

constexpr uint64_t kWaitLimitNs = 2000000000ull;

constexpr int kAttendMaxBlocks = 1024;
// Partials joined at once: what a join's factors take in shared memory bounds it.
template <int ROWS> constexpr int kJoin = ROWS >= 128 ? 32 : 64;
template <int ROWS> constexpr int kRowShift = ROWS == 8 ? 3 : ROWS == 16 ? 4 : ROWS == 128 ? 7 : 8;

// A kernel's dynamic shared memory, allowed once a device: `done` is the launch's
// own bits (the call itself would be a tenth of a small launch).
inline int allow_smem(const void *kern, size_t bytes, std::atomic<uint64_t> &done, int device) {
  const uint64_t bit = (uint64_t)1 << device;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  SHLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.fetch_or(bit);
  return 0;
}

// kv_attend_tiles.cu: tiles of 256 rows (128 of heads wider than 128), float16.
int launch_attend_tiles(const AttendArgs &a, int sms, int device, cudaStream_t st);
size_t attend_tiles_partial_bytes(int sms);

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
  return a.window && pos >= a.window ? pos - a.window + 1 : 0;  // (pos may be negative)
}

// The tile of a slot; returns its granules (0: the slot has no tile here).
// t.seq, when `after` is set, is the owner of an earlier slot: the search goes
// on from it, one sequence at a time.
template <int ROWS, int GRAN>
__device__ __forceinline__ int tile_of_slot(const AttendArgs &a, const int32_t *starts, const int32_t *lens, int slot,
                                            RowTile &t, bool after) {
  constexpr int SH = kRowShift<ROWS>;
  const int tokens = a.batch.tokens, seqs = a.batch.seqs;
  int s;
  if (after) {
    s = t.seq;
    while (s + 1 < seqs && slot_base(starts, tokens, s + 1, a.group, SH, 1) <= slot) s++;
  } else {
    s = slot_owner(starts, tokens, seqs, 0, slot, a.group, SH, 1);
  }
  t.seq = s;
  const SeqSpan sp = seq_span(starts, lens, tokens, s);
  const int64_t rows = (int64_t)sp.n * a.group;
  const int64_t row0 = (int64_t)(slot - slot_base(starts, tokens, s, a.group, SH, 1)) * ROWS;
  if (row0 < 0 || row0 >= rows || rows <= a.above || rows > a.upto) return 0;
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

// The line.
struct Line {
  long long per_head;      // granules a head
  long long total;         // W
  int blocks;              // blocks with work
  long long before, mine;  // this thread's slots' granules on a head's line
};
// A place on it: what is left of a chunk, and the unit and granule that begins at.
struct Place {
  long long at, end;
  int head, slot, off, seq;
};

// The chunk that a granule of the line belongs to.
__device__ __forceinline__ int chunk_of(const Line &c, long long x) {
  return (int)(((x + 1) * c.blocks - 1) / c.total);
}

// The batch's arrays as the block reads them: its own copies where they fit.
struct BatchArrays {
  const int32_t *starts, *lens;
};

// Find the beginning of the block's chunk: the thread that holds its slot writes
// it to `to` (shared memory), which all may read after a barrier.
template <int ROWS, int GRAN, int NT>
__device__ void seek(const AttendArgs &a, const BatchArrays &ba, const Line &c, Place *to) {
  const long long at = c.total * blockIdx.x / c.blocks;
  const int head = (int)(at / c.per_head);
  long long r = at - head * c.per_head - c.before;
  if (r < 0 || r >= c.mine) return;
  const int per = (a.slots + NT - 1) / NT, s0 = min((int)threadIdx.x * per, a.slots);
  RowTile u;
  int s = s0;
  for (; s < a.slots; s++) {
    const int g = tile_of_slot<ROWS, GRAN>(a, ba.starts, ba.lens, s, u, s > s0);
    if (r < g) break;
    r -= g;
  }
  to->at = at;
  to->end = c.total * (blockIdx.x + 1) / c.blocks;
  to->head = head;
  to->slot = s;
  to->off = (int)r;
  to->seq = u.seq;
}

// One unit's part of a chunk: granules off .. off + take of `units`; the unit
// begins at u0 on the line.
struct Segment {
  RowTile t;
  int head, off, take, units;
  long long u0;
};
// The next one from `p` on (false: the chunk is at its end).
template <int ROWS, int GRAN>
__device__ __forceinline__ bool next_segment(const AttendArgs &a, const BatchArrays &ba, Place &p, Segment &g) {
  while (p.at < p.end && p.head < a.pool.heads) {
    g.t.seq = p.seq;
    const int units = tile_of_slot<ROWS, GRAN>(a, ba.starts, ba.lens, p.slot, g.t, true);
    const int off = p.off, slot = p.slot;
    p.seq = g.t.seq;
    g.head = p.head;
    p.off = 0;
    p.slot++;
    if (p.slot == a.slots) {
      p.slot = p.seq = 0;
      p.head++;
    }
    if (units == 0) {
      // A slot without a tile: one before its sequence's first (rows of q that no
      // sequence has), or one after its last, and then neither has the rest of its.
      constexpr int SH = kRowShift<ROWS>;
      if (p.slot > 0) {
        const int own = slot_base(ba.starts, a.batch.tokens, p.seq, a.group, SH, 1);
        if (slot < own) p.slot = own;
        else p.slot = p.seq + 1 < a.batch.seqs ? max(p.slot, slot_base(ba.starts, a.batch.tokens, p.seq + 1, a.group, SH, 1)) : a.slots;
      }
      if (p.slot >= a.slots) {
        p.slot = p.seq = 0;
        p.head++;
      }
      continue;
    }
    g.off = off;
    g.units = units;
    g.take = (int)min((long long)(units - off), p.end - p.at);
    g.u0 = p.at - off;
    p.at += g.take;
    return true;
  }
  return false;
}

// Lay out the line. All threads call it; NT threads, `sh` shared memory of NT +
// 4 long longs, `copy` of `room` ints for the batch's arrays (each thread
// searches them: from global memory every step of a search would wait for L2).
// False: the block has no work. Starts that descend would give the threads, which
// find their sequences by a search, and the segments, which go on from one to the
// next, lines that differ: such a batch has no work, and the host is told.
template <int ROWS, int GRAN, int NT>
__device__ bool schedule(const AttendArgs &a, int min_gran, long long *sh, int *copy, int room, BatchArrays &ba, Line &c) {
  ba.starts = a.batch.starts;
  ba.lens = a.batch.lens;
  const int seqs = a.batch.seqs;
  if (2 * seqs + 1 <= room) {
    for (int i = threadIdx.x; i < 2 * seqs + 1; i += NT) copy[i] = i <= seqs ? __ldg(ba.starts + i) : __ldg(ba.lens + i - seqs - 1);
    __syncthreads();
    ba.starts = copy;
    ba.lens = copy + seqs + 1;
  }
  int descends = 0;
  for (int i = threadIdx.x; i < seqs; i += NT) descends |= ba.starts[i] > ba.starts[i + 1];
  const int chunk = (a.slots + NT - 1) / NT;
  const int s0 = min((int)threadIdx.x * chunk, a.slots), s1 = min(s0 + chunk, a.slots);
  long long mine = 0;
  RowTile t;
  for (int s = s0; s < s1; s++) mine += tile_of_slot<ROWS, GRAN>(a, ba.starts, ba.lens, s, t, s > s0);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(~0u, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) sh[warp] = sum;
  if (__syncthreads_or(descends)) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && a.err) *a.err = 2;
    return false;
  }
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; w++) {
    const long long v = sh[w];
    if (w < warp) before += v;
    all += v;
  }
  c.before = before + sum - mine;
  c.mine = mine;
  c.per_head = all;
  c.total = all * a.pool.heads;
  if (c.total == 0) return false;
  const long long fit = c.total / min_gran;
  c.blocks = (int)(fit < 1 ? 1 : fit < (long long)gridDim.x ? fit : (long long)gridDim.x);
  __syncthreads();
  return (int)blockIdx.x < c.blocks;
}

// Where chunk `i` keeps its partial: 0 of a unit begun in an earlier chunk, 1 of
// one that begins in it.
template <int ROWS, int DP>
__device__ __forceinline__ float *partial_at(const AttendArgs &a, int i, int which) {
  return a.partials + ((int64_t)i * 2 + which) * (ROWS * (DP + 2));
}

// Four values of a row, divided by the sum l (a row that saw nothing: 0). The
// caller's strides may be odd: one 2- or 4-byte store each where they are.
template <typename T>
__device__ __forceinline__ void write_out(const AttendArgs &a, const RowTile &t, int head, int row, int d, float4 v, float l) {
  const int r = t.row0 + row, tok = t.start + r / a.group, h = head * a.group + r % a.group;
  T *o = static_cast<T *>(a.out) + (int64_t)tok * a.out_token + (int64_t)h * a.out_head + d;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) v = make_float4(0.f, 0.f, 0.f, 0.f);
  v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
  if constexpr (sizeof(T) == 2) {
    const __half2 p = __floats2half2_rn(v.x, v.y), q = __floats2half2_rn(v.z, v.w);
    if (a.out_wide) {
      *reinterpret_cast<uint2 *>(o) = make_uint2(*reinterpret_cast<const uint32_t *>(&p), *reinterpret_cast<const uint32_t *>(&q));
    } else {
      o[0] = p.x; o[1] = p.y; o[2] = q.x; o[3] = q.y;
    }
  } else if (a.out_wide) {
    *reinterpret_cast<float4 *>(o) = v;
  } else {
    o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
  }
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

// Join the partials of chunks i0 .. i0 + n - 1 (the first one's slot is
// `which0`, the others' 0; `step` chunks apart) into `dst` (a partial), or into
// the output when dst is null. NT threads; fac: shared memory of 2 (n + 1) ROWS
// floats. Everything is read with all threads' loads in flight at once: one
// after another, each would wait for L2.
template <typename T, int ROWS, int DP, int NT>
__device__ void join(const AttendArgs &a, const RowTile &t, int head, int i0, int n, int step, int which0, float *dst,
                     float *fac) {
  auto src = [&](int k) -> const float * { return partial_at<ROWS, DP>(a, i0 + k * step, k == 0 ? which0 : 0); };
  float *const ms = fac, *const ls = fac + n * ROWS, *const top = ls + n * ROWS, *const sum = top + ROWS;
  for (int i = threadIdx.x; i < 2 * n * ROWS; i += NT) {
    const int k = (i / ROWS) % n;
    fac[i] = __ldcg(src(k) + ROWS * DP + (i >= n * ROWS ? ROWS : 0) + i % ROWS);
  }
  __syncthreads();
  for (int row = threadIdx.x; row < ROWS; row += NT) {
    float m = -INFINITY;
    for (int k = 0; k < n; k++) m = fmaxf(m, ms[k * ROWS + row]);
    top[row] = m;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * ROWS; i += NT) ms[i] = join_factor(ms[i], top[i % ROWS]);
  __syncthreads();
  for (int row = threadIdx.x; row < ROWS; row += NT) {
    float l = 0.0f;
    for (int k = 0; k < n; k++) l = __fmaf_rn(ms[k * ROWS + row], ls[k * ROWS + row], l);
    sum[row] = l;
    if (dst) {
      dst[ROWS * DP + row] = top[row];
      dst[ROWS * DP + ROWS + row] = l;
    } else if (row < t.rows) {
      write_lse(a, t, head, row, top[row], l);
    }
  }
  __syncthreads();
  // In place where dst is the first partial: a thread reads a value of it before it
  // writes it. Sixteen loads a thread on their way: eight vectors of two partials,
  // or two of eight.
  const int items = t.rows * DP / 4;
  auto vectors = [&](auto per, auto batch) {
    constexpr int V = decltype(per)::value, B = decltype(batch)::value;
    for (int first = threadIdx.x; first < items; first += V * NT) {
      float4 o[V];
#pragma unroll
      for (int e = 0; e < V; e++) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k0 = 0; k0 < n; k0 += B) {
        float4 v[V][B];
#pragma unroll
        for (int j = 0; j < B; j++)
#pragma unroll
          for (int e = 0; e < V; e++) {
            v[e][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + j < n && first + e * NT < items) v[e][j] = __ldcg(reinterpret_cast<const float4 *>(src(k0 + j)) + first + e * NT);
          }
#pragma unroll
        for (int j = 0; j < B; j++)
#pragma unroll
          for (int e = 0; e < V; e++) {
            const float f = k0 + j < n && first + e * NT < items ? ms[(k0 + j) * ROWS + (first + e * NT) / (DP / 4)] : 0.0f;
            o[e].x = __fmaf_rn(f, v[e][j].x, o[e].x);
            o[e].y = __fmaf_rn(f, v[e][j].y, o[e].y);
            o[e].z = __fmaf_rn(f, v[e][j].z, o[e].z);
            o[e].w = __fmaf_rn(f, v[e][j].w, o[e].w);
          }
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        const int i = first + e * NT, row = i / (DP / 4), d = (i % (DP / 4)) * 4;
        if (i >= items) break;
        if (dst) *reinterpret_cast<float4 *>(dst + row * DP + d) = o[e];
        else if (d < a.pool.head_dim) write_out<T>(a, t, head, row, d, o[e], sum[row]);
      }
    }
  };
  if (ROWS >= 128 && n <= 2) vectors(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
  else vectors(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
  __syncthreads();
}

// Called by all threads of a block after it wrote its partial of a segment:
// joins what is complete. `flag`: shared memory.
template <typename T, int ROWS, int DP, int NT>
__device__ void arrive(const AttendArgs &a, const Segment &g, const Line &c, float *fac, unsigned *flag) {
  constexpr int J = kJoin<ROWS>;
  const int i0 = chunk_of(c, g.u0), i1 = chunk_of(c, g.u0 + g.units - 1), n = i1 - i0 + 1;
  auto last = [&](unsigned *ctr, int of) {
    // One thread's fences order the whole block's writes (they come before it at
    // the barrier) and reads: a fence of every thread would wait for the copies
    // that all of them have on the way.
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      *flag = atomicInc(ctr, (unsigned)of - 1) == (unsigned)of - 1;  // wraps to 0
      __threadfence();
    }
    __syncthreads();
    return *flag != 0;
  };
  if (n <= J) {
    if (last(a.counters + i0, n)) join<T, ROWS, DP, NT>(a, g.t, g.head, i0, n, 1, 1, nullptr, fac);
    return;
  }
  const int k = ((int)blockIdx.x - i0) / J, g0 = i0 + k * J, gn = min(J, i1 - g0 + 1);
  const int groups = (n + J - 1) / J;
  // (a group of one needs no count; its chunk's counter may be another unit's)
  if (gn > 1) {
    if (!last(a.counters + g0, gn)) return;
    join<T, ROWS, DP, NT>(a, g.t, g.head, g0, gn, 1, k == 0, partial_at<ROWS, DP>(a, g0, k == 0), fac);
  }
  if (last(a.counters + kAttendMaxBlocks + i0, groups))
    join<T, ROWS, DP, NT>(a, g.t, g.head, i0, groups, J, 1, nullptr, fac);
}

}  // namespace shlo
