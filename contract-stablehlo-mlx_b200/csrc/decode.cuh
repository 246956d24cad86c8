// The decoder operators' calls inside the library: rotary positions (rope.cu),
// the 8-bit paged cache (kv_cache.cu) and the attention over it (kv_attend.cu),
// the norm of queries and keys with the rotation (norm_rope.cu), products in 8-bit
// integers (linear8.cu, linear8_tiles.cu), beam search's selection (beam.cu) and the
// reordering of the cache after it (kv_fork.cu).
// The C entry points on caller-owned memory and those on arrays both end here.
#pragma once

#include "common.cuh"

namespace shlo {

struct RopeCall {
  const void *x;
  int64_t x_token, x_head;
  const int32_t *positions;
  const int64_t *phases;
  void *y;
  int64_t y_token, y_head;
  int64_t tokens;
  int32_t heads, dim, rot;
  uint8_t dtype;
  uint32_t flags;
  float factor;
};
int launch_rope(const RopeCall &c, int sms, cudaStream_t st);
// y [tokens][heads][dim] is x itself with its strides, or shares no value with it.
int check_in_place(const void *x, int64_t x_token, int64_t x_head, const void *y, int64_t y_token, int64_t y_head, int64_t tokens,
                   int64_t heads, int64_t dim, size_t size, const char *what, const char *x_name, const char *y_name);
// Whether rows of `bytes` bytes, `step` apart, at p share memory with those at q. (Rows
// side by side in one buffer do not.)
inline bool meet(const void *p, int64_t rows, int64_t step, int64_t bytes, const void *q, int64_t q_rows, int64_t q_step, int64_t q_bytes) {
  if (!p || !q || rows < 1 || q_rows < 1) return false;
  if (rows == 1) step = q_rows > 1 ? q_step : 0;
  if (q_rows == 1) q_step = step;
  const int64_t off = (intptr_t)q - (intptr_t)p;
  auto low = [](int64_t n, int64_t s) { return s < 0 ? (double)(n - 1) * s : 0.0; };
  auto high = [](int64_t n, int64_t s) { return s > 0 ? (double)(n - 1) * s : 0.0; };
  if ((double)off + low(q_rows, q_step) >= high(rows, step) + bytes || (double)off + high(q_rows, q_step) + q_bytes <= low(rows, step)) return false;
  if (step != q_step || step < 1) return true;
  const int64_t at = (off % step + step) % step;
  return at < bytes || at + q_bytes > step;
}
inline bool meet(const void *p, int64_t bytes, const void *q, int64_t q_bytes) { return meet(p, 1, 0, bytes, q, 1, 0, q_bytes); }
// The same of [tokens][heads] rows at p, and `q_bytes` bytes at q.
inline bool meet(const void *p, int64_t tokens, int64_t token, int64_t heads, int64_t head, int64_t bytes, const void *q, int64_t q_bytes) {
  if (!p || !q || tokens < 1 || heads < 1) return false;
  const char *x = static_cast<const char *>(p);
  if (token < 0) x += (tokens - 1) * token, token = -token;
  if (head < 0) x += (heads - 1) * head, head = -head;
  const double off = (double)((intptr_t)q - (intptr_t)x);
  if (off >= (double)(tokens - 1) * token + (double)(heads - 1) * head + bytes || off + q_bytes <= 0.0) return false;
  const bool by_heads = heads <= tokens;  // the shorter axis is gone through
  for (int64_t i = 0; i < (by_heads ? heads : tokens); i++)
    if (by_heads ? meet(x + i * head, tokens, token, bytes, q, 1, 0, q_bytes) : meet(x + i * token, heads, head, bytes, q, 1, 0, q_bytes)) return true;
  return false;
}

// (dy: the gradient)
using NormRopeCall = shlo_norm_rope_args;
size_t norm_rope_work_bytes(int sms);
// A call's operands from arrays, without its result; p: the "shlo_norm_rope" kernel's words.
int norm_rope_call(const char *what, Arr *x, Arr *positions, Arr *phases, Arr *q_weight, Arr *k_weight, const uint32_t *p, NormRopeCall *c);
int launch_norm_rope(const NormRopeCall &c, bool back, int sms, cudaStream_t st);

// Products in 8-bit integers (linear8.cu, linear8_tiles.cu): y = x w^T, scaled.
using Mm8Call = shlo_mul_mat8_args;
// `fill`: zeros behind a row's last value up to a multiple of 16.
int launch_quantise_rows(const void *x, int64_t x_row, uint8_t dtype, int64_t rows, int32_t n, int8_t *q, int64_t q_row, float *scale,
                         bool fill, const char *what, cudaStream_t st);
// `after_rows`: the launch before it on the stream is the one that rounds its x. `err`:
// the device's word for launches that gave up a wait.
int launch_mul_mat8(const Mm8Call &c, bool after_rows, int *err, int sms, cudaStream_t st);
int launch_mul_mat8_tiles(const Mm8Call &c, bool after_rows, int *err, int sms, cudaStream_t st);  // (arguments checked)
size_t linear8_work_bytes(int64_t rows, int32_t n);
int launch_linear8(const Mm8Call &c, int *err, int sms, cudaStream_t st);

// Beam search (beam.cu).
using BeamCall = shlo_beam_args;
size_t beam_work_bytes(int64_t rows, int32_t keep, int32_t vocab);
int launch_beam_select(const BeamCall &c, int sms, cudaStream_t st);

// Checks of a cache's and a batch's descriptors; `what` names the entry point.
int check_pool(const shlo_kv_pool *p, const char *what);
int check_batch(const shlo_kv_batch *b, const char *what);

int launch_kv_append(const shlo_kv_pool &p, const shlo_kv_batch &b, const void *k, int64_t k_token, int64_t k_head,
                     const void *v, int64_t v_token, int64_t v_head, uint8_t dtype, cudaStream_t st);
int launch_kv_gather(const shlo_kv_pool &p, const int32_t *tables, int64_t table_stride, int32_t seqs,
                     int32_t table_pages, const int32_t *seq, const int32_t *pos, int64_t n, void *k, int64_t k_token,
                     int64_t k_head, void *v, int64_t v_token, int64_t v_head, uint8_t dtype, int sms, cudaStream_t st);

int launch_kv_fork(const shlo_kv_pool &p, const shlo_kv_fork_args &c, cudaStream_t st);

struct AttendCall {
  shlo_kv_pool pool;
  shlo_kv_batch batch;
  const void *q;
  int64_t q_token, q_head;
  void *out;
  int64_t out_token, out_head;
  float *lse;  // [tokens][heads], or nullptr
  int32_t heads;
  uint8_t dtype;
  float scale;
  bool causal;
  int32_t window;
  void *work;
  size_t work_bytes;
  int *err;  // the device's word for launches that gave up a wait
};
size_t attend_work_bytes(int sms);
int launch_kv_attend(const AttendCall &c, int sms, int device, cudaStream_t st);

// The new tokens of sequence s and its length, with the caller's arrays held
// to the batch: starts to [0, tokens], the length to 0 and above. `starts` and
// `lens` are the batch's arrays or a block's copies of them.
struct SeqSpan {
  int start, n, len;
};
__device__ __forceinline__ SeqSpan seq_span(const int32_t *starts, const int32_t *lens, int tokens, int s) {
  SeqSpan r;
  r.start = min(max(starts[s], 0), tokens);
  r.n = max(min(max(starts[s + 1], 0), tokens) - r.start, 0);
  r.len = max(lens[s], 0);
  return r;
}
// Slots: sequence s has those from starts[s] * num / 2^shift + extra * s on.
__device__ __forceinline__ int slot_base(const int32_t *starts, int tokens, int s, int num, int shift, int extra) {
  const int64_t at = min(max(starts[s], 0), tokens);
  return (int)((at * num) >> shift) + extra * s;
}
// The owner of a slot: the last sequence, from `lo` on, whose first is not above it.
__device__ __forceinline__ int slot_owner(const int32_t *starts, int tokens, int seqs, int lo, int slot, int num, int shift,
                                          int extra) {
  int hi = seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (slot_base(starts, tokens, mid, num, shift, extra) <= slot) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace shlo
