// The decoder operators' calls inside the library: rotary positions (rope.cu),
// the 8-bit paged cache (kv_cache.cu) and the attention over it (kv_attend.cu).
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

// Checks of a cache's and a batch's descriptors; `what` names the entry point.
int check_pool(const shlo_kv_pool *p, const char *what);
int check_batch(const shlo_kv_batch *b, const char *what);

int launch_kv_append(const shlo_kv_pool &p, const shlo_kv_batch &b, const void *k, int64_t k_token, int64_t k_head,
                     const void *v, int64_t v_token, int64_t v_head, uint8_t dtype, cudaStream_t st);
int launch_kv_gather(const shlo_kv_pool &p, const int32_t *tables, int64_t table_stride, int32_t seqs,
                     int32_t table_pages, const int32_t *seq, const int32_t *pos, int64_t n, void *k, int64_t k_token,
                     int64_t k_head, void *v, int64_t v_token, int64_t v_head, uint8_t dtype, int sms, cudaStream_t st);

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
