// Products in 8-bit integers on the tensor cores: y = x w^T as tiles of 128 (CG
// blocks: 128 CG) channels by N rows of x, channels along the lanes of tensor
// memory, so that few rows cost no more than the weights' bytes. Both operands
// come by TMA in the 128-byte swizzle, 128 values of K a stage, zeros where the
// matrices end; the sums are 32-bit integers.
//
// One warp asks for the bytes, one issues the products, eight turn sums into
// results: a tile's results are written beside the next tile's products, from the
// other of two places in tensor memory. Where there are few tiles their channels are
// fewer (the products then compute lanes that nobody reads), or a cluster's blocks
// share a tile's K.
//
// Bound: the products for many rows (8192 rows by 8192 channels of 4096 values 162 us,
// 3.4 POP/s), the weights' bytes for few (24 rows by 12288 channels of 4096, 50 MB from
// HBM: 12.4 us, 4.5 us of them launch, ramp and tail; 16 by 50257 of 2048, 103 MB: 20.6
// us), results where K is short (6000 rows by 4000 channels of 64: 21 us, 2.3 TB/s: a
// warp's stores are 64 bytes). Measured and left: every K shared by eight blocks and the
// join's loads one after the other (17.5 us instead of 7.1 for 333 x 1999 to 1001), four
// warps for the results (20.5 us instead of 17.0 for 1024 x 4096 to 4096), a tile's
// place worked out at each copy (13 us instead of 10 for weights in L2, 24 rows).
#include <cuda.h>

#include <algorithm>

#include "decode.cuh"
#include "tensor.cuh"

namespace shlo {

namespace {

constexpr int kK = 128;  // values of K a stage
constexpr int kTileThreads = 320;

struct TileArgs {
  const float *x_scale, *w_scale, *bias;
  void *y;
  int64_t y_row, rows;
  int m, kblocks, ch, ch_tiles, tiles, splits;  // ch: channels a block has of a tile
  int stages, stage_bytes;
  bool after_rows;  // the kernel before rounds x, and may still be at it
  int *err;
};

// A stage is ch rows of weights, then N / CG rows of x. The products read 128 rows
// whatever ch is: what lies behind (any byte is a finite value) goes to lanes that
// nobody reads.
constexpr int kMaxStages = 16;
template <int N, int CG> struct Tile {
  static constexpr int B_BYTES = N / CG * kK;
  static constexpr int TM_COLS = N <= 16 ? 32 : 2 * N;
  static constexpr int ROOM = (N <= 64 ? 112 : 224) * 1024;  // (up to 64 rows: two blocks on an SM)
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_block(uint32_t at, uint32_t rank) {  // an address of shared memory, in another block of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void expect(uint64_t *b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(b)), "r"(bytes) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap *map, int k, int row, uint32_t bar) {
  if (CG == 1)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(k),
                 "r"(row), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(k),
                 "r"(row), "r"(bar)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t add) {
  if (CG == 1)
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 x, {%1, %3};\nmov.b64 y, {%2, %3};\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], x, y, %4, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(add)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 x, {%1, %3};\nmov.b64 y, {%2, %3};\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], x, y, %4, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(add)
        : "memory");
}
template <int CG> __device__ __forceinline__ void commit(uint64_t *b) {
  if (CG == 1)
    tm_commit(b);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_at(b)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tm_ldi(uint32_t at, int (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tm_ldi(uint32_t at, int (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\ntcgen05.wait::ld.sync.aligned;"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }

// CG = 2: a pair of blocks on one tile of 256 channels, whose products the first
// of them issues; each has its 128 channels' weights and half of the rows of x.
// splits > 1 (CG = 1): a cluster's blocks have a part of K each, and add up their
// sums through each other's shared memory.
template <int N, int CG, typename Y>
__global__ void __launch_bounds__(kTileThreads, N <= 64 ? 2 : 1)
k_mul_mat8_tiles(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const TileArgs a) {
  using S = Tile<N, CG>;
  const int ST = a.stages, A_BYTES = a.ch * kK;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t full[kMaxStages], free_[kMaxStages], acc_full[2], acc_free[2], drained;
  __shared__ uint32_t tm_slot;
  __shared__ int gone_word;
  volatile int *const gone = &gone_word;
  uint8_t *const base = raw_smem + ((1024 - (smem_at(raw_smem) & 1023)) & 1023);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int rank = CG == 2 || a.splits > 1 ? (int)cluster_rank() : 0;
  const bool leads = CG == 1 || rank == 0;
  if (tid == 0) {
    for (int i = 0; i < ST; i++) {
      bar_init(full + i, 1);
      bar_init(free_ + i, 1);
    }
    for (int i = 0; i < 2; i++) {
      bar_init(acc_full + i, 1);
      bar_init(acc_free + i, 8 * CG);
    }
    bar_init(&drained, 1);
    gone_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(&tm_slot)), "n"(S::TM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(&tm_slot)), "n"(S::TM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  tm_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tm_after();
  const uint32_t tm = tm_slot;

  const int split = CG == 1 ? rank : 0;
  const int k0 = (int)((int64_t)a.kblocks * split / a.splits), k1 = (int)((int64_t)a.kblocks * (split + 1) / a.splits);
  const int step = gridDim.x / (CG * a.splits), first = blockIdx.x / (CG * a.splits);
  const uint32_t begin = smem_at(base);
  uint32_t asked = 0;  // stages asked for
  if (warp == 0) {
    if (elect_one()) {
      // (a thread's instructions between two copies bound their rate: addresses are sums)
      const uint32_t bar0 = CG == 1 ? smem_at(full) : in_block(smem_at(full), 0);
      auto ch_at = [&](int t) { return (t % a.ch_tiles * CG + (CG == 2 ? rank : 0)) * a.ch; };
      bool on = true;
      // Of the first tile as many weights as there are stages come before x is there.
      const int early = a.after_rows && first < a.tiles ? min(ST, k1 - k0) : 0;
      for (int i = 0, ch = ch_at(first); i < early; i++) {
        if (leads) expect(full + i, CG * a.stage_bytes);
        tma_load<CG>(begin + i * a.stage_bytes, &wmap, (k0 + i) * kK, ch, bar0 + 8 * i);
      }
      if (a.after_rows) cudaGridDependencySynchronize();
      int s = 0;
      uint32_t phase = 1, to = begin, bar = bar0;
      for (int t = first; t < a.tiles && on; t += step) {
        const int ch = ch_at(t), row = t / a.ch_tiles * N + (CG == 2 ? rank * (N / 2) : 0);
        for (int k = k0 * kK; k < k1 * kK; k += kK, asked++) {
          // (the first round finds every stage free)
          if (asked >= (uint32_t)ST && !(on = bar_wait(free_ + s, phase, gone))) break;
          if (asked >= (uint32_t)early) {
            if (leads) expect(full + s, CG * a.stage_bytes);
            tma_load<CG>(to, &wmap, k, ch, bar);
          }
          tma_load<CG>(to + A_BYTES, &xmap, k, row, bar);
          to += a.stage_bytes;
          bar += 8;
          if (++s == ST) s = 0, phase ^= 1, to = begin, bar = bar0;
        }
      }
    }
    asked = __reduce_max_sync(~0u, asked);
  } else if (warp == 1 && leads) {
    if (elect_one()) {
      // sums of 32 bits from signed bytes, both operands with K contiguous
      constexpr uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(N / 8) << 17 | (uint32_t)(128 * CG / 16) << 24;
      // (an operand's upper half never changes, its lower half is a sum)
      const uint32_t at0 = (uint32_t)operand(begin, 16), desc_hi = (uint32_t)(operand(begin, 16) >> 32), b_off = (uint32_t)A_BYTES >> 4;
      uint32_t phase = 0, turn = 0, at = at0;
      int s = 0;
      bool on = true;
      for (int t = first; t < a.tiles && on; t += step, turn++) {
        const uint32_t place = turn & 1;
        if (!(on = bar_wait(acc_free + place, (turn / 2 & 1) ^ 1, gone))) break;
        tm_after();
        uint32_t add = 0;
        for (int k = k0; k < k1; k++) {
          if (!(on = bar_wait(full + s, phase, gone))) break;
          tm_after();
#pragma unroll
          for (int j = 0; j < kK / 32; j++) mma_i8<CG>(tm + place * N, at + 2 * j, at + b_off + 2 * j, desc_hi, idesc, add | j);
          add = 1;
          commit<CG>(free_ + s);
          at += a.stage_bytes >> 4;
          if (++s == ST) s = 0, phase ^= 1, at = at0;
        }
        if (on) commit<CG>(acc_full + place);
      }
      if (!on) {
        commit<CG>(&drained);
        bar_drain(&drained, 0);
      }
    }
  } else if (warp >= 2) {
    if (a.after_rows) cudaGridDependencySynchronize();  // (the rows' scales)
    // Which lanes of tensor memory a warp reads, and which rows of x: half of them.
    constexpr int CHUNK = N >= 64 ? 32 : 16, HALF = N == 16 ? 16 : N / 2;
    const int part = warp % 4, c_lo = (warp - 2) / 4 * HALF, c_hi = min(c_lo + HALF, N);
    uint32_t turn = 0;
    for (int t = first; t < a.tiles; t += step, turn++) {
      const int mine = part * 32 + lane, ch = (t % a.ch_tiles * CG + (CG == 2 ? rank : 0)) * a.ch + mine;
      const int64_t row0 = (int64_t)(t / a.ch_tiles) * N;
      const bool there = mine < a.ch && ch < a.m;
      const float ws = there ? a.w_scale[ch] : 0.0f, b = there && a.bias ? a.bias[ch] : 0.0f;
      const uint32_t place = turn & 1;
      const int have = (int)min((int64_t)N, a.rows - row0);
      float xs[(HALF + 31) / 32];
#pragma unroll
      for (int i = 0; i < (HALF + 31) / 32; i++) xs[i] = c_lo + 32 * i + lane < have ? a.x_scale[row0 + c_lo + 32 * i + lane] : 0.0f;
      if (!warp_wait(acc_full + place, turn / 2 & 1, gone)) break;
      tm_after();
      if (CG == 1 && a.splits > 1) {
        int *const sums = reinterpret_cast<int *>(base);  // [N][128]; all products are done, and all copies with them
        for (int c = c_lo; c < c_hi; c += 16) {
          if (c >= have || part * 32 >= a.ch) break;
          int v[16];
          tm_ldi(tm + ((uint32_t)(part * 32) << 16) + c, v);
#pragma unroll
          for (int j = 0; j < 16; j++) sums[(c + j) * 128 + part * 32 + lane] = v[j];
        }
        break;
      }
      Y *y = static_cast<Y *>(a.y) + (row0 + c_lo) * a.y_row + ch;
#pragma unroll
      for (int i = 0; i < HALF / CHUNK; i++) {
        const int c = c_lo + i * CHUNK;
        if (c >= have || c >= c_hi || part * 32 >= a.ch) break;
        int v[CHUNK];
        tm_ldi(tm + ((uint32_t)(part * 32) << 16) + place * N + c, v);
        float f[CHUNK];
#pragma unroll
        for (int j = 0; j < CHUNK; j++) {
          f[j] = (float)v[j] * __shfl_sync(~0u, xs[i * CHUNK / 32], (i * CHUNK + j) % 32) * ws;
          if (a.bias) f[j] += b;
        }
        if (there) {
          if (c + CHUNK <= have) {
#pragma unroll
            for (int j = 0; j < CHUNK; j++) put(y + j * a.y_row, f[j]);
          } else {
#pragma unroll
            for (int j = 0; j < CHUNK; j++)
              if (c + j < have) put(y + j * a.y_row, f[j]);
          }
        }
        y += CHUNK * a.y_row;
      }
      tm_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 1) bar_arrive(acc_free + place);
        else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_block(smem_at(acc_free + place), 0)) : "memory");
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (*gone && warp == 0 && leads && lane == 0)  // what was asked for lands before the block leaves
    for (uint32_t i = asked > (uint32_t)ST ? asked - ST : 0; i < asked; i++) bar_drain(full + i % ST, i / ST & 1);
  if (CG == 1 && a.splits > 1) {
    cluster_sync();
    if (first < a.tiles && warp >= 2) {
      // Four channels a lane, a row a warp: the blocks take the rows in turn.
      const int at_ch = lane * 4, ch = first % a.ch_tiles * a.ch + at_ch;
      const int64_t row0 = (int64_t)(first / a.ch_tiles) * N;
      const int have = (int)min((int64_t)N, a.rows - row0);
      float ws[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ws[i] = at_ch + i < a.ch && ch + i < a.m ? a.w_scale[ch + i] : 0.0f;
        b[i] = at_ch + i < a.ch && ch + i < a.m && a.bias ? a.bias[ch + i] : 0.0f;
      }
      for (int j = rank + a.splits * (warp - 2); j < have; j += 8 * a.splits) {
        const uint32_t at = smem_at(base) + (uint32_t)(j * 128 + lane * 4) * 4;
        int sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {  // (all on their way at once; splits is uniform)
          if (i >= a.splits) break;
          int v[4];
          asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(in_block(at, i)) : "memory");
#pragma unroll
          for (int l = 0; l < 4; l++) sum[l] += v[l];
        }
        const float xs = a.x_scale[row0 + j];
        Y *const y = static_cast<Y *>(a.y) + (row0 + j) * a.y_row + ch;
#pragma unroll
        for (int l = 0; l < 4; l++) {
          float f = (float)sum[l] * xs * ws[l];
          if (a.bias) f += b[l];
          if (at_ch + l < a.ch && ch + l < a.m) put(y + l, f);
        }
      }
    }
  }
  tm_before();
  __syncwarp();
  __syncthreads();
  if (CG == 2 || a.splits > 1) cluster_sync();
  if (warp == 1) {
    tm_after();
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(S::TM_COLS));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(S::TM_COLS));
  }
  if (tid == 0 && *gone && a.err) *a.err = 1;
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static const EncodeFn f = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
    return (EncodeFn)p;
  }();
  return f;
}

// [rows][n] bytes, read in boxes of 128 by `box` rows.
int encode(CUtensorMap *map, const int8_t *p, int64_t row, int64_t rows, int n, int box) {
  const EncodeFn f = encoder();
  if (!f) return fail("mul_mat8: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(rows > 1 ? row : ((int64_t)n + 15) / 16 * 16)};
  const cuuint32_t boxes[2] = {(cuuint32_t)kK, (cuuint32_t)box}, ones[2] = {1, 1};
  const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)p, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail("mul_mat8: cuTensorMapEncodeTiled: error %d", (int)r);
  return 0;
}

template <int N, int CG, typename Y>
int launch(const Mm8Call &c, int ch, int splits, bool after_rows, int *err, int sms, cudaStream_t st) {
  using S = Tile<N, CG>;
  TileArgs a;
  a.x_scale = c.x_scale; a.w_scale = c.w_scale; a.bias = c.bias; a.y = c.y; a.y_row = c.y_row; a.rows = c.rows;
  a.m = c.m;
  a.kblocks = (c.n + kK - 1) / kK;
  a.ch = CG == 2 ? 128 : ch;
  a.ch_tiles = (c.m + a.ch * CG - 1) / (a.ch * CG);
  const int64_t tiles = (int64_t)a.ch_tiles * ((c.rows + N - 1) / N);
  if (tiles > (1 << 30)) return fail("mul_mat8: %lld rows by %d channels", (long long)c.rows, c.m);
  a.tiles = (int)tiles;
  a.splits = splits;
  a.after_rows = after_rows;
  a.err = err;
  a.stage_bytes = a.ch * kK + S::B_BYTES;
  const int beyond = (128 - a.ch) * kK;  // what the products read behind the last stage's weights
  a.stages = std::min(kMaxStages, (S::ROOM - 1024 - beyond) / a.stage_bytes);
  const int bytes = 1024 + beyond + std::max(a.stages * a.stage_bytes, splits > 1 ? N * 512 : 0);
  CUtensorMap wmap, xmap;
  SHLO_TRY(encode(&wmap, c.w, c.w_row, c.m, c.n, a.ch));
  SHLO_TRY(encode(&xmap, (const int8_t *)c.x, c.x_row, c.rows, c.n, N / CG));
  const auto kernel = k_mul_mat8_tiles<N, CG, Y>;
  static std::atomic<uint64_t> set{0};
  int device;
  SHLO_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !(set.load(std::memory_order_relaxed) >> device & 1)) {
    SHLO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::ROOM));
    if (device < 64) set.fetch_or(1ull << device);
  }
  const int per = CG * splits, slots = sms * (N <= 64 ? 2 : 1) / per;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((splits > 1 ? a.tiles : std::min(a.tiles, slots)) * per));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (per > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = per;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  if (after_rows) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs++;
  }
  SHLO_CUDA(cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, a));
  return launch_check("mul_mat8");
}

// Which tiles: the shape whose estimate in cycles is the smallest. A stage of 128
// values takes a block 100 cycles and 2.4 a row of either side (two blocks on an SM
// share the first), up to 520, which copies and products side by side reach; the pair
// 620. Blocks that share a tile's K cost 75 cycles a row for their join, and a tile's
// results 12. Measured in us, weights from HBM, N / ch / splits:
//   1 x 4096 to 4096     16/128/4 8.2   16/64/2 8.8   16/48/1 9.0   16/128/1 10.8
//   24 x 4096 to 12288   32/88/1 12.9   32/128/1 13.7   32/88/2 13.9
//   128 x 4096 to 4096   32/64/1 11.0   64/64/1 11.5   64/128/4 12.1   128/128/4 13.8
//   333 x 1999 to 1001   64/64/1 8.0   64/128/1 9.4   64/128/4 9.9   256 rows, 8 splits 17.5
//   32 x 16384 to 1024   32/64/8 10.0   16/64/8 10.4   32/128/1 29.8
//   1000 x 8192 to 8192  the pair 52.6   128/128/1 71   64/128/1 90
struct Shape {
  int n, ch, splits;
};
Shape choose(const Mm8Call &c, int sms) {
  const int64_t kblocks = (c.n + kK - 1) / kK;
  Shape best{256, 128, 1};
  auto tiles = [&](int n, int ch) { return (c.rows + n - 1) / n * ((c.m + ch - 1) / ch); };
  int64_t least = INT64_MAX;
  if (c.rows > 128) {
    const int64_t turns = (2 * tiles(256, 256) + sms - 1) / sms;
    least = turns * (kblocks * 620 + 256 * 20);
  }
  for (int n = 16; n <= 128; n *= 2) {
    if (n < 128 && c.rows > 8 * n) continue;      // (many narrow tiles read the weights again and again)
    if (n > 16 && c.rows <= n / 2) break;
    for (const int ch : {128, 88, 64, 48, 32}) {
      const int64_t t = tiles(n, ch);
      for (int splits = 1; splits <= 8 && (splits == 1 || (t * splits <= 2 * sms && kblocks >= 2 * splits)); splits *= 2) {
        const int64_t turns = (t * splits + sms - 1) / sms, k = (kblocks + splits - 1) / splits;
        const int64_t fixed = 100 * (n <= 64 ? (turns + 1) / 2 : turns), each = std::min((int64_t)24 * (ch + n) / 10, (int64_t)420);
        const int64_t cost = k * (turns * each + fixed) + turns * n * 12 + (splits > 1 ? 75 * n : 0);
        if (cost < least) least = cost, best = Shape{n, ch, splits};
      }
    }
  }
  return best;
}

template <typename Y>
int launch_for(const Mm8Call &c, bool after_rows, int *err, int sms, cudaStream_t st) {
  const Shape s = choose(c, sms);
  switch (s.n) {
    case 16: return launch<16, 1, Y>(c, s.ch, s.splits, after_rows, err, sms, st);
    case 32: return launch<32, 1, Y>(c, s.ch, s.splits, after_rows, err, sms, st);
    case 64: return launch<64, 1, Y>(c, s.ch, s.splits, after_rows, err, sms, st);
    case 128: return launch<128, 1, Y>(c, s.ch, s.splits, after_rows, err, sms, st);
    default: return launch<256, 2, Y>(c, 128, 1, after_rows, err, sms, st);
  }
}

}  // namespace

int launch_mul_mat8_tiles(const Mm8Call &c, bool after_rows, int *err, int sms, cudaStream_t st) {
  return c.dtype == kF16 ? launch_for<__half>(c, after_rows, err, sms, st) : launch_for<float>(c, after_rows, err, sms, st);
}

}  // namespace shlo
