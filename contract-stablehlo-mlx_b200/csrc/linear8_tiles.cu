// Products in 8-bit integers on the tensor cores: y = x w^T as tiles of 128 (CG
// blocks: 128 CG) channels by N rows of x, channels along the lanes of tensor
// memory, so that few rows cost no more than the weights' bytes. Both operands
// come by TMA in the 128-byte swizzle, 128 values of K a stage, zeros where the
// matrices end; the sums are 32-bit integers.
//
// One warp asks for the bytes, one issues the products, four turn sums into
// results: a tile's results are written beside the next tile's products, from the
// other of two places in tensor memory.
#include <cuda.h>

#include <algorithm>

#include "decode.cuh"
#include "tensor.cuh"

namespace shlo {

namespace {

constexpr int kK = 128;  // values of K a stage
constexpr int kTileThreads = 192;

struct TileArgs {
  const float *x_scale, *w_scale, *bias;
  void *y;
  int64_t y_row, rows;
  int m, kblocks, ch_tiles, tiles, splits;
  int *err;
};

template <int N, int CG> struct Tile {
  static constexpr int A_BYTES = 128 * kK, B_BYTES = N / CG * kK, STAGE = A_BYTES + B_BYTES;
  // (up to 64 rows: two blocks on an SM)
  static constexpr int STAGES = N <= 64 ? 100 * 1024 / STAGE : 200 * 1024 / STAGE;
  static constexpr int BYTES = 1024 + STAGES * STAGE;
  static constexpr int TM_COLS = N <= 16 ? 32 : 2 * N;
  static_assert(N * 512 <= STAGES * STAGE, "a block's sums in the stages' place");
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
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if (CG == 1)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
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
  constexpr int ST = S::STAGES;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t full[ST], free_[ST], acc_full[2], acc_free[2], drained;
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
      bar_init(acc_free + i, 4 * CG);
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
  uint32_t asked = 0;  // stages asked for
  if (warp == 0) {
    if (elect_one()) {
      bool on = true;
      for (int t = first; t < a.tiles && on; t += step) {
        const int ch = (t % a.ch_tiles * CG + (CG == 2 ? rank : 0)) * 128, row = t / a.ch_tiles * N + (CG == 2 ? rank * (N / 2) : 0);
        for (int k = k0; k < k1; k++, asked++) {
          const uint32_t s = asked % ST;
          if (!(on = bar_wait(free_ + s, (asked / ST & 1) ^ 1, gone))) break;
          if (leads) expect(full + s, CG * S::STAGE);
          const uint32_t to = smem_at(base) + s * S::STAGE, bar = CG == 1 ? smem_at(full + s) : in_block(smem_at(full + s), 0);
          tma_load<CG>(to, &wmap, k * kK, ch, bar);
          tma_load<CG>(to + S::A_BYTES, &xmap, k * kK, row, bar);
        }
      }
    }
    asked = __reduce_max_sync(~0u, asked);
  } else if (warp == 1 && leads) {
    if (elect_one()) {
      // sums of 32 bits from signed bytes, both operands with K contiguous
      constexpr uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(N / 8) << 17 | (uint32_t)(128 * CG / 16) << 24;
      uint32_t it = 0, turn = 0;
      bool on = true;
      for (int t = first; t < a.tiles && on; t += step, turn++) {
        const uint32_t place = turn & 1;
        if (!(on = bar_wait(acc_free + place, (turn / 2 & 1) ^ 1, gone))) break;
        tm_after();
        for (int k = k0; k < k1; k++, it++) {
          const uint32_t s = it % ST;
          if (!(on = bar_wait(full + s, it / ST & 1, gone))) break;
          tm_after();
          const uint32_t at = smem_at(base) + s * S::STAGE;
          const uint64_t da = operand(at, 16), db = operand(at + S::A_BYTES, 16);
#pragma unroll
          for (int j = 0; j < kK / 32; j++) mma_i8<CG>(tm + place * N, da + 2 * j, db + 2 * j, idesc, k > k0 || j);
          commit<CG>(free_ + s);
        }
        if (on) commit<CG>(acc_full + place);
      }
      if (!on) {
        commit<CG>(&drained);
        bar_drain(&drained, 0);
      }
    }
  } else if (warp >= 2) {
    const int part = warp % 4;  // which lanes of tensor memory a warp reads
    uint32_t turn = 0;
    for (int t = first; t < a.tiles; t += step, turn++) {
      const int ch = (t % a.ch_tiles * CG + (CG == 2 ? rank : 0)) * 128 + part * 32 + lane;
      const int64_t row0 = (int64_t)(t / a.ch_tiles) * N;
      const float ws = ch < a.m ? a.w_scale[ch] : 0.0f, b = ch < a.m && a.bias ? a.bias[ch] : 0.0f;
      const uint32_t place = turn & 1;
      if (!warp_wait(acc_full + place, turn / 2 & 1, gone)) break;
      tm_after();
      const int have = (int)min((int64_t)N, a.rows - row0);
      if (CG == 1 && a.splits > 1) {
        int *const sums = reinterpret_cast<int *>(base);  // [N][128]; all products are done, and all copies with them
        for (int c = 0; c < N; c += 16) {
          if (c >= have) break;
          int v[16];
          tm_ldi(tm + ((uint32_t)(part * 32) << 16) + c, v);
#pragma unroll
          for (int j = 0; j < 16; j++) sums[(c + j) * 128 + part * 32 + lane] = v[j];
        }
        break;
      }
      Y *y = static_cast<Y *>(a.y) + row0 * a.y_row + ch;
      for (int c = 0; c < N; c += 16) {
        if (c >= have) break;
        const float xs = c + lane % 16 < have ? a.x_scale[row0 + c + lane % 16] : 0.0f;
        int v[16];
        tm_ldi(tm + ((uint32_t)(part * 32) << 16) + place * N + c, v);
#pragma unroll
        for (int j = 0; j < 16; j++) {
          float f = (float)v[j] * __shfl_sync(~0u, xs, j) * ws;
          if (a.bias) f += b;
          if (c + j < have && ch < a.m) put(y, f);
          y += a.y_row;
        }
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
    for (uint32_t i = asked > ST ? asked - ST : 0; i < asked; i++) bar_drain(full + i % ST, i / ST & 1);
  if (CG == 1 && a.splits > 1) {
    cluster_sync();
    if (first < a.tiles && warp >= 2) {
      const int c = tid - 64, ch = first % a.ch_tiles * 128 + c;
      const int64_t row0 = (int64_t)(first / a.ch_tiles) * N;
      const int have = (int)min((int64_t)N, a.rows - row0);
      const float ws = ch < a.m ? a.w_scale[ch] : 0.0f, b = ch < a.m && a.bias ? a.bias[ch] : 0.0f;
      for (int j = rank; j < have; j += a.splits) {
        int sum = 0;
        const uint32_t at = smem_at(base) + (uint32_t)(j * 128 + c) * 4;
        for (int i = 0; i < a.splits; i++) {
          int v;
          asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(in_block(at, i)) : "memory");
          sum += v;
        }
        float f = (float)sum * a.x_scale[row0 + j] * ws;
        if (a.bias) f += b;
        if (ch < a.m) put(static_cast<Y *>(a.y) + (row0 + j) * a.y_row + ch, f);
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
int launch(const Mm8Call &c, int splits, int sms, cudaStream_t st) {
  using S = Tile<N, CG>;
  CUtensorMap wmap, xmap;
  SHLO_TRY(encode(&wmap, c.w, c.w_row, c.m, c.n, 128));
  SHLO_TRY(encode(&xmap, c.x, c.x_row, c.rows, c.n, N / CG));
  TileArgs a;
  a.x_scale = c.x_scale; a.w_scale = c.w_scale; a.bias = c.bias; a.y = c.y; a.y_row = c.y_row; a.rows = c.rows;
  a.m = c.m;
  a.kblocks = (c.n + kK - 1) / kK;
  a.ch_tiles = (c.m + 128 * CG - 1) / (128 * CG);
  a.tiles = a.ch_tiles * (int)((c.rows + N - 1) / N);
  a.splits = splits;
  a.err = c.err;
  const auto kernel = k_mul_mat8_tiles<N, CG, Y>;
  static std::atomic<uint64_t> set{0};
  int device;
  SHLO_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !(set.load(std::memory_order_relaxed) >> device & 1)) {
    SHLO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
    if (device < 64) set.fetch_or(1ull << device);
  }
  const int per = CG * splits, slots = sms * (N <= 64 ? 2 : 1) / per;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((splits > 1 ? a.tiles : std::min(a.tiles, slots)) * per));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = S::BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = per;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = per > 1 ? 1 : 0;
  SHLO_CUDA(cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, a));
  return launch_check("mul_mat8");
}

template <typename Y>
int choose(const Mm8Call &c, int sms, cudaStream_t st) {
  const int kblocks = (c.n + kK - 1) / kK, ch = (c.m + 127) / 128;
  const int N = c.rows <= 16 ? 16 : c.rows <= 32 ? 32 : c.rows <= 64 ? 64 : c.rows <= 128 ? 128 : 256;
  const int64_t tiles = ch * ((c.rows + N - 1) / N);
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= sms && kblocks >= 4 * splits) splits *= 2;
  switch (N) {
    case 16: return launch<16, 1, Y>(c, splits, sms, st);
    case 32: return launch<32, 1, Y>(c, splits, sms, st);
    case 64: return launch<64, 1, Y>(c, splits, sms, st);
    case 128: return launch<128, 1, Y>(c, splits, sms, st);
    default:
      if (splits > 1) return launch<256, 1, Y>(c, splits, sms, st);
      return launch<256, 2, Y>(c, 1, sms, st);
  }
}

}  // namespace

int launch_mul_mat8_tiles(const Mm8Call &c, int sms, cudaStream_t st) {
  return c.dtype == kF16 ? choose<__half>(c, sms, st) : choose<float>(c, sms, st);
}

}  // namespace shlo
