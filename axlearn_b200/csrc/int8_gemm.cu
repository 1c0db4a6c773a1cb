// y[M, N] = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k] (+ y) of 8-bit whole numbers on CTA pairs (`gemm_2cta.cu` is the same
// division of work for bf16): sums are 32-bit integers in tensor memory, exact for K up to 2^17.  A sum above 2^24 is rounded on its
// way to fp32, as are its products with the two scales; behind that comes the rounding to y.
//
// Two CTAs on neighbouring SMs share a tile of 256 rows.  Each stages its own 128 rows of x and its own half of the tile's
// features, 128 values of K a stage; one thread of the first CTA issues `tcgen05.mma.cta_group::2.kind::i8`; both drain their
// 128 rows: a thread owns a row of x, so its scale is one register, and the features' scales are loads that a warp shares.
// The next tile runs into the other half of tensor memory meanwhile.
//
// Measured: 8192 x 4096 x 22016 441 to 465 us on a cool GPU (444 at twice the measured rate of bf16) and 520 for as long as one likes,
// under the power cap; 333 x 2048 x 8192 12.2 us (3.5): one wave of 64 tiles of 256 x 256 for 74 pairs, of whose 512 rows 333 are
// there.  In a row of calls 333 x K x 8192 takes 7.6 us at K = 128 and 2.5 for each 1024 of K (13.3 at 2048): what lies beside the MMAs is
// the launch, the pair's barriers and tensor memory, the first loads, and the drain of a tile, 128 features a warp.
#include "chain.cuh"
#include "cta_pair.cuh"
#include "host_utils.cuh"
#include "int8.cuh"
#include "opt_in.cuh"
#include "sm100.cuh"

namespace axb {

constexpr int kI8Rows = 128, kI8K = 128;  // rows of x a CTA, values of K a stage
constexpr int kI8Epilogue = 8;            // warps: two for each quarter of the rows, one for either half of the features
constexpr int kI8Threads = 32 * (2 + kI8Epilogue);  // + producer, issuer

template <int TN>  // features of a tile
struct Int8PairCfg {
  static constexpr int kHalf = TN / 2;
  static constexpr int kABytes = kI8Rows * kI8K, kBBytes = kHalf * kI8K, kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = TN == 256 ? 6 : 8;
  static constexpr int kStagingPerWarp = 4096;  // 32 rows x 64 features
  static constexpr int kRingBytes = kStages * kStageBytes, kStagingBytes = kI8Epilogue * kStagingPerWarp;
  static constexpr int kScaleBytes = TN * 4;  // of the features
  static constexpr int kSmem = kRingBytes + kStagingBytes + kScaleBytes + 512 + 1024;  // barriers, alignment slack
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct Int8GemmParams {
  int M, N, K;
  int accumulate;
  const float *x_scales, *w_scales;
  __nv_bfloat16* y;
  int64_t ldy;
  int* status;
  int group_m;  // row blocks of a rasterisation group
};

template <int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8Threads, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_y, Int8GemmParams p) {
  using S = Int8PairCfg<TN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  // (The window starts at the same offset in both CTAs, so both have the same layout.)
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* staging = smem + S::kRingBytes;
  float* feature_scales = reinterpret_cast<float*>(staging + S::kStagingBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + S::kStagingBytes + S::kScaleBytes);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* tmem_full = empty_bar + kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1), num_pairs = static_cast<int>(gridDim.x >> 1);
  const int m_blocks = (p.M + 2 * kI8Rows - 1) / (2 * kI8Rows), n_blocks = (p.N + TN - 1) / TN;
  const int num_tiles = m_blocks * n_blocks;
  const int num_kb = (p.K + kI8K - 1) / kI8K;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_y);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * kI8Epilogue);  // the epilogue warps of both CTAs
    }
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * TN);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before anyone signals across the pair
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  // Row block fastest within a group of `group_m` of them, so that a wave's operands stay in the L2.
  auto tile_at = [&](int t, int& m_blk, int& n_blk) {
    const int per_group = p.group_m * n_blocks, first_m = t / per_group * p.group_m, r = t % per_group;
    const int size = min(m_blocks - first_m, p.group_m);
    m_blk = first_m + r % size;
    n_blk = r / size;
  };

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        int m_blk, n_blk;
        tile_at(t, m_blk, n_blk);
        const int m0 = m_blk * 2 * kI8Rows + static_cast<int>(rank) * kI8Rows;
        const int n0 = n_blk * TN + static_cast<int>(rank) * S::kHalf;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.status, kStatusWaitTimeoutProducer)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * S::kStageBytes;
          // The first CTA's barrier counts the bytes of both CTAs.
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * S::kStageBytes);
          const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          tma_load_2d_pair(sa, &map_x, bar, kb * kI8K, m0);
          tma_load_2d_pair(sa + S::kABytes, &map_w, bar, kb * kI8K, n0);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      constexpr uint32_t idesc = umma_idesc_i8(2 * kI8Rows, TN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        if (!mbar_wait(&tmem_empty[acc], acc_phase ^ 1, p.status, kStatusWaitTimeoutMma)) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, p.status, kStatusWaitTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + stage * S::kStageBytes), sb = sa + S::kABytes;
#pragma unroll
          for (int k = 0; k < kI8K / 32; ++k)
            tc_mma_i8_pair(d_tmem, umma_smem_desc(sa + k * 32, 16, 1024), umma_smem_desc(sb + k * 32, 16, 1024), idesc,
                           (kb > 0 || k > 0) ? 1u : 0u);
          // The stage is free in BOTH CTAs once these MMAs retire.
          const uint32_t eb = smem_u32(&empty_bar[stage]);
          tc_commit_pair(eb);
          tc_commit_pair(map_to_cta(eb, 1));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) {
          const uint32_t fb = smem_u32(&tmem_full[acc]);
          tc_commit_pair(fb);
          tc_commit_pair(map_to_cta(fb, 1));
        }
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    const int quarter = warp & 3, side = (warp - 2) >> 2;  // tensor-memory lanes [32 * quarter, +32), either half of the columns
    const int thread = threadIdx.x - 64;
    uint8_t* tile = staging + (warp - 2) * S::kStagingPerWarp;
    const uint32_t empty_addr = map_to_cta(smem_u32(&tmem_empty[0]), 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles; t += num_pairs) {
      int m_blk, n_blk;
      tile_at(t, m_blk, n_blk);
      const int row0 = m_blk * 2 * kI8Rows + static_cast<int>(rank) * kI8Rows + quarter * 32, n0 = n_blk * TN;
      const bool inside = row0 + lane < p.M;
      const float xs = inside ? p.x_scales[row0 + lane] : 0.f;
      // (All epilogue warps pass these barriers for every tile, also behind a wait that gave up.)
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kI8Epilogue) : "memory");  // the tile before has been multiplied by its scales
      if (thread < TN && n0 + thread < p.N) feature_scales[thread] = p.w_scales[n0 + thread];
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kI8Epilogue) : "memory");
      if (ok) ok = mbar_wait_warp_relaxed(&tmem_full[acc], acc_phase, p.status, kStatusWaitTimeoutEpilogue);
      if (!ok) continue;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * TN;
#pragma unroll 1
      for (int ch = side * (TN / 128); ch < (side + 1) * (TN / 128); ++ch) {
        const int n = n0 + ch * 64;
        // The staging tile was read by the store issued a chunk ago.
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + ch * 64 + half * 32, r);
          const float4* ws = reinterpret_cast<const float4*>(feature_scales + ch * 64 + half * 32);
          tmem_ld_wait();
          if (ch == (side + 1) * (TN / 128) - 1 && half == 1) {
            // All of this warp's reads of the accumulator are done: hand it back early.
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_addr + acc * 8);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 w4 = ws[2 * v + (i >> 2)];
              const float w = (i & 3) == 0 ? w4.x : (i & 3) == 1 ? w4.y : (i & 3) == 2 ? w4.z : w4.w;
              f[i] = __int2float_rn(static_cast<int>(r[8 * v + i])) * xs * w;
            }
            if (p.accumulate && inside && n + half * 32 + v * 8 < p.N) {
              const uint4 old = *reinterpret_cast<const uint4*>(p.y + static_cast<int64_t>(row0 + lane) * p.ldy + n + half * 32 + v * 8);
              const uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                f[2 * i] += __uint_as_float(o[i] << 16);
                f[2 * i + 1] += __uint_as_float(o[i] & 0xffff0000u);
              }
            }
            // 128-byte swizzle: 16-byte unit j of row `lane` lives at unit j ^ (lane & 7).
            *reinterpret_cast<uint4*>(tile + lane * 128 + (((half * 4 + v) ^ (lane & 7)) << 4)) =
                make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          if (row0 < p.M && n < p.N) tma_store_2d(&map_y, tile, n, row0);
          tma_store_commit();
        }
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) tma_store_wait<0>();
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1 && p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != 0) {
    // A wait gave up: let copies that may still be in flight land before the CTAs exit.
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  // Neither CTA may exit (or free tensor memory) while its partner can still touch it.
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 2 * TN);
  }
}

template <int TN>
static int launch_int8_pair(const void* x, const void* w, int64_t ldx, int64_t ldw, const Int8GemmParams& p, cudaStream_t stream) {
  using S = Int8PairCfg<TN>;
  CUtensorMap mx, mw, my;
  const uint64_t m = static_cast<uint64_t>(p.M), n = static_cast<uint64_t>(p.N), k = static_cast<uint64_t>(p.K);
  const uint64_t x_dims[2] = {k, m}, w_dims[2] = {k, n}, y_dims[2] = {n, m};
  const uint64_t x_pitch[1] = {static_cast<uint64_t>(ldx)}, w_pitch[1] = {static_cast<uint64_t>(ldw)};
  const uint64_t y_pitch[1] = {static_cast<uint64_t>(p.ldy) * 2};
  const uint32_t x_box[2] = {kI8K, kI8Rows}, w_box[2] = {kI8K, S::kHalf}, y_box[2] = {64, 32};
  int rc = make_tensor_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, x, x_dims, x_pitch, x_box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == 0) rc = make_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, w_dims, w_pitch, w_box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == 0) rc = make_tensor_map(&my, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.y, y_dims, y_pitch, y_box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != 0) return rc;
  constexpr auto kernel = int8_pair_kernel<TN>;
  static OptIn opt_in;
  if (!opt_in.done(kernel, S::kSmem)) return -3;
  const int64_t tiles = static_cast<int64_t>((p.M + 2 * kI8Rows - 1) / (2 * kI8Rows)) * ((p.N + TN - 1) / TN);
  const int pairs = static_cast<int>(tiles < sm_count() / 2 ? tiles : sm_count() / 2);
  kernel<<<2 * pairs, kI8Threads, S::kSmem, stream>>>(mx, mw, my, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace axb

// y[M, N] of x [M, K] and w [N, K], all one row behind the other and 16-byte aligned; N a multiple of 8, K one of 16 and at most
// 2^17.  `plan`: features of a tile, 256 or 128.  -10: not supported.
extern "C" int axb_int8_gemm(const axb::Int8LinearCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8LinearCall& a = *call;
  if (a.M <= 0 || a.N <= 0) return 0;
  if (a.K < 16 || a.K > (1 << 17) || a.K % 16 || a.N % 8 || (a.plan != 256 && a.plan != 128) || a.M > 0x40000000 || a.N > 0x40000000)
    return -10;
  for (const void* x : {a.x, a.w, static_cast<const void*>(a.y), static_cast<const void*>(a.w_scales)})
    if (reinterpret_cast<uintptr_t>(x) & 15) return -10;
  if ((a.M + 255) / 256 * ((a.N + a.plan - 1) / a.plan) > 0x7fffff00) return -10;
  const Int8GemmParams p{static_cast<int>(a.M), static_cast<int>(a.N), static_cast<int>(a.K), a.accumulate != 0,
                         a.x_scales, a.w_scales, static_cast<__nv_bfloat16*>(a.y), a.N, a.status, 8};
  return a.plan == 256 ? launch_int8_pair<256>(a.x, a.w, a.K, a.K, p, stream) : launch_int8_pair<128>(a.x, a.w, a.K, a.K, p, stream);
}

// y of x [M, K] in bf16 (pitch ldx), whose rows are quantised first.  The product of few rows is put on the GPU behind that at once:
// its stages fill with the weight, which was there before the rows' kernel started, while that still runs (16 x 14336 x 4096:
// 15.0 us where it was 17.6, and 18 as a call, of 31 as two).
extern "C" int axb_int8_dense(const axb::Int8DenseCall* call, cudaStream_t stream) {
  using namespace axb;
  const Int8DenseCall& a = *call;
  if (a.M <= 0 || a.N <= 0) return 0;
  if (a.K < 16 || a.K % 16 || a.K > (1 << 17)) return -10;
  int8_t* codes = static_cast<int8_t*>(a.held);
  float* scales = reinterpret_cast<float*>(codes + a.M * a.K);
  const Int8RowsCall rows{a.x, codes, scales, a.M, a.K, a.ldx, 0};
  const int rc = axb_int8_rows(&rows, stream);
  if (rc != 0) return rc;
  const Int8LinearCall product{codes, scales, a.w, a.w_scales, a.y, a.M, a.N, a.K, a.accumulate, a.features, 1, a.status};
  if (a.features != 0) return axb_int8_gemm(&product, stream);
  if (chain_launches && !a.resident) {
    Int8LinearCall plain = product;
    plain.resident = 0;
    return axb_gemm_skinny_int8(&plain, stream);
  }
  ChainedBehind chained;
  return axb_gemm_skinny_int8(&product, stream);
}
