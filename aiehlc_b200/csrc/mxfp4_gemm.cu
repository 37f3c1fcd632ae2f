// Products of microscaled 4-bit matrices (format: mxfp4.cuh) on the tcgen05 tensor cores, kind::mxf4:
//     C[m][n] = sum_k A[m][k] * B[n][k],  each factor an e2m1 number times its block's power of two.
// The products are exact, the sums are held in 32 bits (TMEM).  C leaves as f32 (optionally added to what is there),
// bf16, f16, or quantised again along its rows.
#include <algorithm>
#include <type_traits>

#include "context.h"
#include "mxfp4.cuh"
#include "sm100_ptx.cuh"

namespace aiehlc {

namespace {

enum : int { MX_F32 = 0, MX_F32_ADD = 1, MX_BF16 = 2, MX_F16 = 3, MX_MX = 4 };

constexpr int kStepK = 256;                    // elements of K per step: one 128-byte swizzle span of codes
constexpr int kStepScales = 2 * kMxScaleTile;  // two scale tiles of 4 blocks each
constexpr int kMmaK = 64;                      // elements of K per tcgen05.mma
constexpr int kKPer = 2;                       // steps per pipeline stage
constexpr int kMaxSplit = 8;                   // CTAs that share the K of a narrow product

struct MxGemmParams {
  int M, N, K;
  int k_steps;              // steps of 256 elements
  int words;                // scale tiles along K (of 128 elements)
  const uint8_t* a_scales;
  const uint8_t* b_scales;
  void* C;                  // f32 / bf16 / f16, leading dimension ldc; MX_MX: codes
  uint8_t* c_scales;        // MX_MX
  long long ldc;
  int vec_ok;               // rows of C start on 16 bytes: vector stores
  int m_tiles, n_tiles;
  int tail_first;           // CTA pairs: tiles from this one on run as two column halves each (the number of tiles: none do)
  int tile_store;           // CTA pairs: results leave as TMA tile stores
  int stages;               // narrow form: stages in flight
  int group_m;              // CTA pairs: row blocks walked before the next column block
  int wide_boxes;           // one box brings all steps of a stage (K a multiple of 256)
  int* status;
  int debug;                // 3: the producer withholds its loads, so every wait runs out
};

// ---------------------------------------------------------------------------------------- few rows of A
// The rows of B are the 128 rows of the MMA and the rows of A its kTN columns, so that a product with few rows of A
// streams B through as many SMs as there are: each output tile (128 columns of C x kTN rows) is one cluster of
// `split` CTAs, each of which takes an equal range of K.  The partial sums meet in distributed shared memory, added in the order
// of the CTAs' ranks (the result does not depend on timing), and every CTA writes its share of the tile's rows.
// A stage holds 512 elements of K: the issuing warp's wait and commit take about 400 cycles a stage, whatever it holds (a
// product with 16 columns takes 32), and with 256 elements they set the pace.
template <int kTN>
struct NarrowShape {
  static constexpr int kBBlock = 128 * 128;                   // 256 elements of K of the tile's rows of B
  static constexpr int kABlock = kTN * 128;
  static constexpr int kBBytes = kBBlock * kKPer;
  static constexpr int kABytes = kABlock * kKPer;
  static constexpr int kScaleBytes = kStepScales * kKPer;     // of each operand
  static constexpr int kStageBytes = kBBytes + kABytes + 2 * kScaleBytes;
  static constexpr int kPartialBytes = kTN * 128 * 4;         // over the stages, once they are done
  static constexpr int kLimit = 227 * 1024 - 1024 - 256;
  static constexpr int kMaxStages = kLimit / kStageBytes;     // 5, 5, 4, 3
  static constexpr int pool(int stages) { return stages * kStageBytes > kPartialBytes ? stages * kStageBytes : kPartialBytes; }
  static constexpr int total(int stages) { return 1024 + pool(stages) + 256; }
  static constexpr int kSetCols = 8 * kKPer;                  // columns of each operand's scales per stage
  static constexpr int kScaleCols = 2 * kSetCols * kMaxStages;
  static constexpr int kTmemCols = 256;                       // two CTAs per SM at most
  static_assert(kTN + kScaleCols <= kTmemCols, "TMEM");
};

// Stores four consecutive results of a row; `n` is the first one's column.  Adding is a reduction, as in the other form: nothing
// is waited for, and each element is added to once.
template <int kOut>
__device__ __forceinline__ void store4(const MxGemmParams& p, int m, int n, const float4& v) {
  const long long at = static_cast<long long>(m) * p.ldc + n;
  const float f[4] = {v.x, v.y, v.z, v.w};
  if constexpr (kOut == MX_F32 || kOut == MX_F32_ADD) {
    float* c = static_cast<float*>(p.C) + at;
    if (p.vec_ok && n + 4 <= p.N) {
      if constexpr (kOut == MX_F32_ADD) red_add_f32x4(c, v);
      else *reinterpret_cast<float4*>(c) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) {
          if constexpr (kOut == MX_F32_ADD) red_add_f32(c + i, f[i]);
          else c[i] = f[i];
        }
    }
  } else {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kOut == MX_BF16) h[i] = __bfloat16_as_ushort(__float2bfloat16_rn(f[i]));
      else h[i] = __half_as_ushort(__float2half_rn(f[i]));
    }
    uint16_t* c = static_cast<uint16_t*>(p.C) + at;
    if (p.vec_ok && n + 4 <= p.N) {
      *reinterpret_cast<uint2*>(c) = make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) c[i] = h[i];
    }
  }
}

// The whole warp holds 128 consecutive results of row m, four per lane, first column n0 (a multiple of 128): four blocks
// of eight lanes.  Writes their codes and the row's scale word.
__device__ __forceinline__ void store_blocks(const MxGemmParams& p, int m, int n0, int lane, float4 v) {
  const int n = n0 + 4 * lane;
  float f[8] = {v.x, v.y, v.z, v.w, 0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= p.N) f[i] = 0.0f;
    most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  const int s = mx_scale_of(most);
  const float inv = mx_inverse(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= inv;
  const uint16_t codes = s == kMxNan ? 0 : static_cast<uint16_t>(mx_codes8(f));
  const int blocks = static_cast<int>(mx_blocks(p.N));
  const bool there = n / kMxBlock < blocks;
  if (there) *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(p.C) + static_cast<long long>(m) * blocks * 16 + n / 2) = codes;
  uint32_t word = static_cast<uint32_t>(there ? s : 0) << (8 * (lane >> 3));
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 16);
  if (lane == 0)
    *reinterpret_cast<uint32_t*>(p.c_scales + (static_cast<long long>(m / 128) * mx_words(p.N) + n0 / 128) * kMxScaleTile +
                                 mx_scale_word(m & 127)) = word;
}

// Adds the cluster's partial sums of rows first .. last - 1 of the tile (those of one row by one warp, four columns a lane, in
// the order of the ranks) and sends them through the output stage.  A read of another CTA's shared memory takes most of a
// microsecond, so kRows rows of up to kSplit shares are on their way together: 16 reads a thread.
template <int kRows, int kSplit, int kOut>
__device__ __forceinline__ void sum_rows(const MxGemmParams& p, const float* partial, int split, int first, int last, int m0, int n0) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t mine = smem_u32(partial) + lane * 16;
  for (int j0 = first + warp; j0 < last; j0 += 4 * kRows) {
    float4 o[kRows][kSplit];
#pragma unroll
    for (int c = 0; c < kSplit; ++c) {
      if (c < split) {
        const uint32_t at = mapa_u32(mine, c);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (j0 + 4 * i < last) o[i][c] = ld_cluster_f4(at + (j0 + 4 * i) * 512);
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = j0 + 4 * i;
      if (j < last) {
        float4 v = o[i][0];
#pragma unroll
        for (int c = 1; c < kSplit; ++c)
          if (c < split) { v.x += o[i][c].x; v.y += o[i][c].y; v.z += o[i][c].z; v.w += o[i][c].w; }
        if constexpr (kOut == MX_MX) store_blocks(p, m0 + j, n0, lane, v);
        else if (n0 + 4 * lane < p.N) store4<kOut>(p, m0 + j, n0 + 4 * lane, v);
      }
    }
  }
}

template <int kTN, int kOut>
__global__ void __launch_bounds__(128)
mx_gemm_narrow_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const MxGemmParams p) {
  using S = NarrowShape<kTN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::pool(p.stages));
  uint64_t* empty_bar = full_bar + S::kMaxStages;
  uint64_t* done_bar = empty_bar + S::kMaxStages;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int split = gridDim.x / (p.m_tiles * p.n_tiles);
  const int tile = blockIdx.x / split;
  const int m0 = tile % p.m_tiles * kTN;
  const int n0 = tile / p.m_tiles * 128;
  const int k_stages = (p.k_steps + kKPer - 1) / kKPer;
  const int k_first = static_cast<int>(static_cast<long long>(k_stages) * rank / split) * kKPer;
  const int k_last = static_cast<int>(static_cast<long long>(k_stages) * (rank + 1) / split) * kKPer;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    mbar_init(smem_u32(done_bar), 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_base_slot), S::kTmemCols);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint8_t* sa = p.a_scales + static_cast<long long>(m0 / 128) * p.words * kMxScaleTile;
    const uint8_t* sb = p.b_scales + static_cast<long long>(n0 / 128) * p.words * kMxScaleTile;
    for (int k = k_first; k < k_last; k += kKPer) {
      ok = mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.status, ST_TIMEOUT_EMPTY);
      if (!ok) break;
      if (p.debug != 3) {
        const uint32_t bar = smem_u32(&full_bar[stage]);
        const uint32_t at = smem_u32(smem + stage * S::kStageBytes);
        const uint32_t scales = at + S::kBBytes + S::kABytes;
        const uint32_t scale_bytes = min(2 * kKPer, p.words - 2 * k) * kMxScaleTile;  // K may end inside the stage
        mbar_expect_tx(bar, S::kBBytes + S::kABytes + 2 * scale_bytes);
        if (p.wide_boxes) {                                    // steps past the end of K read as zero
          tma_load_3d(at, &tmap_b, bar, 0, n0, k);
          tma_load_3d(at + S::kBBytes, &tmap_a, bar, 0, m0, k);
        } else {
#pragma unroll
          for (int kk = 0; kk < kKPer; ++kk) {
            tma_load_2d(at + kk * S::kBBlock, &tmap_b, bar, (k + kk) * 128, n0);
            tma_load_2d(at + S::kBBytes + kk * S::kABlock, &tmap_a, bar, (k + kk) * 128, m0);
          }
        }
        bulk_load_g2s(scales, sb + static_cast<long long>(k) * kStepScales, scale_bytes, bar);
        bulk_load_g2s(scales + S::kScaleBytes, sa + static_cast<long long>(k) * kStepScales, scale_bytes, bar);
      }
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (!ok)
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land before the CTA retires
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int k = k_first; k < k_last; k += kKPer) {
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&full_bar[stage]), phase, abort_flag, p.status, ST_TIMEOUT_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = smem_u32(smem + stage * S::kStageBytes);
      const uint32_t t_scales = tmem_base + kTN + stage * 2 * S::kSetCols;  // B's scales, then A's; free like the stage
      const int mmas = min(kKPer * kStepK, p.K - k * kStepK + kMmaK - 1) / kMmaK;
      const uint64_t sdesc = make_scale_desc(at + S::kBBytes + S::kABytes);
      const uint64_t bdesc = make_kmajor_desc(at, 1024, 2);
      const uint64_t adesc = make_kmajor_desc(at + S::kBBytes, 1024, 2);
      if (elect_one()) {
        constexpr int kPerStep = kStepK / kMmaK;
        const auto copy = [&](int w) {
          tmem_copy_scales<1>(t_scales + 4 * w, sdesc + w * (kMxScaleTile >> 4));
          tmem_copy_scales<1>(t_scales + S::kSetCols + 4 * w, sdesc + ((S::kScaleBytes + w * kMxScaleTile) >> 4));
        };
        const auto product = [&](int i, bool accumulate) {
          umma_mxf4<1>(tmem_base, bdesc + ((i / kPerStep) * (S::kBBlock >> 4) + 2 * (i % kPerStep)),
                       adesc + ((i / kPerStep) * (S::kABlock >> 4) + 2 * (i % kPerStep)), make_idesc_mxf4(128, kTN, 2 * (i & 1)),
                       t_scales + 4 * (i >> 1), t_scales + S::kSetCols + 4 * (i >> 1), accumulate);
        };
        if (mmas == kKPer * kPerStep) {
#pragma unroll
          for (int w = 0; w < 2 * kKPer; ++w) copy(w);
          product(0, k > k_first);
#pragma unroll
          for (int i = 1; i < kKPer * kPerStep; ++i) product(i, true);
        } else {
#pragma unroll
          for (int w = 0; w < 2 * kKPer; ++w)
            if (2 * w < mmas) copy(w);
          product(0, k > k_first);
#pragma unroll
          for (int i = 1; i < kKPer * kPerStep; ++i)
            if (i < mmas) product(i, true);
        }
        umma_commit(smem_u32(&empty_bar[stage]));
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (ok && elect_one()) umma_commit(smem_u32(done_bar));
  }
  __syncwarp();

  // Every warp turns its 32 rows of the accumulator (columns of C) into rows of 128 floats [row of C][column of C].
  bool ok = mbar_wait(smem_u32(done_bar), 0, abort_flag, p.status, ST_TIMEOUT_TMEM_FULL);
  ok = __all_sync(0xFFFFFFFFu, ok);
  const int valid = min(kTN, p.M - m0);
  float* partial = reinterpret_cast<float*>(smem);
  if (ok) {
    tc_fence_after();
#pragma unroll
    for (int c = 0; c < kTN; c += 16) {
      if (c < valid) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) partial[(c + j) * 128 + warp * 32 + lane] = __uint_as_float(r[j]);
      }
    }
  }
  tc_fence_before();
  if (split > 1) cluster_sync_all();  // every CTA's partial sums are in place
  else __syncthreads();

  if (ok) {
    const int first = valid * rank / split, last = valid * (rank + 1) / split;
    if (split <= 2) sum_rows<8, 2, kOut>(p, partial, split, first, last, m0, n0);
    else if (split <= 4) sum_rows<4, 4, kOut>(p, partial, split, first, last, m0, n0);
    else sum_rows<2, kMaxSplit, kOut>(p, partial, split, first, last, m0, n0);
    if constexpr (kOut == MX_MX) {
      // rows of the last scale tile that do not exist
      if (rank == 0 && m0 + kTN >= p.M)
        for (int m = p.M + threadIdx.x; m < (p.M + 127) / 128 * 128; m += 128)
          *reinterpret_cast<uint32_t*>(p.c_scales + (static_cast<long long>(m / 128) * mx_words(p.N) + n0 / 128) * kMxScaleTile +
                                       mx_scale_word(m & 127)) = 0;
    }
  }
  if (split > 1) cluster_sync_all();  // the others may still read this CTA's partial sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, S::kTmemCols);
  }
}

}  // namespace
}  // namespace aiehlc

#include "mxfp4_gemm_pair.cuh"

namespace aiehlc {
namespace {

int encode_codes_map(aiehlc_ctx* ctx, CUtensorMap* map, const uint8_t* codes, long long rows, long long cols, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(mx_pitch(cols)), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(mx_pitch(cols))};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = ctx->encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIEHLC_ERR_CUDA, "cuTensorMapEncodeTiled failed for the codes of a 4-bit operand");
  return AIEHLC_OK;
}

// Codes as a 3-D tensor {128 bytes, rows, K / 256}: one box brings `steps` steps of K.  K a multiple of 256.
int encode_codes_map_3d(aiehlc_ctx* ctx, CUtensorMap* map, const uint8_t* codes, long long rows, long long cols, int box_rows, int steps) {
  const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(cols / kStepK)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(mx_pitch(cols)), 128};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(steps)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = ctx->encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(codes), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIEHLC_ERR_CUDA, "cuTensorMapEncodeTiled (3-D) failed for the codes of a 4-bit operand");
  return AIEHLC_OK;
}

// How many CTAs share the K of a tile of the narrow form: as many as there are SMs for with one CTA on each, all clusters
// resident at once (clusters do not straddle GPCs, so fewer large ones fit than the SM count says: 128 CTAs ran in 5.2 us as
// clusters of four and in 11.8 us, two waves, as clusters of eight), and each CTA with two stages to do (with 128 columns, where a
// stage takes longer, one).
template <int kTN, int kOut>
int narrow_split(aiehlc_ctx* ctx, long long tiles, int k_stages) {
  using S = NarrowShape<kTN>;
  const int sms = ctx->usable_sms();
  if (tiles > sms) return 1;
  auto kern = mx_gemm_narrow_kernel<kTN, kOut>;
  KernelSetup& ks = ctx->kernel_setup[reinterpret_cast<const void*>(kern)];
  int split = std::min(static_cast<int>(sms / tiles), kTN == 128 ? k_stages : k_stages / 2);
  for (split = std::min(split, kMaxSplit); split > 1; --split) {
    int& fit = ks.clusters_of[split];
    if (fit == 0) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = split;
      attr.val.clusterDim.y = 1;
      attr.val.clusterDim.z = 1;
      cfg.gridDim = dim3(split);
      cfg.blockDim = dim3(128);
      cfg.dynamicSmemBytes = S::total(S::kMaxStages);
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (ensure_dynamic_smem(ctx->device, reinterpret_cast<const void*>(kern), S::total(S::kMaxStages), &ks.smem_attr)) return 1;
      if (cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) != cudaSuccess || fit <= 0) {
        cudaGetLastError();
        fit = -1;
      }
    }
    if (tiles <= fit) return split;
  }
  return 1;
}

template <int kTN, int kOut>
int launch_narrow(aiehlc_ctx* ctx, const MxGemmCall& c, MxGemmParams& p, cudaStream_t st) {
  using S = NarrowShape<kTN>;
  CUtensorMap ma, mb;
  if (p.wide_boxes) {
    if (int rc = encode_codes_map_3d(ctx, &ma, c.A, c.M, c.K, kTN, kKPer)) return rc;
    if (int rc = encode_codes_map_3d(ctx, &mb, c.B, c.N, c.K, 128, kKPer)) return rc;
  } else {
    if (int rc = encode_codes_map(ctx, &ma, c.A, c.M, c.K, kTN)) return rc;
    if (int rc = encode_codes_map(ctx, &mb, c.B, c.N, c.K, 128)) return rc;
  }
  p.m_tiles = (c.M + kTN - 1) / kTN;
  p.n_tiles = (c.N + 127) / 128;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  auto kern = mx_gemm_narrow_kernel<kTN, kOut>;
  KernelSetup& ks = ctx->kernel_setup[reinterpret_cast<const void*>(kern)];
  // One CTA per SM has a ring as deep as shared memory allows; with more tiles than SMs two share one, with two stages each.
  const int split = narrow_split<kTN, kOut>(ctx, tiles, (p.k_steps + kKPer - 1) / kKPer);
  p.stages = tiles > ctx->usable_sms() && 2 * S::total(2) <= 226 * 1024 ? 2 : S::kMaxStages;
  const int smem_bytes = S::total(p.stages);
  if (int rc = ensure_dynamic_smem(ctx->device, reinterpret_cast<const void*>(kern), S::total(S::kMaxStages), &ks.smem_attr)) return rc;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * split));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->pdl ? 2 : 1;
  AIEHLC_CUDA(cudaLaunchKernelEx(&cfg, kern, ma, mb, p));
  ctx->launches++;
  return AIEHLC_OK;
}

// Scales as a matrix with one row per 128 rows of the operand, in 8-byte elements; a box brings `steps` steps of K of
// `box_rows` such rows.  What lies outside reads as zero.
int encode_scales_map(aiehlc_ctx* ctx, CUtensorMap* map, const uint8_t* scales, long long rows, long long cols, int box_rows, int steps) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(mx_words(cols) * (kMxScaleTile / 8)), static_cast<cuuint64_t>((rows + 127) / 128)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(mx_words(cols) * kMxScaleTile)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(steps * kStepScales / 8), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = ctx->encode(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<uint8_t*>(scales), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIEHLC_ERR_CUDA, "cuTensorMapEncodeTiled failed for the scales of a 4-bit operand");
  return AIEHLC_OK;
}

// C as the output warps of a CTA pair store it: 32 rows x 64 bytes (codes: all kBN / 2 bytes of the tile's rows).
template <int kBN, int kOut>
int encode_result_map(aiehlc_ctx* ctx, CUtensorMap* map, const MxGemmCall& c) {
  constexpr int esize = kOut == MX_MX ? 1 : kOut == MX_F32 || kOut == MX_F32_ADD ? 4 : 2;
  constexpr int row_bytes = kOut == MX_MX ? kBN / 2 : 64;
  const long long cols = kOut == MX_MX ? mx_pitch(c.N) : c.N;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(c.M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(kOut == MX_MX ? cols : c.ldc * esize)};
  const cuuint32_t box[2] = {row_bytes / esize, 32};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = kOut == MX_MX ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : kOut == MX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : kOut == MX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const CUresult r = ctx->encode(map, type, 2, c.C, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIEHLC_ERR_CUDA, "cuTensorMapEncodeTiled failed for the result of a 4-bit product");
  return AIEHLC_OK;
}

template <int kBN, int kOut>
int launch_pair(aiehlc_ctx* ctx, const MxGemmCall& c, MxGemmParams& p, cudaStream_t st) {
  using S = MxPairShape<kBN>;
  CUtensorMap ma, mb, mbh, mas, mbs, mc;
  if (p.wide_boxes) {
    if (int rc = encode_codes_map_3d(ctx, &ma, c.A, c.M, c.K, 128, kKPer)) return rc;
    if (int rc = encode_codes_map_3d(ctx, &mb, c.B, c.N, c.K, kBN / 2, kKPer)) return rc;
  } else {
    if (int rc = encode_codes_map(ctx, &ma, c.A, c.M, c.K, 128)) return rc;
    if (int rc = encode_codes_map(ctx, &mb, c.B, c.N, c.K, kBN / 2)) return rc;
  }
  if (int rc = encode_scales_map(ctx, &mas, c.As, c.M, c.K, 1, kKPer)) return rc;
  if (int rc = encode_scales_map(ctx, &mbs, c.Bs, c.N, c.K, S::kBTiles, kKPer)) return rc;
  constexpr int esize = kOut == MX_F32 || kOut == MX_F32_ADD ? 4 : 2;
  // a tile store is clipped at the tensor's edge in pieces of 16 bytes: a row that ends inside one would be written past its end
  p.tile_store = kOut == MX_MX || (reinterpret_cast<uintptr_t>(c.C) % 16 == 0 && c.ldc * esize % 16 == 0 && static_cast<long long>(c.N) * esize % 16 == 0);
  mc = ma;  // unused without tile stores
  if (p.tile_store)
    if (int rc = encode_result_map<kBN, kOut>(ctx, &mc, c)) return rc;
  p.m_tiles = (c.M + 255) / 256;
  p.n_tiles = (c.N + kBN - 1) / kBN;
  p.group_m = ctx->group_m > 0 ? ctx->group_m : 8;
  const int tiles = p.m_tiles * p.n_tiles;
  const int limit = ctx->usable_sms() / 2 > 0 ? ctx->usable_sms() / 2 : 1;
  // A last wave that keeps at most half of the pairs busy: its tiles are cut into two column halves that run side by side
  int parts = 1;
  narrow_tail(tiles, limit, kBN, tiles > limit ? ctx->split_tail : 0, &p.tail_first, &parts);
  mbh = mb;
  if (parts == 2) {
    if (p.wide_boxes) {
      if (int rc = encode_codes_map_3d(ctx, &mbh, c.B, c.N, c.K, kBN / 4, kKPer)) return rc;
    } else if (int rc = encode_codes_map(ctx, &mbh, c.B, c.N, c.K, kBN / 4)) return rc;
  }
  const int units = 2 * tiles - p.tail_first;
  auto kern = mx_gemm_pair_kernel<kBN, kOut>;
  KernelSetup& ks = ctx->kernel_setup[reinterpret_cast<const void*>(kern)];
  if (int rc = ensure_dynamic_smem(ctx->device, reinterpret_cast<const void*>(kern), S::kTotal, &ks.smem_attr)) return rc;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min(units, limit)));
  cfg.blockDim = dim3(kMxPairThreads);
  cfg.dynamicSmemBytes = S::kTotal;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->pdl ? 2 : 1;
  AIEHLC_CUDA(cudaLaunchKernelEx(&cfg, kern, ma, mb, mbh, mas, mbs, mc, p));
  ctx->launches++;
  return AIEHLC_OK;
}

template <int kOut>
int launch_out(aiehlc_ctx* ctx, const MxGemmCall& c, cudaStream_t st) {
  MxGemmParams p{};
  p.M = c.M; p.N = c.N; p.K = c.K;
  p.k_steps = (c.K + kStepK - 1) / kStepK;
  p.words = static_cast<int>(mx_words(c.K));
  p.wide_boxes = c.K % kStepK == 0 && ctx->k_per_load != 1;
  p.a_scales = c.As; p.b_scales = c.Bs;
  p.C = c.C; p.c_scales = c.Cs; p.ldc = c.ldc;
  const int esize = kOut == MX_F32 || kOut == MX_F32_ADD ? 4 : 2;
  p.vec_ok = reinterpret_cast<uintptr_t>(c.C) % 16 == 0 && c.ldc * esize % 16 == 0;
  p.status = ctx->d_status;
  p.debug = ctx->debug_mode;
  // Up to 64 rows of A: the narrow form.  More: CTA pairs, unless there are so few tiles that most SMs would be idle and K is
  // long enough for splitting it to pay (narrow form, 128 columns).  Measured, us, narrow / pairs: 128 x 4096 x 1024 7.1 / 5.0,
  // 128 x 4096 x 4096 8.4 / 7.5, 128 x 8192 x 8192 11.5 / 11.7, 128 x 512 x 16384 8.4 / 16.4, 67 x 1001 x 4103 6.9 / 7.9:
  // about 0.41 us per stage for a wave of pairs, 0.5 for a narrow CTA, and 2.7 us for joining the partial sums.
  const int sms = ctx->usable_sms(), k_stages = (p.k_steps + kKPer - 1) / kKPer;
  bool pairs = ctx->pair_mode == 1 || (ctx->pair_mode != 0 && c.M > 64 && sms >= 2);
  if (pairs && ctx->pair_mode != 1) {
    const long long tiles = ((c.M + 127LL) / 128) * ((c.N + 127LL) / 128);
    const int split = narrow_split<128, kOut>(ctx, tiles, k_stages);
    if (split > 1 && 0.41 * k_stages > 0.5 * k_stages / split + 2.7) pairs = false;
  }
  if (pairs) {
    // half as wide tiles where that at least doubles the SMs at work
    const long long tiles = ((c.M + 255LL) / 256) * ((c.N + 255LL) / 256);
    if (ctx->force_tile_n == 128 || (ctx->force_tile_n == 0 && tiles * 2 <= sms / 2)) return launch_pair<128, kOut>(ctx, c, p, st);
    return launch_pair<256, kOut>(ctx, c, p, st);
  }
  if (c.M <= 16) return launch_narrow<16, kOut>(ctx, c, p, st);
  if (c.M <= 32) return launch_narrow<32, kOut>(ctx, c, p, st);
  if (c.M <= 64) return launch_narrow<64, kOut>(ctx, c, p, st);
  return launch_narrow<128, kOut>(ctx, c, p, st);
}

}  // namespace

int launch_mx_gemm(aiehlc_ctx* ctx, const MxGemmCall& c, cudaStream_t st) {
  if (c.Cs) return launch_out<MX_MX>(ctx, c, st);
  switch (c.type) {
    case AIEHLC_TYPE_F32: return c.accumulate ? launch_out<MX_F32_ADD>(ctx, c, st) : launch_out<MX_F32>(ctx, c, st);
    case AIEHLC_TYPE_BF16: return launch_out<MX_BF16>(ctx, c, st);
    default: return launch_out<MX_F16>(ctx, c, st);
  }
}

}  // namespace aiehlc
