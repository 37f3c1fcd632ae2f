// Quantisation to microscaled 4-bit blocks and back (format: mxfp4.cuh).
#include "context.h"
#include "mxfp4.cuh"
#include "sm100_ptx.cuh"

namespace aiehlc {

namespace {

constexpr int kTile = 128;          // a CTA takes 128 x 128 elements: one scale tile along the rows and one along the columns
constexpr int kQuantThreads = 256;
constexpr int kLanesPerRow = kTile / 8;                      // a thread holds 8 consecutive elements of a row
constexpr int kRowsPerPass = kQuantThreads / kLanesPerRow;   // 16
constexpr int kPasses = kTile / kRowsPerPass;                // 8

// Eight consecutive elements of a row; elements at or past `cols` are zero.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* row, long long col, long long cols, T (&v)[8]) {
  if (kVec && col + 8 <= cols) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(&v[0]) = *reinterpret_cast<const uint4*>(row + col);
      *reinterpret_cast<uint4*>(&v[4]) = *reinterpret_cast<const uint4*>(row + col + 4);
    } else {
      *reinterpret_cast<uint4*>(&v[0]) = *reinterpret_cast<const uint4*>(row + col);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? row[col + i] : mx_from_float<T>(0.0f);
  }
}

// One pass over the matrix.  Bound by memory: sizeof(T) bytes read and 17/32 written per element and direction.
//   rows   : the four lanes that hold a block agree on its maximum with two shuffles; each writes four bytes of codes
//   columns: the tile turns through shared memory; a thread takes 32 rows of two neighbouring columns, and the codes
//            of a column's four blocks leave as 64 contiguous bytes
// A 128 x 128 tile makes exactly one 512-byte scale tile each way, which leaves as one contiguous store.
template <typename T, bool kVec, bool kRows, bool kCols>
__global__ void __launch_bounds__(kQuantThreads)
mx_quantize_kernel(const T* __restrict__ x, long long rows, long long cols, long long ld, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ qs, uint8_t* __restrict__ t, uint8_t* __restrict__ ts, int col_tiles) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* row_scales = smem;                        // 512 bytes
  uint8_t* col_scales = smem + kMxScaleTile;         // 512 bytes
  uint8_t* turned = smem + 2 * kMxScaleTile;         // codes along the columns, [128][64 + 16]: the pad spreads the banks
  constexpr int kTurnedPitch = 80;
  T* tile = reinterpret_cast<T*>(smem + 2 * kMxScaleTile + kTile * kTurnedPitch);  // [128][128]

  pdl_launch_dependents();
  pdl_wait();
  const long long row_tile = blockIdx.x / col_tiles;
  const int col_tile = static_cast<int>(blockIdx.x - row_tile * col_tiles);
  const long long r0 = row_tile * kTile;
  const long long c0 = static_cast<long long>(col_tile) * kTile;
  const int tid = threadIdx.x;
  const int sub = tid & (kLanesPerRow - 1);          // which eight columns of the tile
  const int line = tid / kLanesPerRow;
  const long long col = c0 + sub * 8;
  const long long blocks = mx_blocks(cols);

  alignas(16) T v[kPasses][8];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const long long r = r0 + p * kRowsPerPass + line;
    if (r < rows) load8<T, kVec>(x + r * ld, col, cols, v[p]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[p][i] = mx_from_float<T>(0.0f);
    }
  }
  if constexpr (kCols) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      T* dst = tile + (p * kRowsPerPass + line) * kTile + sub * 8;
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(&v[p][0]);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst + 4) = *reinterpret_cast<const uint4*>(&v[p][4]);
    }
  }
  if constexpr (kRows) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int in_tile = p * kRowsPerPass + line;
      float f[8];
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = mx_to_float(v[p][i]);
        most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
      }
      most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
      most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
      const int s = mx_scale_of(most);
      const float inv = mx_inverse(s);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = mx_scaled(f[i], inv);
      const uint32_t codes = mx_codes8(f);
      const long long r = r0 + in_tile;
      const long long block = c0 / kMxBlock + sub / 4;
      const bool there = r < rows && block < blocks;
      if (there) *reinterpret_cast<uint32_t*>(q + r * blocks * 16 + col / 2) = codes;
      if ((sub & 3) == 0) row_scales[mx_scale_word(in_tile) + sub / 4] = there ? static_cast<uint8_t>(s) : 0;
    }
  }
  __syncthreads();
  if constexpr (kRows) {
    if (tid < kMxScaleTile / 16)
      reinterpret_cast<uint4*>(qs + (row_tile * mx_words(cols) + col_tile) * kMxScaleTile)[tid] =
          reinterpret_cast<const uint4*>(row_scales)[tid];
  }
  if constexpr (kCols) {
    const long long row_blocks = mx_blocks(rows);
    const int pair = tid & 63, rb = tid >> 6;        // columns 2 pair, 2 pair + 1; rows 32 rb ...
    const T* src = tile + rb * kMxBlock * kTile + 2 * pair;
    float f0[kMxBlock], f1[kMxBlock];
    uint32_t m0 = 0, m1 = 0;
#pragma unroll
    for (int i = 0; i < kMxBlock; ++i) {
      f0[i] = mx_to_float(src[i * kTile]);
      f1[i] = mx_to_float(src[i * kTile + 1]);
      m0 = max(m0, __float_as_uint(f0[i]) & 0x7FFFFFFFu);
      m1 = max(m1, __float_as_uint(f1[i]) & 0x7FFFFFFFu);
    }
    const bool block_there = r0 / kMxBlock + rb < row_blocks;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 2 * pair + h;
      const int s = mx_scale_of(h ? m1 : m0);
      const float inv = mx_inverse(s);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = mx_scaled(h ? f1[8 * j + i] : f0[8 * j + i], inv);
        w[j] = mx_codes8(g);
      }
      *reinterpret_cast<uint4*>(turned + c * kTurnedPitch + rb * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      col_scales[mx_scale_word(c) + rb] = block_there && c0 + c < cols ? static_cast<uint8_t>(s) : 0;
    }
    __syncthreads();
    // four threads per column: its four blocks' codes are 64 contiguous bytes
#pragma unroll
    for (int i = tid; i < kTile * 4; i += kQuantThreads) {
      const int c = i >> 2, b = i & 3;
      const long long block = r0 / kMxBlock + b;
      if (c0 + c < cols && block < row_blocks)
        *reinterpret_cast<uint4*>(t + ((c0 + c) * row_blocks + block) * 16) =
            *reinterpret_cast<const uint4*>(turned + c * kTurnedPitch + b * 16);
    }
    if (tid < kMxScaleTile / 16)
      reinterpret_cast<uint4*>(ts + (static_cast<long long>(col_tile) * mx_words(rows) + row_tile) * kMxScaleTile)[tid] =
          reinterpret_cast<const uint4*>(col_scales)[tid];
  }
}

// Values of a quantised matrix.  Bound by memory: 17/32 byte read, sizeof(T) written per element.  A CTA takes the
// 128 x 128 elements of one scale tile; a thread turns four bytes of codes into eight values.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ qs, long long rows, long long cols,
                     T* __restrict__ y, long long ld, int col_tiles) {
  pdl_launch_dependents();
  pdl_wait();
  const long long row_tile = blockIdx.x / col_tiles;
  const int col_tile = static_cast<int>(blockIdx.x - row_tile * col_tiles);
  const long long r0 = row_tile * kTile;
  const int sub = threadIdx.x & (kLanesPerRow - 1);
  const int line = threadIdx.x / kLanesPerRow;
  const long long col = static_cast<long long>(col_tile) * kTile + sub * 8;
  if (col >= cols) return;
  const long long pitch = mx_pitch(cols);
  const uint8_t* scales = qs + (row_tile * mx_words(cols) + col_tile) * kMxScaleTile + sub / 4;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int in_tile = p * kRowsPerPass + line;
    const long long r = r0 + in_tile;
    if (r >= rows) break;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(q + r * pitch + col / 2);
    const float scale = mx_scale_value(scales[mx_scale_word(in_tile)]);
    __half2 h[4];
    mx_decode8(codes, h);
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = mx_from_float<T>(f.x * scale);
      v[2 * i + 1] = mx_from_float<T>(f.y * scale);
    }
    T* dst = y + r * ld + col;
    if (kVec && col + 8 <= cols) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(&v[0]);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst + 4) = *reinterpret_cast<const uint4*>(&v[4]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < cols) dst[i] = v[i];
    }
  }
}

cudaLaunchConfig_t tile_grid(const aiehlc_ctx* ctx, unsigned tiles, int smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles);
  cfg.blockDim = dim3(kQuantThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->pdl ? 1 : 0;
  return cfg;
}

template <typename T, bool kVec, bool kRows, bool kCols>
int quantize_as(aiehlc_ctx* ctx, const MxQuantizeCall& c, cudaStream_t st) {
  auto kern = mx_quantize_kernel<T, kVec, kRows, kCols>;
  const int smem = 2 * kMxScaleTile + (kCols ? kTile * 80 + kTile * kTile * static_cast<int>(sizeof(T)) : 0);
  KernelSetup& ks = ctx->kernel_setup[reinterpret_cast<const void*>(kern)];
  if (int rc = ensure_dynamic_smem(ctx->device, reinterpret_cast<const void*>(kern), smem, &ks.smem_attr)) return rc;
  const int col_tiles = static_cast<int>((c.cols + kTile - 1) / kTile);
  const long long tiles = (c.rows + kTile - 1) / kTile * col_tiles;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = tile_grid(ctx, static_cast<unsigned>(tiles), smem, st, &attr);
  AIEHLC_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(c.x), c.rows, c.cols, c.ld, c.q, c.qs, c.t, c.ts, col_tiles));
  ctx->launches++;
  return AIEHLC_OK;
}

template <typename T>
int quantize_typed(aiehlc_ctx* ctx, const MxQuantizeCall& c, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(c.x) % 16 == 0 && c.ld * sizeof(T) % 16 == 0;
  if (c.q && c.t) return vec ? quantize_as<T, true, true, true>(ctx, c, st) : quantize_as<T, false, true, true>(ctx, c, st);
  if (c.q) return vec ? quantize_as<T, true, true, false>(ctx, c, st) : quantize_as<T, false, true, false>(ctx, c, st);
  return vec ? quantize_as<T, true, false, true>(ctx, c, st) : quantize_as<T, false, false, true>(ctx, c, st);
}

template <typename T>
int dequantize_typed(aiehlc_ctx* ctx, const uint8_t* q, const uint8_t* qs, long long rows, long long cols, void* y,
                     long long ld, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(y) % 16 == 0 && ld * sizeof(T) % 16 == 0;
  const int col_tiles = static_cast<int>((cols + kTile - 1) / kTile);
  const long long tiles = (rows + kTile - 1) / kTile * col_tiles;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = tile_grid(ctx, static_cast<unsigned>(tiles), 0, st, &attr);
  if (vec) AIEHLC_CUDA(cudaLaunchKernelEx(&cfg, mx_dequantize_kernel<T, true>, q, qs, rows, cols, static_cast<T*>(y), ld, col_tiles));
  else AIEHLC_CUDA(cudaLaunchKernelEx(&cfg, mx_dequantize_kernel<T, false>, q, qs, rows, cols, static_cast<T*>(y), ld, col_tiles));
  ctx->launches++;
  return AIEHLC_OK;
}

}  // namespace

int launch_mx_quantize(aiehlc_ctx* ctx, const MxQuantizeCall& c, cudaStream_t st) {
  switch (c.type) {
    case AIEHLC_TYPE_F32: return quantize_typed<float>(ctx, c, st);
    case AIEHLC_TYPE_BF16: return quantize_typed<__nv_bfloat16>(ctx, c, st);
    default: return quantize_typed<__half>(ctx, c, st);
  }
}

int launch_mx_dequantize(aiehlc_ctx* ctx, const uint8_t* q, const uint8_t* qs, long long rows, long long cols, void* y,
                         int type, long long ld, cudaStream_t st) {
  switch (type) {
    case AIEHLC_TYPE_F32: return dequantize_typed<float>(ctx, q, qs, rows, cols, y, ld, st);
    case AIEHLC_TYPE_BF16: return dequantize_typed<__nv_bfloat16>(ctx, q, qs, rows, cols, y, ld, st);
    default: return dequantize_typed<__half>(ctx, q, qs, rows, cols, y, ld, st);
  }
}

}  // namespace aiehlc
