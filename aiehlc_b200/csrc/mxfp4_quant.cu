// Quantisation to microscaled 4-bit blocks and back (format: mxfp4.cuh).
#include "context.h"
#include "mxfp4.cuh"
#include "sm100_ptx.cuh"

namespace aiehlc {

namespace {

constexpr int kTile = 128;          // a CTA takes 128 x 128 elements: one scale tile along the rows and one along the columns
constexpr int kQuantThreads = 256;

// Consecutive elements of a row as they come from memory, two to a register for the 16-bit types.
template <typename T, int kCount>
struct alignas(16) Run {
  static constexpr int kWords = kCount * static_cast<int>(sizeof(T)) / 4;
  static constexpr int kPieces = kWords / 4;   // of 16 bytes
  uint32_t w[kWords];
};
// The larger magnitudes of two pairs; NaN stays NaN.
template <typename T> __device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max_abs2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(__habs2(*reinterpret_cast<__nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<__nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <> __device__ __forceinline__ uint32_t max_abs2<__half>(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2_nan(__habs2(*reinterpret_cast<__half2*>(&a)), __habs2(*reinterpret_cast<__half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T> __device__ __forceinline__ float2 split2(uint32_t w);
template <> __device__ __forceinline__ float2 split2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 split2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Two results to a pair, each rounded to nearest even, in one conversion.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Largest magnitude as float bits; a NaN or infinity keeps the exponent 255.
template <typename T, int kCount>
__device__ __forceinline__ uint32_t max_bits(const Run<T, kCount>& v) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kCount; ++i) m = max(m, v.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kCount / 2; ++i) m = max_abs2<T>(m, v.w[i]);
    const float2 f = split2<T>(m);
    return max(__float_as_uint(f.x), __float_as_uint(f.y)) & 0x7FFFFFFFu;
  }
}
template <typename T, int kCount>
__device__ __forceinline__ void codes_of(const Run<T, kCount>& v, int s, uint32_t (&codes)[kCount / 8]) {
  const float inv = mx_inverse(s);
#pragma unroll
  for (int g = 0; g < kCount / 8; ++g) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(v.w[8 * g + i]) * inv;
        f[i + 1] = __uint_as_float(v.w[8 * g + i + 1]) * inv;
      } else {
        const float2 p = split2<T>(v.w[4 * g + (i >> 1)]);
        f[i] = p.x * inv;
        f[i + 1] = p.y * inv;
      }
    }
    codes[g] = s == kMxNan ? 0u : mx_codes8(f);
  }
}

// One pass over the matrix: sizeof(T) bytes read and 17/32 written per element and direction.  What bounds it next to memory is
// the ALU pipe (maxima, splitting pairs, conversions; 70 % of its rate at 13 instructions an element, before a block's own
// work was shared by two threads instead of four).
//   rows   : the lanes that hold a block agree on its maximum with shuffles; each writes the codes of its elements
//   columns: the tile turns through shared memory; a thread takes 32 rows of two neighbouring columns, and the codes
//            of a column's four blocks leave as 64 contiguous bytes
// Four CTAs on an SM keep the loads of one under the arithmetic of others (16384 x 16384 bf16, rows: 96 us and 7.1 TB/s, of which
// part comes from L2, against 105 us with three; both ways 148 against 160 us).
// A 128 x 128 tile makes exactly one 512-byte scale tile each way, which leaves as one contiguous store.
// Where rows do not start on 16 bytes (kVec false) the tile comes in by four-byte asynchronous copies and the rows are read back
// from shared memory.
// Elements from one staged row of the tile to the next: unaligned rows of a 16-bit type take one more word.
template <typename T, bool kVec>
__host__ __device__ constexpr int tile_pitch() { return sizeof(T) == 2 && !kVec ? kTile + 2 : kTile; }

template <typename T, bool kVec, bool kRows, bool kCols>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : 4)
mx_quantize_kernel(const T* __restrict__ x, long long rows, long long cols, long long ld, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ qs, uint8_t* __restrict__ t, uint8_t* __restrict__ ts, int col_tiles) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* row_scales = smem;                        // 512 bytes
  uint8_t* col_scales = smem + kMxScaleTile;         // 512 bytes
  T* tile = reinterpret_cast<T*>(smem + 2 * kMxScaleTile);                          // [128][128]
  uint8_t* turned = smem + 2 * kMxScaleTile + kTile * tile_pitch<T, kVec>() * sizeof(T);   // codes along the columns
  // Elements of a row a thread takes.  Half a block where rows are quantised (4096 x 4096 bf16, rows: 6.2 us against 8.9 us with
  // a quarter); a quarter of f32 tiles that pass through shared memory, where 64-byte strides cost bank conflicts
  // (both ways, 8192 x 8192: 79 against 89 us), and of tiles that only pass through.
  constexpr int kRun = kCols && (!kRows || sizeof(T) == 4) ? 8 : 16;
  // Two 16-byte pieces a thread: in the second half of a row neighbouring pieces change places, so that eight threads that
  // store their first (or second) pieces together meet all banks once.
  constexpr bool kSwap = kVec && kCols && kRun == 16 && sizeof(T) == 2;
  constexpr int kLanesPerRow = kTile / kRun;
  constexpr int kRowsPerPass = kQuantThreads / kLanesPerRow;
  constexpr int kPasses = kTile / kRowsPerPass;
  using R = Run<T, kRun>;
  constexpr int kPitch = tile_pitch<T, kVec>();

  pdl_launch_dependents();
  pdl_wait();
  const long long row_tile = blockIdx.x / col_tiles;
  const int col_tile = static_cast<int>(blockIdx.x - row_tile * col_tiles);
  const long long r0 = row_tile * kTile;
  const long long c0 = static_cast<long long>(col_tile) * kTile;
  const int tid = threadIdx.x;
  const int sub = tid & (kLanesPerRow - 1);
  const int line = tid / kLanesPerRow;
  const long long col = c0 + sub * kRun;
  const long long blocks = mx_blocks(cols);
  const int rows_here = static_cast<int>(min(static_cast<long long>(kTile), rows - r0));

  R v[kPasses];
  if constexpr (kVec) {
    const bool whole = col + kRun <= cols;
    const T* src = x + (r0 + line) * ld + col;
#pragma unroll
    for (int p = 0; p < kPasses; ++p, src += kRowsPerPass * ld) {
      const bool row_there = p * kRowsPerPass + line < rows_here;
#pragma unroll
      for (int i = 0; i < R::kWords; ++i) v[p].w[i] = 0;
      if (row_there && whole) {
#pragma unroll
        for (int i = 0; i < R::kPieces; ++i)
          *reinterpret_cast<uint4*>(&v[p].w[4 * i]) = __ldg(reinterpret_cast<const uint4*>(src) + i);
      } else if (row_there) {
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          if (col + i < cols) {
            if constexpr (sizeof(T) == 4) v[p].w[i] = reinterpret_cast<const uint32_t*>(src)[i];
            else v[p].w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(src)[i]) << (16 * (i & 1));
          }
      }
    }
    if constexpr (kCols) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int i = 0; i < R::kPieces; ++i)
          reinterpret_cast<uint4*>(tile + (p * kRowsPerPass + line) * kTile + sub * kRun)[kSwap ? i ^ (sub >> 2) : i] =
              *reinterpret_cast<const uint4*>(&v[p].w[4 * i]);
    }
  } else {
    // Four bytes at a time, all of them on their way at once.  A row of a 16-bit type may start in the middle of four: its
    // elements then start in the middle of the staged row's first word (`odd`).
    const int cols_here = static_cast<int>(min(static_cast<long long>(kTile), cols - c0));
    const int warp = tid >> 5, lane = tid & 31;
    constexpr int kWords = kPitch * static_cast<int>(sizeof(T)) / 4;
    constexpr int kWarps = kQuantThreads / 32;
    if (rows_here == kTile && cols_here == kTile && blockIdx.x != 0) {
      // a whole tile, and not the first (whose first word may start before the matrix): nothing to test per word
      uintptr_t row = reinterpret_cast<uintptr_t>(x + ((r0 + warp) * ld + c0));
      uint32_t dst = smem_u32(tile + warp * kPitch) + 4 * lane;
#pragma unroll 4
      for (int i = 0; i < kTile / kWarps; ++i) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(row & ~static_cast<uintptr_t>(3)) + 4 * lane;
#pragma unroll
        for (int w = 0; w < kTile * static_cast<int>(sizeof(T)) / 128; ++w) cp_async_4(dst + 128 * w, src + 128 * w, 4);
        // the last element, where the row starts in the middle of a word
        if (sizeof(T) == 2 && (row & 2) && lane == 0) cp_async_4(dst + 2 * kTile, src + 2 * kTile, 2);
        row += kWarps * ld * sizeof(T);
        dst += kWarps * kPitch * sizeof(T);
      }
    } else
#pragma unroll 1
    for (int r = warp; r < kTile; r += kWarps) {
      const uintptr_t row = reinterpret_cast<uintptr_t>(x + ((r0 + r) * ld + c0));
      const int odd = static_cast<int>(row & 2) >> 1;
      const int bytes = r < rows_here ? cols_here * static_cast<int>(sizeof(T)) + 2 * odd : 0;
      T* dst = tile + r * kPitch;
#pragma unroll
      for (int w = lane; w < kWords; w += 32) {
        if (4 * w >= bytes) reinterpret_cast<uint32_t*>(dst)[w] = 0;
        else if (odd && w == 0 && r0 + r == 0 && c0 == 0) dst[1] = x[0];   // nothing before the matrix is read
        else cp_async_4(smem_u32(dst) + 4 * w, reinterpret_cast<const uint8_t*>(row - 2 * odd) + 4 * w, min(4, bytes - 4 * w));
      }
    }
    cp_async_wait_all();
    __syncthreads();
    if constexpr (kRows) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const T* src = tile + (p * kRowsPerPass + line) * kPitch + sub * kRun;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < R::kPieces; ++i) *reinterpret_cast<uint4*>(&v[p].w[4 * i]) = reinterpret_cast<const uint4*>(src)[i];
        } else {
          const bool odd = reinterpret_cast<uintptr_t>(x + ((r0 + p * kRowsPerPass + line) * ld + c0)) & 2;
          uint32_t w[R::kWords + 1];
#pragma unroll
          for (int i = 0; i <= R::kWords; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
#pragma unroll
          for (int i = 0; i < R::kWords; ++i) v[p].w[i] = odd ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
        }
      }
    }
  }
  if constexpr (kRows) {
    constexpr int kSharers = kMxBlock / kRun;        // lanes that hold a block
    const bool block_there = c0 / kMxBlock + sub / kSharers < blocks;
    uint8_t* dst = q + (r0 + line) * blocks * 16 + col / 2;
#pragma unroll
    for (int p = 0; p < kPasses; ++p, dst += kRowsPerPass * blocks * 16) {
      const int r = p * kRowsPerPass + line;
      uint32_t most = max_bits(v[p]);
#pragma unroll
      for (int o = 1; o < kSharers; o <<= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
      const int s = mx_scale_of(most);
      uint32_t codes[kRun / 8];
      codes_of(v[p], s, codes);
      const bool there = r < rows_here && block_there;
      if (there) {
        if constexpr (kRun == 16) *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
        else *reinterpret_cast<uint32_t*>(dst) = codes[0];
      }
      if (sub % kSharers == 0) row_scales[mx_scale_word(r) + sub / kSharers] = there ? static_cast<uint8_t>(s) : 0;
    }
  }
  __syncthreads();
  if constexpr (kRows) {
    if (tid < kMxScaleTile / 16)
      reinterpret_cast<uint4*>(qs + (row_tile * mx_words(cols) + col_tile) * kMxScaleTile)[tid] =
          reinterpret_cast<const uint4*>(row_scales)[tid];
  }
  if constexpr (kCols) {
    constexpr int kTurnedPitch = 80;                 // 64 bytes of codes per column; the pad spreads the banks
    const long long row_blocks = mx_blocks(rows);
    const int pair = tid & 63, rb = tid >> 6;        // columns 2 pair, 2 pair + 1; rows 32 rb ...
    const T* src = tile + rb * kMxBlock * kPitch + (kSwap ? (pair * 2) ^ ((pair >> 5) << 3) : 2 * pair);
    const bool block_there = r0 / kMxBlock + rb < row_blocks;
    // codes and scale of column 2 pair + h
    const auto column = [&](int h, uint32_t most, const auto& value) {
      const int c = 2 * pair + h;
      const int s = mx_scale_of(most & 0x7FFFFFFFu);
      const float inv = mx_inverse(s);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = value(8 * j + i) * inv;
        w[j] = s == kMxNan ? 0u : mx_codes8(g);
      }
      *reinterpret_cast<uint4*>(turned + c * kTurnedPitch + (rb ^ ((c >> 3) & 1)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      col_scales[mx_scale_word(c) + rb] = block_there && c0 + c < cols ? static_cast<uint8_t>(s) : 0;
    };
    if constexpr (sizeof(T) == 4) {
      float2 f[kMxBlock];
      uint32_t m0 = 0, m1 = 0;
#pragma unroll
      for (int i = 0; i < kMxBlock; ++i) {
        f[i] = *reinterpret_cast<const float2*>(src + i * kPitch);
        m0 = max(m0, __float_as_uint(f[i].x) & 0x7FFFFFFFu);
        m1 = max(m1, __float_as_uint(f[i].y) & 0x7FFFFFFFu);
      }
      column(0, m0, [&](int i) { return f[i].x; });
      column(1, m1, [&](int i) { return f[i].y; });
    } else {
      uint32_t w[kMxBlock], m = 0;
#pragma unroll
      for (int i = 0; i < kMxBlock; ++i) {
        w[i] = *reinterpret_cast<const uint32_t*>(src + i * kPitch);
        if constexpr (!kVec) {
          const uint32_t next = *reinterpret_cast<const uint32_t*>(src + i * kPitch + 2);
          if (reinterpret_cast<uintptr_t>(x + ((r0 + rb * kMxBlock + i) * ld + c0)) & 2) w[i] = __funnelshift_r(w[i], next, 16);
        }
        m = max_abs2<T>(m, w[i]);
      }
      const float2 f = split2<T>(m);
      column(0, __float_as_uint(f.x), [&](int i) { return split2<T>(w[i]).x; });
      column(1, __float_as_uint(f.y), [&](int i) { return split2<T>(w[i]).y; });
    }
    __syncthreads();
    // four threads per column: its four blocks' codes are 64 contiguous bytes
#pragma unroll
    for (int i = tid; i < kTile * 4; i += kQuantThreads) {
      const int c = i >> 2, b = i & 3;
      const long long block = r0 / kMxBlock + b;
      if (c0 + c < cols && block < row_blocks)
        *reinterpret_cast<uint4*>(t + ((c0 + c) * row_blocks + block) * 16) =
            *reinterpret_cast<const uint4*>(turned + c * kTurnedPitch + (b ^ ((c >> 3) & 1)) * 16);
    }
    if (tid < kMxScaleTile / 16)
      reinterpret_cast<uint4*>(ts + (static_cast<long long>(col_tile) * mx_words(rows) + row_tile) * kMxScaleTile)[tid] =
          reinterpret_cast<const uint4*>(col_scales)[tid];
  }
}

// Values of a quantised matrix.  Bound by memory: 17/32 byte read, sizeof(T) written per element.  A CTA takes the
// 128 x 128 elements of one scale tile; a thread turns four bytes of codes into eight values.  f32 values, and those of a y whose
// rows do not start on 16 bytes (kVec false), turn through shared memory, two rows a warp, so that neighbouring lanes store
// neighbours (4793 x 4304 f32 with 32 bytes a lane: 24 us).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ qs, long long rows, long long cols,
                     T* __restrict__ y, long long ld, int col_tiles) {
  constexpr int kLanesPerRow = kTile / 8;
  constexpr int kRowsPerPass = kQuantThreads / kLanesPerRow;
  constexpr int kPasses = kTile / kRowsPerPass;
  constexpr bool kTurn = !kVec || sizeof(T) == 4;
  __shared__ __align__(16) T turned[kTurn ? kQuantThreads / 32 : 1][kTurn ? 2 : 1][kTurn ? kTile : 8];
  pdl_launch_dependents();
  pdl_wait();
  const long long row_tile = blockIdx.x / col_tiles;
  const int col_tile = static_cast<int>(blockIdx.x - row_tile * col_tiles);
  const long long r0 = row_tile * kTile;
  const long long c0 = static_cast<long long>(col_tile) * kTile;
  const int sub = threadIdx.x & (kLanesPerRow - 1);
  const int line = threadIdx.x / kLanesPerRow;
  const int rows_here = static_cast<int>(min(static_cast<long long>(kTile), rows - r0));
  const int cols_here = static_cast<int>(min(static_cast<long long>(kTile), cols - c0));
  const bool col_there = sub * 8 < cols_here;
  const long long pitch = mx_pitch(cols);
  const uint8_t* src = q + (r0 + line) * pitch + c0 / 2 + sub * 4;
  const uint8_t* scales = qs + (row_tile * mx_words(cols) + col_tile) * kMxScaleTile + sub / 4;
  uint32_t codes[kPasses];
  int s[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p, src += kRowsPerPass * pitch) {
    const int r = p * kRowsPerPass + line;
    const bool there = r < rows_here && col_there;
    codes[p] = there ? *reinterpret_cast<const uint32_t*>(src) : 0u;
    s[p] = there ? scales[mx_scale_word(r)] : 0;
  }
  T* row = y + (r0 + line) * ld + c0 + sub * 8;
#pragma unroll
  for (int p = 0; p < kPasses; ++p, row += kRowsPerPass * ld) {
    if (p * kRowsPerPass >= rows_here) break;
    const int r = p * kRowsPerPass + line;
    const float scale = mx_scale_value(s[p]);
    __half2 h[4];
    mx_decode8(codes[p], h);
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      if constexpr (sizeof(T) == 4) {
        v[2 * i] = f.x * scale;
        v[2 * i + 1] = f.y * scale;
      } else {
        reinterpret_cast<uint32_t*>(v)[i] = pack2<T>(f.x * scale, f.y * scale);
      }
    }
    if constexpr (!kTurn) {
      T* dst = row;
      if (r < rows_here && col_there) {
        if (sub * 8 + 8 <= cols_here) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (sub * 8 + i < cols_here) dst[i] = v[i];
        }
      }
    } else {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        reinterpret_cast<uint4*>(&turned[warp][lane >> 4][sub * 8])[i] = reinterpret_cast<const uint4*>(v)[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = p * kRowsPerPass + 2 * warp + i;
        T* dst = y + (r0 + row) * ld + c0;
        if (kVec && 4 * lane + 4 <= cols_here) {
          if (row < rows_here) reinterpret_cast<uint4*>(dst)[lane] = reinterpret_cast<const uint4*>(turned[warp][i])[lane];
        } else if (kVec) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (row < rows_here && 4 * lane + j < cols_here) dst[4 * lane + j] = turned[warp][i][4 * lane + j];
        } else {
#pragma unroll
          for (int j = 0; j < kTile / 32; ++j)
            if (row < rows_here && 32 * j + lane < cols_here) dst[32 * j + lane] = turned[warp][i][32 * j + lane];
        }
      }
      __syncwarp();
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
  const int smem = 2 * kMxScaleTile + (kCols || !kVec ? kTile * tile_pitch<T, kVec>() * static_cast<int>(sizeof(T)) : 0) + (kCols ? kTile * 80 : 0);
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
