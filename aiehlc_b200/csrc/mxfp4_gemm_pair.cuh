// Products of microscaled 4-bit matrices by CTA pairs (tcgen05 cta_group::2): two CTAs on neighbouring SMs share one
// 256 x kBN tile of C, persistent over the tiles.  Included by mxfp4_gemm.cu.
//
//   warp 0 (both CTAs)  fetches this CTA's 128 rows of A, its half of B's rows, the scales of its A rows and the scales of all
//                       of the tile's B rows (each CTA multiplies with all of B); everything is credited to the
//                       leader's "full" barrier
//   warp 1 (leader)     copies the scales to both CTAs' TMEM and issues the products, M = 256, K = 64 each
//   warps 2-5           drain this CTA's 128 accumulator rows through the output stage
//
// What the products take is set by the issuing warp as much as by the tensor cores (256 x 256 x 64: 128 cycles).  Under
// `if (lane == 0)` a product took 155 cycles and the scale copies 75 more; with the whole warp walking the loop and one elected
// lane issuing, 129 and nothing (512 x 9472 x 65536, operands not loaded; 160 with them).  Four warps that wrote
// the scales with tcgen05.st instead of the copies: 199 against 193 us on 8192^3, 13.5 against 12.8 on 4096 x 4096 x 1024.
//
// TMEM (512 columns per CTA): two accumulators of kBN columns and two sets of scales, one per stage in flight: for each
// 128 elements of K, 4 columns of A's scales and kBN / 32 of B's.  With kBN = 256 the accumulators share 96 columns, which
// makes the room: accumulator 0 takes columns 0-255, accumulator 1 columns 160-415.  The output stage reads the
// half of a tile that holds the shared columns first and hands them back at once, so that the next tile's products
// wait for one read of TMEM, not for the whole output stage.
#pragma once

namespace aiehlc {

namespace {

constexpr int kMxPairThreads = 192;
// A stage holds kKPer steps of K: a commit costs the tensor cores' queue about 50 cycles (measured: 166 cycles per product
// with one commit per eight products, 179 with one more per four), so a stage is as long as shared memory allows.
template <int kBN>
struct MxPairShape {
  static constexpr int kABlock = 128 * 128;                    // 256 elements of K of this CTA's rows of A
  static constexpr int kBBlock = kBN / 2 * 128;
  static constexpr int kBTiles = kBN / 128;                    // scale tiles (of 128 rows) across the tile's columns
  static constexpr int kABytes = kABlock * kKPer;
  static constexpr int kBBytes = kBBlock * kKPer;
  static constexpr int kAScales = kStepScales * kKPer;
  static constexpr int kBScales = kStepScales * kKPer * kBTiles;
  static constexpr int kStageBytes = kABytes + kBBytes + kAScales + kBScales;
  static constexpr int kStagingBytes = 4 * 4096;               // one buffer of 32 rows x 128 bytes per output warp
  static constexpr int kBarBytes = 1024;
  static constexpr int kLimit = 227 * 1024;
  static constexpr int kStages = (kLimit - kStagingBytes - kBarBytes) / kStageBytes > 8 ? 8 : (kLimit - kStagingBytes - kBarBytes) / kStageBytes;
  static constexpr int kTotal = kStages * kStageBytes + kStagingBytes + kBarBytes;
  static constexpr bool kShared = kBN == 256;
  static constexpr int kAcc1 = kBN == 256 ? 160 : kBN;         // first column of accumulator 1
  static constexpr int kWordCols = 4 + 4 * kBTiles;            // columns of scales per 128 elements of K
  static constexpr int kSetCols = 2 * kKPer * kWordCols;
  static constexpr int kSets = 2;
  static constexpr int kScaleCol = kAcc1 + kBN;
  static constexpr int kTmemCols = 512;
  static_assert(kStageBytes % 1024 == 0 && kScaleCol + kSets * kSetCols <= kTmemCols && kSets <= kStages, "layout");
};

// Unit `u` of the launch: a tile, or (thin last wave: p.tail_first) one of the two column halves of a tail tile.  Tiles walk
// group_m row blocks before the next column block.
__device__ __forceinline__ void mx_unit(const MxGemmParams& p, int u, int& mb, int& nb, int& part) {
  int t = u;
  part = -1;
  if (u >= p.tail_first) {
    t = p.tail_first + ((u - p.tail_first) >> 1);
    part = (u - p.tail_first) & 1;
  }
  const int per_group = p.group_m * p.n_tiles;
  const int g = t / per_group;
  const int first = g * p.group_m;
  const int rows = min(p.group_m, p.m_tiles - first);
  const int r = t - g * per_group;
  mb = first + r % rows;
  nb = r / rows;
}

// 32 rows x 32 columns of C, one row per lane, through this warp's staging buffer and out one row at a time, neighbouring lanes
// on neighbouring columns: for a C that allows no tile stores.  One warp per scheduler does this, so what counts is
// the number of instructions a row takes: 26 with tests and addresses worked out per row made a 4793 x 4299 result take 62 us,
// where tile stores take 15.  Adding is one reduction per element: nothing is waited for, and as an element is added to once, the
// result does not depend on timing.
template <int kOut>
__device__ __forceinline__ void store_rows(const MxGemmParams& p, uint8_t* buf, const uint32_t (&r)[32], int row0, int col0, int lane) {
  using T = std::conditional_t<kOut == MX_BF16, __nv_bfloat16, std::conditional_t<kOut == MX_F16, __half, float>>;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
  __syncwarp();
  const int n = col0 + lane;
  const int rows = n < p.N ? min(32, p.M - row0) : 0;
  T* c = static_cast<T*>(p.C) + (static_cast<long long>(row0) * p.ldc + n);
  const uint8_t* src = buf + ((lane & 3) << 2);
#pragma unroll 1
  for (int i0 = 0; i0 < rows; i0 += 8, src += 8 * 128) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float*>(src + i * 128 + (((lane >> 2) ^ i) << 4));
    if (i0 + 8 <= rows) {
#pragma unroll
      for (int i = 0; i < 8; ++i, c += p.ldc) {
        if constexpr (kOut == MX_F32_ADD) red_add_f32(c, v[i]);
        else *c = mx_from_float<T>(v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i, c += p.ldc)
        if (i0 + i < rows) {
          if constexpr (kOut == MX_F32_ADD) red_add_f32(c, v[i]);
          else *c = mx_from_float<T>(v[i]);
        }
    }
  }
  __syncwarp();
}

template <int kBN, int kOut>
__global__ void __launch_bounds__(kMxPairThreads, 1)
mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_b_half, const __grid_constant__ CUtensorMap tmap_as, const __grid_constant__ CUtensorMap tmap_bs,
                    const __grid_constant__ CUtensorMap tmap_c, const MxGemmParams p) {
  using S = MxPairShape<kBN>;
  constexpr int kStages = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];   // nothing static: the dynamic part starts on its 1024-byte boundary
  uint8_t* staging = smem + kStages * S::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + S::kStagingBytes);  // used in the leader
  uint64_t* empty_bar = full_bar + kStages;           // one set per CTA
  uint64_t* tmem_full_bar = empty_bar + kStages;      // one set per CTA
  uint64_t* tmem_free_bar = tmem_full_bar + 2;        // used in the leader: one per accumulator, or one for what they share
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_free_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int pair_id = static_cast<int>(cluster_id_x());
  const int num_pairs = static_cast<int>(cluster_count_x());

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&tmem_full_bar[a]), 1);
      mbar_init(smem_u32(&tmem_free_bar[a]), 8);      // every output warp of the two CTAs
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_as);
    tma_prefetch_desc(&tmap_bs);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(tmem_base_slot), S::kTmemCols);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  pdl_launch_dependents();
  pdl_wait();
  const int num_tiles = p.m_tiles * p.n_tiles;
  const int num_units = 2 * num_tiles - p.tail_first;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair_id; ok && t < num_units; t += num_pairs) {
        int mb, nb, part;
        mx_unit(p, t, mb, nb, part);
        const int b_rows = kBN / (part < 0 ? 2 : 4);
        const int row_b = nb * kBN + (part > 0 ? kBN / 2 : 0) + rank * b_rows;
        const int scales_b = nb * S::kBTiles + (part > 0 ? S::kBTiles / 2 : 0);
        const CUtensorMap* map_b = part < 0 ? &tmap_b : &tmap_b_half;
        for (int k = 0; k < p.k_steps; k += kKPer) {
          ok = mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.status, ST_TIMEOUT_EMPTY);
          if (!ok) break;
          if (p.debug != 3) {
            if (leader) mbar_expect_tx(smem_u32(&full_bar[stage]), 2 * (S::kABytes + kKPer * 128 * b_rows + S::kAScales + S::kBScales));
            const uint32_t bar = mapa_u32(smem_u32(&full_bar[stage]), 0);
            const uint32_t sa = smem_u32(smem + stage * S::kStageBytes);
            const uint32_t sb = sa + S::kABytes;
            const uint32_t ss = sb + S::kBBytes;
            const int row_a = mb * 256 + rank * 128;
            // steps past the end of K read as zero
            if (p.wide_boxes) {
              tma_load_3d_pair(sa, &tmap_a, bar, 0, row_a, k);
              tma_load_3d_pair(sb, map_b, bar, 0, row_b, k);
            } else {
#pragma unroll
              for (int kk = 0; kk < kKPer; ++kk) {
                tma_load_2d_pair(sa + kk * S::kABlock, &tmap_a, bar, (k + kk) * 128, row_a);
                tma_load_2d_pair(sb + kk * 128 * b_rows, map_b, bar, (k + kk) * 128, row_b);
              }
            }
            tma_load_2d_pair(ss, &tmap_as, bar, k * (kStepScales / 8), mb * 2 + rank);
            tma_load_2d_pair(ss + S::kAScales, &tmap_bs, bar, k * (kStepScales / 8), scales_b);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok)
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land before the CTA retires
    }
  } else if (warp == 1) {
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      int set = 0;
      int old_stage = 0;                              // whose products have read the set before it is written again
      uint32_t old_phase = 0;
      bool reuse = false;
      int it = 0;
      bool ok = true;
      for (int t = pair_id; ok && t < num_units; t += num_pairs, ++it) {
        // The output stage has drained the accumulator's tile before this one.  Where the accumulators share columns, what
        // it signals is that it has read the shared ones of the last tile, for which it was through with the tile before.
        if constexpr (S::kShared) ok = it == 0 || mbar_wait(smem_u32(tmem_free_bar), (it - 1) & 1, abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY);
        else ok = it < 2 || mbar_wait(smem_u32(&tmem_free_bar[it & 1]), ((it >> 1) - 1) & 1, abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (it & 1) * S::kAcc1;
        const bool halved = t >= p.tail_first;
        const uint32_t idesc = halved ? make_idesc_mxf4(256, kBN / 2, 0) : make_idesc_mxf4(256, kBN, 0);
        const uint32_t b_block = S::kBBlock >> (halved ? 5 : 4);   // descriptor units from one step of K to the next
        for (int k = 0; k < p.k_steps; k += kKPer) {
          ok = mbar_wait(smem_u32(&full_bar[stage]), phase, abort_flag, p.status, ST_TIMEOUT_FULL);
          if (reuse) {
            // the stage before keeps the tensor cores busy meanwhile
            ok = ok && mbar_wait(smem_u32(&empty_bar[old_stage]), old_phase, abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY);
            if (++old_stage == kStages) { old_stage = 0; old_phase ^= 1; }
          }
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * S::kStageBytes);
          const uint64_t adesc = make_kmajor_desc(sa, 1024, 2);
          const uint64_t bdesc = make_kmajor_desc(sa + S::kABytes, 1024, 2);
          const uint32_t t_scales = tmem_base + S::kScaleCol + set * S::kSetCols;
          const int mmas = min(kKPer * kStepK, p.K - k * kStepK + kMmaK - 1) / kMmaK;
          if (elect_one()) {
            constexpr int kPerStep = kStepK / kMmaK;
            const auto product = [&](int i, bool accumulate) {
              umma_mxf4<2>(d_tmem, adesc + ((i / kPerStep) * (S::kABlock >> 4) + 2 * (i % kPerStep)),
                           bdesc + ((i / kPerStep) * b_block + 2 * (i % kPerStep)), idesc | make_idesc_mxf4_scale(2 * (i & 1)),
                           t_scales + (i >> 1) * S::kWordCols, t_scales + (i >> 1) * S::kWordCols + 4, accumulate);
            };
            const uint64_t sdesc = make_scale_desc(sa + S::kABytes + S::kBBytes);
#pragma unroll
            for (int w = 0; w < 2 * kKPer; ++w) {
              tmem_copy_scales<2>(t_scales + w * S::kWordCols, sdesc + ((w * kMxScaleTile) >> 4));
#pragma unroll
              for (int b = 0; b < S::kBTiles; ++b)
                tmem_copy_scales<2>(t_scales + w * S::kWordCols + 4 + 4 * b, sdesc + ((S::kAScales + (b * 2 * kKPer + w) * kMxScaleTile) >> 4));
            }
            product(0, k > 0);
            if (mmas == kKPer * kPerStep) {   // straight through: a test per product costs the issuing thread 20 to 40 cycles
#pragma unroll
              for (int i = 1; i < kKPer * kPerStep; ++i) product(i, true);
            } else {
#pragma unroll
              for (int i = 1; i < kKPer * kPerStep; ++i)
                if (i < mmas) product(i, true);
            }
            umma_commit_pair_mask(smem_u32(&empty_bar[stage]), 3);
          }
          __syncwarp();
          if (++set == S::kSets) { set = 0; reuse = true; }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (ok && elect_one()) umma_commit_pair_mask(smem_u32(&tmem_full_bar[it & 1]), 3);
        __syncwarp();
      }
    }
  } else {
    const int quad = warp & 3;
    uint8_t* buf = staging + quad * 4096;
    const int swz = lane & 7;
    int it = 0;
    for (int t = pair_id; t < num_units; t += num_pairs, ++it) {
      int mb, nb, part;
      mx_unit(p, t, mb, nb, part);
      const int acc = it & 1;
      bool ok = mbar_wait(smem_u32(&tmem_full_bar[acc]), (it >> 1) & 1, abort_flag, p.status, ST_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      tc_fence_after();
      const int row0 = mb * 256 + rank * 128 + quad * 32;
      const int n0 = nb * kBN + (part > 0 ? kBN / 2 : 0);
      const int halves = part < 0 ? kBN / 128 : 1;   // a column half of a 256-column tile is 128 columns
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * S::kAcc1;
      uint32_t words[kBN / 128] = {};                  // MX_MX: this row's scales
#pragma unroll 1
      for (int half = 0; half < halves; ++half) {
        // accumulator 0 of 256 columns shares its last ones, accumulator 1 its first
        const int c_half = S::kShared && acc == 0 && part < 0 ? 128 - 128 * half : 128 * half;
        uint32_t all[4][32];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(taddr + c_half + 32 * i, all[i]);
        tmem_ld_wait();
        if (half == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(smem_u32(&tmem_free_bar[S::kShared ? 0 : acc]), 0);
        }
#pragma unroll
        for (int step = 0; step < 2; ++step) {
        const int c = c_half + 64 * step;
        uint32_t (&r)[2][32] = *reinterpret_cast<uint32_t (*)[2][32]>(&all[2 * step]);
        if constexpr (kOut == MX_MX) {
          if (half == 0 && step == 0) {
            if (lane == 0) tma_store_wait_read<0>();   // the tile before has left the buffer
            __syncwarp();
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = n0 + c + 32 * h;
            if (n + 32 > p.N) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (n + j >= p.N) r[h][j] = 0;
            }
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) most = max(most, r[h][j] & 0x7FFFFFFFu);
            const int s = mx_scale_of(most);
            const float inv = mx_inverse(s);
            uint32_t w[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(r[h][8 * g + j]) * inv;
              w[g] = s == kMxNan ? 0 : mx_codes8(f);
            }
            const int piece = c / 32 + h;              // 16 bytes of codes per block
            if (part >= 0) {                           // a column half is not the tile store's box
              if (row0 + lane < p.M && n < p.N)
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.C) + (static_cast<long long>(row0 + lane) * mx_pitch(p.N) + n / 2)) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            } else
              *reinterpret_cast<uint4*>(buf + lane * (kBN / 2) + ((piece ^ (kBN == 256 ? swz : (lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            const uint32_t byte = row0 + lane < p.M && n < p.N ? static_cast<uint32_t>(s) << (8 * (piece & 3)) : 0u;
            if (kBN == 256 && piece >= 4) words[kBN / 128 - 1] |= byte;
            else words[0] |= byte;
          }
        } else if (p.tile_store) {
          // 64-byte pieces of 32 rows, through the two halves of this warp's buffer in turn
          constexpr int kCols = kOut == MX_F32 || kOut == MX_F32_ADD ? 16 : 32;
#pragma unroll
          for (int h = 0; h < 64 / kCols; ++h) {
            uint8_t* piece = buf + (h & 1) * 2048;
            if (lane == 0) tma_store_wait_read<1>();   // the store before the last has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (kOut == MX_F32 || kOut == MX_F32_ADD) {
                  w[i] = r[h >> 1][16 * (h & 1) + 4 * j + i];
                } else {
                  const float lo = __uint_as_float(r[h][8 * j + 2 * i]), hi = __uint_as_float(r[h][8 * j + 2 * i + 1]);
                  if constexpr (kOut == MX_BF16) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&v);
                  } else {
                    const __half2 v = __floats2half2_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&v);
                  }
                }
              }
              *reinterpret_cast<uint4*>(piece + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if constexpr (kOut == MX_F32_ADD) tma_reduce_add_2d(&tmap_c, smem_u32(piece), n0 + c + kCols * h, row0);
              else tma_store_2d(&tmap_c, smem_u32(piece), n0 + c + kCols * h, row0);
              tma_store_commit();
            }
          }
        } else {
          store_rows<kOut>(p, buf, r[0], row0, n0 + c, lane);
          store_rows<kOut>(p, buf, r[1], row0, n0 + c + 32, lane);
        }
        }
      }
      if constexpr (kOut == MX_MX) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && part < 0) {
          tma_store_2d(&tmap_c, smem_u32(buf), n0 / 2, row0);
          tma_store_commit();
        }
        // scale words of this row; rows past M are zeros up to the end of their scale tile
        const long long c_words = mx_words(p.N);
        if (row0 / 128 < (p.M + 127) / 128) {
#pragma unroll
          for (int w = 0; w < kBN / 128; ++w)
            if (w < halves && n0 / 128 + w < c_words)
              *reinterpret_cast<uint32_t*>(p.c_scales + (static_cast<long long>(row0 / 128) * c_words + n0 / 128 + w) * kMxScaleTile +
                                           mx_scale_word((row0 + lane) & 127)) = words[w];
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }

  // Neither CTA retires or frees TMEM while its partner can still read its shared memory or signal its barriers.
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, S::kTmemCols);
  }
}

}  // namespace

}  // namespace aiehlc
