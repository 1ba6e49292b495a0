// FP8 matrix products with one fp32 scale per 128 columns of K, dense and over row-concatenated groups:
//
//   y[t, n] = row_scale[t] * sum_c sa[c, t] sb[n / 128, c] * sum_{k in block c} a[t, k] w[n, k]
//
// a, w e4m3; sa one fp32 scale per token and 128 columns, sb one per 128 x 128 block of the weights.
// The hardware's own block scales are powers of two (ue8m0), so the outer sum cannot stay in the
// tensor core: each K block of 128 is a product of its own in tensor memory, and the consumer warps add it,
// times its two scales, to sums in their registers (fp32 throughout).
//
// A CTA pair takes 256 tokens (the MMA's M side, 128 per CTA, tensor-memory lane = token) by 256 weight rows
// (N, both CTAs supply half).  A consumer thread then has one token, so one scale per K block and 128
// columns: a K block costs it one multiplication and an addition per value, and no shared memory.  The two
// consumer groups take 128 columns, that is a weight block, each.  Two accumulators of 256 columns alternate.
//
// Tiles of up to 64 tokens (a decode step, what is left over of a group) exchange the roles: 256 weight rows
// are the M side and the tokens N, rounded up to 32, so that a tile costs little more than its weights'
// way into shared memory.  A lane then is a weight row and a register a token; the tokens' scales come by shuffle.
#include "gemm_common.cuh"

#include <cuda_fp16.h>

namespace msc {

struct Fp8Params {
  const float* sfa;          // (kblocks, pitch)
  const float* sfb;          // [l][nblocks][kblocks]
  const float* row_scale;    // [rows_total] or null
  const int* group_rows;     // [l], null: one group of all rows
  const int* group_offsets;  // [l]
  void* out;                 // [rows_total][n]
  int* status;
  int out_type;              // 0 bf16, 1 f32, 2 f16
  int l, n, rows_total, pitch;
  int kblocks, nblocks;
};

struct Fp8Smem {
  static constexpr int kW = 128 * 128;             // this CTA's 128 weight rows of a stage
  static constexpr int kTileTokens = 256;          // most tokens of a tile
  static constexpr int kFewTokens = 64;            // up to here the weights are the M side
  static constexpr int kParts = 2;                 // of a tile's columns, four consumer warps and a weight block each
  static constexpr int kPartCols = 128;
  static constexpr int kEpiWarps = 4 * kParts;
  static constexpr int kThreads = (kEpiWarps + 4) * 32;   // whole warpgroups: two of the last four idle
  // Registers a thread: the consumers need more than the block was launched with, the others less.
  static constexpr int kLaunchRegs = 168, kConsumerRegs = 208, kOtherRegs = 88;
  static_assert(kEpiWarps * kConsumerRegs + 4 * kOtherRegs <= (kEpiWarps + 4) * kLaunchRegs, "the block was launched with no more");
  static constexpr int kMaxStages = 10;
  static constexpr int kSlots = 2;                 // accumulators
  static constexpr int kBoxPitch = 80;             // a token's 32 16-bit columns, padded: no bank conflicts
  static constexpr int kBoxBytes = 32 * kBoxPitch;
  // barriers and flags | operand ring | epilogue boxes
  static constexpr int kOffRing = 1024;
  static constexpr int kRing = 5 * (kW + 128 * 128);
  static constexpr int kOffBox = kOffRing + kRing;
  static constexpr int kTotal = kOffBox + kEpiWarps * kBoxBytes;
  static constexpr int kAlloc = kTotal + 1024;
  static_assert(kAlloc <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
  // barrier offsets
  static constexpr int kBarFull = 0;
  static constexpr int kBarEmpty = kBarFull + 8 * kMaxStages;
  static constexpr int kBarAccFull = kBarEmpty + 8 * kMaxStages;
  static constexpr int kBarAccEmpty = kBarAccFull + 8 * kSlots;
  static_assert(kBarAccEmpty + 8 * kSlots <= 1000, "barriers and flags share the first 1024 bytes");
  static constexpr int kTmemSlot = 1000, kAbort = 1004;
};

// Rows of a group as the tiles see them: they start at a multiple of 4 (the scales arrive as 16-byte
// pieces), up to three rows before the group, which are computed and not stored.
__device__ __forceinline__ void fp8_group(const Fp8Params& p, int g, int& rows, int& off) {
  if (!p.group_rows) {
    rows = p.rows_total;
    off = 0;
    return;
  }
  load_group(p.group_rows, p.group_offsets, p.rows_total, g, rows, off);
  if (rows > 0) rows += off & 3;
}

__device__ __forceinline__ int fp8_token_tiles(int rows) { return (rows + 255) >> 8; }

struct Fp8Tile {
  int g, nt;        // group, weight tile of 256 rows
  int row0, lead;   // first token row (a multiple of 4); rows of it that belong to somebody else
  int tn;           // tokens
  bool few;         // the weights are the M side
  int width;        // the N side: weight rows, or tokens where they are few, rounded up to 32
};

struct Fp8Cursor {
  GroupWindow<true> win;
  __device__ __forceinline__ bool seek(const Fp8Params& p, int ntiles, int t, Fp8Tile& tile) {
    int rows, off, first;
    if (!win.find(p.l, t, [&](int gi, int& r, int& o) { fp8_group(p, gi, r, o); },
                  [=](int r) { return fp8_token_tiles(r) * ntiles; }, tile.g, rows, off, first))
      return false;
    const int u = t - first, tt = u / ntiles;
    tile.nt = u - tt * ntiles;
    tile.lead = tt == 0 ? (off & 3) : 0;
    tile.row0 = (off & ~3) + tt * 256;
    tile.tn = min(rows - tt * 256, 256);
    tile.few = tile.tn <= Fp8Smem::kFewTokens;
    tile.width = tile.few ? (tile.tn + 31) & ~31 : min((p.n - tile.nt * 256 + 31) & ~31, 256);
    return true;
  }
};

// D[tmem] (+)= A[smem] * B[smem]^T of e4m3 operands, K = 32.
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t pack_16bit(float lo, float hi, int out_type) {
  if (out_type == 0) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_value(const Fp8Params& p, size_t at, float v) {
  if (p.out_type == 0) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  else if (p.out_type == 1) static_cast<float*>(p.out)[at] = v;
  else static_cast<__half*>(p.out)[at] = __float2half_rn(v);
}
// Writes a box of 32 rows x 64 bytes out: rows [first, last) of the matrix, columns col .. of `bytes` each.
__device__ __forceinline__ void store_box(const Fp8Params& p, uint32_t box, int row0, int first, int last, int col, int bytes,
                                          int lane) {
  const int piece = lane & 3;
  const bool in = col + piece * (16 / bytes) < p.n;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = row0 + r * 8 + (lane >> 2);
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(box + (r * 8 + (lane >> 2)) * Fp8Smem::kBoxPitch + piece * 16) : "memory");
    if (in && row >= first && row < last)
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + ((size_t)row * p.n + col) * bytes + piece * 16) = v;
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Fp8Smem::kThreads, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w16,
                      const __grid_constant__ CUtensorMap tmap_t128, const __grid_constant__ CUtensorMap tmap_t32,
                      const __grid_constant__ CUtensorMap tmap_t16,
                      const Fp8Params p) {
  using L = Fp8Smem;
  constexpr int kMmaWarp = L::kEpiWarps, kProducerWarp = L::kEpiWarps + 1;
  constexpr uint32_t kIdescBase = (1u << 4) | (16u << 24);   // fp32 accumulators, e4m3 x e4m3, M = 256

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(sgen + L::kTmemSlot);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(sgen + L::kAbort);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = __shfl_sync(0xffffffffu, cluster_ctarank(), 0);
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int ntiles = (p.n + 255) >> 8;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kMaxStages; ++s) {
      mbar_init(sbase + L::kBarFull + 8 * s, 1);
      mbar_init(sbase + L::kBarEmpty + 8 * s, 1);
    }
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(sbase + L::kBarAccFull + 8 * s, 1);
      mbar_init(sbase + L::kBarAccEmpty + 8 * s, 2 * L::kEpiWarps);   // both CTAs' (used in the leader)
    }
    *abort_flag = 0u;
    fence_barrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_t128);
    tma_prefetch_desc(&tmap_t32);
    tma_prefetch_desc(&tmap_w16);
    tma_prefetch_desc(&tmap_t16);
  }
  if (warp == 0) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_dependency_wait();
  grid_launch_dependents();

  // the largest group decides what a stage holds, and so the depth of the ring
  int most = 0;
  for (int g = lane; g < p.l; g += 32) {
    int rows, off;
    fp8_group(p, g, rows, off);
    most = max(most, rows);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  const int stage_bytes = L::kW + (most <= L::kFewTokens ? ((most + 31) & ~31) * 64 : min((most + 31) & ~31, 128) * 128);
  const int stages = min(L::kRing / stage_bytes, L::kMaxStages);

  if (warp >= L::kEpiWarps) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kConsumerRegs));

  // (consumers first: with their branch last the compiler spilled 1.8 KB a thread)
  if (warp < L::kEpiWarps) {
    // ------------------------------ consumers (both CTAs) -----------------------
    Fp8Cursor cur;
    Fp8Tile tile;
    const int quad = warp & 3, part = warp >> 2;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t box = sbase + L::kOffBox + warp * L::kBoxBytes;
    uint32_t slot = 0, parity = 0;     // of the accumulators
    bool ok = true;
    for (int t = pair; ok; t += npairs) {
      if (!cur.seek(p, ntiles, t, tile)) break;
      const int col0 = part * (tile.few ? 32 : L::kPartCols);   // this part's accumulator columns
      // the tokens of this warp's lanes' scales: its accumulator lanes, or where tokens are few its columns
      const int mine = tile.row0 + (tile.few ? col0 : (int)rank * 128 + quad * 32);
      // nothing to add up for this warp (it still hands the accumulators back); columns behind the tile's are
      // added up all the same, and not stored
      const bool idle = mine >= tile.row0 + tile.tn || col0 >= tile.width;
      const float* sa_row = p.sfa + min(mine + lane, p.pitch - 1);
      const float* sb_row = p.sfb + ((size_t)tile.g * p.nblocks +
                                     min(tile.nt * 2 + (tile.few ? (int)rank : part), p.nblocks - 1)) * p.kblocks;
      float acc[L::kPartCols];
#pragma unroll
      for (int i = 0; i < L::kPartCols; ++i) acc[i] = 0.0f;
      // The scales of four K blocks are on their way while four are used: they come from L2, which under
      // this load takes longer than a block.
      float s_next[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s_next[i] = i < p.kblocks ? ld_ordered(sa_row + (size_t)i * p.pitch) * ld_ordered(sb_row + i) : 0.0f;
      for (int kb0 = 0; kb0 < p.kblocks && ok; kb0 += 4) {
        float s_now[4], sa[4], sb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s_now[i] = s_next[i];
          const int kb = min(kb0 + 4 + i, p.kblocks - 1);
          sa[i] = ld_ordered(sa_row + (size_t)kb * p.pitch);
          sb[i] = ld_ordered(sb_row + kb);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb0 + i < p.kblocks && ok) {
            ok = warp_wait(sbase + L::kBarAccFull + 8 * slot, parity, abort_flag, p.status, 4);
            tc_fence_after_sync();
            const uint32_t tacc = tmem_base + lane_base + slot * 256 + col0;
            const uint32_t empty = (sbase + L::kBarAccEmpty + 8 * slot) & kLeaderMask;
            if (++slot == L::kSlots) {
              slot = 0;
              parity ^= 1u;
            }
            if (idle || !ok) {
              tc_fence_before_sync();
              if (lane == 0) mbar_arrive_cluster(empty);
            } else if (tile.few) {
              uint32_t d[32];
              tmem_ld_32x32b_x32(tacc, d);
              tmem_ld_wait();
              tc_fence_before_sync();
              if (lane == 0) mbar_arrive_cluster(empty);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                acc[e] = fmaf(__uint_as_float(d[e]), __shfl_sync(0xffffffffu, s_now[i], e), acc[e]);
            } else {
              // (no branches in here: the compiler then reads the next piece while it adds this one)
#pragma unroll
              for (int c = 0; c < L::kPartCols / 32; ++c) {
                uint32_t d[32];
                tmem_ld_32x32b_x32(tacc + c * 32, d);
                tmem_ld_wait();
                if (c == L::kPartCols / 32 - 1) {   // all read: the accumulator may be overwritten
                  tc_fence_before_sync();
                  if (lane == 0) mbar_arrive_cluster(empty);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[c * 32 + e] = fmaf(__uint_as_float(d[e]), s_now[i], acc[c * 32 + e]);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s_next[i] = sa[i] * sb[i];
      }
      if (!ok) break;

      // ---- the sums leave, 32 columns at a time: turned around in the warp's box so that four lanes write
      // 64 neighbouring bytes of a token
      if (idle) continue;
      const float rs = p.row_scale && mine + lane < p.rows_total ? ld_ordered(p.row_scale + mine + lane) : 1.0f;
      const int first = tile.row0 + tile.lead, last = tile.row0 + tile.tn;
      if (tile.few) {
        // lanes are neighbouring columns of a token already
        const int col = tile.nt * 256 + (int)rank * 128 + quad * 32 + lane;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float v = acc[e] * __shfl_sync(0xffffffffu, rs, e);
          const int row = mine + e;
          if (row >= first && row < last && col < p.n) store_value(p, (size_t)row * p.n + col, v);
        }
        continue;
      }
#pragma unroll
      for (int c = 0; c < L::kPartCols / 32; ++c) {
        const int col = tile.nt * 256 + col0 + c * 32;
        if (col >= p.n) break;
        if (p.out_type == 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {   // 16 columns are 64 bytes
            __syncwarp();                 // the box has been read
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* v = acc + c * 32 + h * 16 + i * 4;
              st_shared_v4(box + lane * L::kBoxPitch + i * 16, __float_as_uint(v[0] * rs), __float_as_uint(v[1] * rs),
                           __float_as_uint(v[2] * rs), __float_as_uint(v[3] * rs));
            }
            __syncwarp();
            store_box(p, box, mine, first, last, col + h * 16, 4, lane);
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack_16bit(acc[c * 32 + 8 * i + 2 * j] * rs, acc[c * 32 + 8 * i + 2 * j + 1] * rs, p.out_type);
            st_shared_v4(box + lane * L::kBoxPitch + i * 16, w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          store_box(p, box, mine, first, last, col, 2, lane);
        }
      }
    }
  } else if (warp == kProducerWarp) {
    // ------------------------------ producer (both CTAs) ------------------------
    Fp8Cursor cur;
    Fp8Tile tile;
    uint32_t bits = 0;                 // parity per stage
    int s = 0;
    bool ok = true;
    for (int t = pair; ok; t += npairs) {
      if (!cur.seek(p, ntiles, t, tile)) break;
      // rows of this CTA: weights in boxes of 128 or 16, tokens in boxes of 128, 32 or 16
      const int wrows = tile.few ? 128 : tile.width >> 1;
      const int wrow = tile.g * p.n + tile.nt * 256 + (int)rank * wrows;
      const int tokens0 = tile.few ? tile.width >> 1 : (min(tile.tn, 128) + 31) & ~31;
      const int tokens1 = tile.few ? tile.width >> 1 : (max(tile.tn - 128, 0) + 31) & ~31;
      const int tokens = leader ? tokens0 : tokens1, trow = tile.row0 + (int)rank * (tile.few ? tokens0 : 128);
      const uint32_t bytes = (uint32_t)(2 * wrows + tokens0 + tokens1) * 128u;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        ok = warp_wait(sbase + L::kBarEmpty + 8 * s, ((bits >> s) & 1u) ^ 1u, abort_flag, p.status, 1);
        if (!ok) break;
        bits ^= 1u << s;
        const uint32_t full = sbase + L::kBarFull + 8 * s;
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(full, bytes);
          uint32_t dst = sbase + L::kOffRing + s * stage_bytes;
          if (wrows == 128) {
            tma_load_2d_pair(dst, &tmap_w, full, kb * 128, wrow);
          } else {
            for (int i = 0; i < wrows; i += 16) tma_load_2d_pair(dst + i * 128, &tmap_w16, full, kb * 128, wrow + i);
          }
          dst += L::kW;
          if (tokens == 128) {
            tma_load_2d_pair(dst, &tmap_t128, full, kb * 128, trow);
          } else {
            int i = 0;
            for (; i + 32 <= tokens; i += 32) tma_load_2d_pair(dst + i * 128, &tmap_t32, full, kb * 128, trow + i);
            if (i < tokens) tma_load_2d_pair(dst + i * 128, &tmap_t16, full, kb * 128, trow + i);
          }
        }
        __syncwarp();
        s = (s + 1 == stages) ? 0 : s + 1;
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------ MMA issuer (leader only) --------------------
    if (leader) {
      Fp8Cursor cur;
      Fp8Tile tile;
      uint32_t bits = 0, slot = 0, parity = 1;
      int s = 0;
      bool ok = true;
      const uint64_t wdesc0 = operand_desc_sw128(sbase + L::kOffRing);
      const uint64_t tdesc0 = operand_desc_sw128(sbase + L::kOffRing + L::kW);
      for (int t = pair; ok; t += npairs) {
        if (!cur.seek(p, ntiles, t, tile)) break;
        const uint32_t idesc = kIdescBase | ((uint32_t)(tile.width >> 3) << 17);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = warp_wait(sbase + L::kBarFull + 8 * s, (bits >> s) & 1u, abort_flag, p.status, 3) &&
               warp_wait(sbase + L::kBarAccEmpty + 8 * slot, parity, abort_flag, p.status, 2);
          if (!ok) break;
          bits ^= 1u << s;
          tc_fence_after_sync();
          const uint32_t at = (uint32_t)s * ((uint32_t)stage_bytes >> 4);   // descriptors count 16-byte units
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tc_mma_f8_pair(tmem_base + slot * 256, (tile.few ? wdesc0 : tdesc0) + at + 2 * j, (tile.few ? tdesc0 : wdesc0) + at + 2 * j, idesc, j > 0 ? 1u : 0u);
            tc_commit_pair(sbase + L::kBarAccFull + 8 * slot, 3);
            tc_commit_pair(sbase + L::kBarEmpty + 8 * s, 3);
          }
          __syncwarp();
          s = (s + 1 == stages) ? 0 : s + 1;
          if (++slot == L::kSlots) {
            slot = 0;
            parity ^= 1u;
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up somewhere: give loads still in flight time to land before the shared memory they
    // target is released
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  cluster_sync();   // neither CTA leaves while the other may still read its memory or signal it
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

static int gemm_fp8_block(const void* a_q, const float* a_sf, const void* b_q, const float* b_sf,
                          const int32_t* group_offsets, const int32_t* group_rows, const float* row_scale, void* out,
                          int out_type, int l, int rows_total, int n, int k, int max_ctas, void* stream) {
  if (!a_q || !a_sf || !b_q || !b_sf || !out) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (l <= 0 || n <= 0 || k <= 0 || rows_total < 0)
    return fail(MSC_ERR_BAD_ARG, "l=%d, n=%d, k=%d must be positive, rows=%d must not be negative", l, n, k, rows_total);
  if (k % 16) return fail(MSC_ERR_BAD_ARG, "k=%d must be a multiple of 16", k);
  if (n % 8) return fail(MSC_ERR_BAD_ARG, "n=%d must be a multiple of 8", n);
  if (out_type < 0 || out_type > 2) return fail(MSC_ERR_UNSUPPORTED, "out_dtype must be 0 (bf16), 1 (f32) or 2 (f16), got %d", out_type);
  if (max_ctas < 0) return fail(MSC_ERR_BAD_ARG, "max_ctas=%d must not be negative", max_ctas);
  for (const void* ptr : {a_q, static_cast<const void*>(a_sf), b_q, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16)
      return fail(MSC_ERR_BAD_ARG, "operands, a_sf and out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(b_sf) % 4 || reinterpret_cast<uintptr_t>(row_scale) % 4)
    return fail(MSC_ERR_BAD_ARG, "b_sf and row_scale must be 4-byte aligned");
  // tile coordinates are 32 bits
  if ((long long)l * n > 0x7fffff00LL) return fail(MSC_ERR_UNSUPPORTED, "l * n = %lld weight rows are too many", (long long)l * n);
  if (rows_total > 0x7ffffe00) return fail(MSC_ERR_UNSUPPORTED, "rows=%d are too many", rows_total);
  const long long ntiles = (n + 255) / 256;
  const long long max_tiles = ((long long)rows_total / 256 + (group_rows ? 2LL * l : 1LL)) * ntiles;
  if (max_tiles > 0x7fff0000LL) return fail(MSC_ERR_UNSUPPORTED, "the problem has too many tiles");
  if (rows_total == 0) return MSC_OK;
  int* status = status_word();
  if (!status) return fail(MSC_ERR_CUDA, "status word unavailable on this device");

  CUtensorMap tw, tw16, t128, t32, t16;
  if (int rc = make_tmap_bytes_2d(&tw, b_q, (uint64_t)l * n, (uint64_t)k, 128)) return rc;
  if (int rc = make_tmap_bytes_2d(&tw16, b_q, (uint64_t)l * n, (uint64_t)k, 16)) return rc;
  if (int rc = make_tmap_bytes_2d(&t128, a_q, (uint64_t)rows_total, (uint64_t)k, 128)) return rc;
  if (int rc = make_tmap_bytes_2d(&t32, a_q, (uint64_t)rows_total, (uint64_t)k, 32)) return rc;
  if (int rc = make_tmap_bytes_2d(&t16, a_q, (uint64_t)rows_total, (uint64_t)k, 16)) return rc;

  Fp8Params p;
  p.sfa = a_sf; p.sfb = b_sf; p.row_scale = row_scale;
  p.group_rows = group_rows; p.group_offsets = group_offsets;
  p.out = out; p.out_type = out_type; p.status = status;
  p.l = l; p.n = n; p.rows_total = rows_total; p.pitch = (rows_total + 3) & ~3;
  p.kblocks = (k + 127) / 128; p.nblocks = (n + 127) / 128;
  const int sms = num_sms();
  if (sms <= 0) return fail(MSC_ERR_CUDA, "could not query the SM count");
  int pairs = (max_ctas > 0 && max_ctas < sms ? max_ctas : sms) / 2;
  if (pairs < 1) pairs = 1;
  if (pairs > max_tiles) pairs = (int)max_tiles;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(gemm_fp8_block_kernel), Fp8Smem::kAlloc)) return rc;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config(2 * pairs, Fp8Smem::kThreads, Fp8Smem::kAlloc, static_cast<cudaStream_t>(stream), attr);
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, gemm_fp8_block_kernel, tw, tw16, t128, t32, t16, p));
  return MSC_OK;
}

}  // namespace msc

extern "C" {

int msc_gemm_fp8_block(const void* a_q, const float* a_sf, const void* b_q, const float* b_sf, void* out, int out_dtype,
                       int m, int n, int k, int max_ctas, void* stream) {
  return msc::gemm_fp8_block(a_q, a_sf, b_q, b_sf, nullptr, nullptr, nullptr, out, out_dtype, 1, m, n, k, max_ctas, stream);
}

int msc_grouped_gemm_fp8_block_ragged(const void* a_q, const float* a_sf, const void* b_q, const float* b_sf,
                                      const int32_t* group_offsets, const int32_t* group_rows, const float* row_scale,
                                      void* out, int out_dtype, int l, int rows_total, int n, int k, int max_ctas,
                                      void* stream) {
  if (!group_offsets || !group_rows) return msc::fail(MSC_ERR_BAD_ARG, "group_offsets and group_rows are required");
  return msc::gemm_fp8_block(a_q, a_sf, b_q, b_sf, group_offsets, group_rows, row_scale, out, out_dtype, l, rows_total, n, k,
                             max_ctas, stream);
}

}  // extern "C"
