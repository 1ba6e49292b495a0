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
// (64 groups of 48 tokens, 4096 x 2048: 135 us, 147 with tokens on M; of 64 tokens 139 against 150.)
//
// A dense product with fewer tiles than half the chip has CTA pairs is split along K: clusters of two or
// four pairs take a tile, leave their sums in shared memory and each adds up its share of the columns, in the order
// of K.  And where the last round of a dense product's tiles would keep only a few pairs busy, its tiles are
// taken in quarters of 64 tokens.
//
// What bounds it.  Large products: the consumers, who read 256 columns of a K block out of tensor memory, add them and hand
// them back.  The MMAs of a K block take 513 cycles, and a block, with its share of a tile's stores, 890: over 8192 x
// 8192 x 7168 the tensor pipe is active in 57 % of the cycles, and it runs in 420 to 450 us, 2.1 to 2.3
// PFLOP/s, 65 to 69 % of twice the measured bf16 rate (the MX kernel, whose scales the tensor core applies, 307 us).
// Wider or more consumer groups do not fit the registers, scales from a ring in shared memory cost more of its bandwidth
// than they save (490 us), and accumulators of 128 columns in turn double the hand-overs.  Few tokens: the weights'
// traffic (64 groups of 0 to 16 rows, 4096 x 7168: 306 us back to back, 338 in turn with others, 5.4 to 6 TB/s) or, for one
// small matrix, the launch and the ring's first fill (16 x 7168 x 2048: 10 to 12 us).
#include "gemm_common.cuh"
#include "quantize_common.cuh"

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
  int splits;                // pairs of a cluster, each with a share of K; > 1: one tile per cluster
  int quarters_from;         // dense: tiles from this one on are taken as four of 64 tokens
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

__device__ __forceinline__ void fp8_group(const Fp8Params& p, int g, int& rows, int& off) {
  if (!p.group_rows) {
    rows = p.rows_total;
    off = 0;
    return;
  }
  load_group(p.group_rows, p.group_offsets, p.rows_total, g, rows, off);
}

__device__ __forceinline__ int fp8_token_tiles(int rows) { return (rows + 255) >> 8; }

struct Fp8Tile {
  int g, nt;        // group, weight tile of 256 rows
  int row0;         // first token row
  int tn;           // tokens
  bool few;         // the weights are the M side
  int width;        // the N side: weight rows, or tokens where they are few, rounded up to 32
};

struct Fp8Cursor {
  GroupWindow<true> win;
  __device__ __forceinline__ bool seek(const Fp8Params& p, int ntiles, int t, Fp8Tile& tile) {
    if (!p.group_rows) {   // (a tile may come out empty)
      const int q = max(t - p.quarters_from, 0), tid = t < p.quarters_from ? t : p.quarters_from + (q >> 2);
      const int tt = tid / ntiles;
      tile.g = 0;
      tile.nt = tid - tt * ntiles;
      tile.row0 = tt * 256 + (q & 3) * 64;
      tile.tn = min(p.rows_total - tile.row0, t < p.quarters_from ? 256 : 64);
      shape(p, tile);
      return tt < fp8_token_tiles(p.rows_total);
    }
    int rows, off, first;
    if (!win.find(p.l, t, [&](int gi, int& r, int& o) { fp8_group(p, gi, r, o); },
                  [=](int r) { return fp8_token_tiles(r) * ntiles; }, tile.g, rows, off, first))
      return false;
    const int u = t - first, tt = u / ntiles;
    tile.nt = u - tt * ntiles;
    tile.row0 = off + tt * 256;
    tile.tn = min(rows - tt * 256, 256);
    shape(p, tile);
    return true;
  }
  static __device__ __forceinline__ void shape(const Fp8Params& p, Fp8Tile& tile) {
    tile.few = tile.tn <= Fp8Smem::kFewTokens;
    tile.width = tile.few ? (tile.tn + 31) & ~31 : min((p.n - tile.nt * 256 + 31) & ~31, 256);
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

__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
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
// Writes a box of 32 rows x 64 bytes out: rows [row0, last) of the matrix, columns col .. of `bytes` each.
__device__ __forceinline__ void store_box(const Fp8Params& p, uint32_t box, int row0, int last, int col, int bytes, int lane) {
  const int piece = lane & 3;
  const bool in = col + piece * (16 / bytes) < p.n;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = row0 + r * 8 + (lane >> 2);
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(box + (r * 8 + (lane >> 2)) * Fp8Smem::kBoxPitch + piece * 16) : "memory");
    if (in && row < last)
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + ((size_t)row * p.n + col) * bytes + piece * 16) = v;
  }
}

// The consumers' wait, made of as little code as its bound allows: it stands four times in the loop that sets the
// kernel's pace.  A probe suspends the warp for up to 20 us.
__device__ __forceinline__ bool wait_accumulators(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  for (int tries = 0; tries < 100000; ++tries) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0u)) return false;
  }
  return false;
}

// 32 accumulator columns of a warp's 32 lanes: piece pc of the tile.
__device__ __forceinline__ void store_piece(const Fp8Params& p, const Fp8Tile& tile, const float* v, int pc, int rank, int quad,
                                            int lane, uint32_t box) {
  const int mine = tile.row0 + (tile.few ? pc * 32 : rank * 128 + quad * 32);
  const float rs = p.row_scale && mine + lane < p.rows_total ? ld_ordered(p.row_scale + mine + lane) : 1.0f;
  const int last = tile.row0 + tile.tn;
  if (tile.few) {   // lanes are neighbouring columns of a token already
    const int col = tile.nt * 256 + rank * 128 + quad * 32 + lane;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const float x = v[e] * __shfl_sync(0xffffffffu, rs, e);
      if (mine + e < last && col < p.n) store_value(p, (size_t)(mine + e) * p.n + col, x);
    }
    return;
  }
  // turned around in the warp's box so that four lanes write 64 neighbouring bytes of a token
  const int col = tile.nt * 256 + pc * 32;
  if (col >= p.n) return;
  if (p.out_type == 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // 16 columns are 64 bytes
      __syncwarp();                 // the box has been read
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* x = v + h * 16 + i * 4;
        st_shared_v4(box + lane * Fp8Smem::kBoxPitch + i * 16, __float_as_uint(x[0] * rs), __float_as_uint(x[1] * rs),
                     __float_as_uint(x[2] * rs), __float_as_uint(x[3] * rs));
      }
      __syncwarp();
      store_box(p, box, mine, last, col + h * 16, 4, lane);
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_16bit(v[8 * i + 2 * j] * rs, v[8 * i + 2 * j + 1] * rs, p.out_type);
      st_shared_v4(box + lane * Fp8Smem::kBoxPitch + i * 16, w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    store_box(p, box, mine, last, col, 2, lane);
  }
}

__global__ void __launch_bounds__(Fp8Smem::kThreads, 1)
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
  const uint32_t cluster_rank = __shfl_sync(0xffffffffu, cluster_ctarank(), 0);
  const uint32_t rank = cluster_rank & 1u;   // in the pair
  const bool leader = rank == 0;
  const uint16_t both = (uint16_t)(3u << (cluster_rank & ~1u));
  const int pair = (int)blockIdx.x / (2 * p.splits), npairs = (int)gridDim.x / (2 * p.splits);   // or cluster
  const int share = (int)(cluster_rank >> 1);
  const int kb_lo = (int)((long long)p.kblocks * share / p.splits), kb_hi = (int)((long long)p.kblocks * (share + 1) / p.splits);
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
      if (tile.tn <= 0) continue;
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
      // One K block: waits for its accumulators, hands them back as soon as they are read.
      auto block = [&](float s) {
        if (!wait_accumulators(sbase + L::kBarAccFull + 8 * slot, parity, abort_flag)) {
          ok = false;
          return;
        }
        tc_fence_after_sync();
        const uint32_t tacc = tmem_base + lane_base + slot * 256 + col0;
        const uint32_t empty = (sbase + L::kBarAccEmpty + 8 * slot) & kLeaderMask;
        parity ^= slot;   // (two accumulators)
        slot ^= 1u;
        if (idle) {
          tc_fence_before_sync();
          if (lane == 0) mbar_arrive_cluster(empty);
        } else if (tile.few) {
          uint32_t d[32];
          tmem_ld_32x32b_x32(tacc, d);
          tmem_ld_wait();
          tc_fence_before_sync();
          if (lane == 0) mbar_arrive_cluster(empty);
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[e] = fmaf(__uint_as_float(d[e]), __shfl_sync(0xffffffffu, s, e), acc[e]);
        } else {
          // (no branches in here: the compiler then reads the next piece while it adds this one)
          const uint64_t s2 = pair_f32(s, s);
#pragma unroll
          for (int c = 0; c < L::kPartCols / 16; ++c) {
            uint32_t d[16];
            tmem_ld_32x32b_x16(tacc + c * 16, d);
            tmem_ld_wait();
            if (c == L::kPartCols / 16 - 1) {   // all read: the accumulator may be overwritten
              tc_fence_before_sync();
              if (lane == 0) mbar_arrive_cluster(empty);
            }
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float* a = acc + c * 16 + e;
              const float2 sum = unpair_f32(fma_f32x2(pair_f32(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), s2, pair_f32(a[0], a[1])));
              a[0] = sum.x;
              a[1] = sum.y;
            }
          }
        }
      };
      // The scales of four K blocks are on their way while four are used: they come from L2, which under
      // this load takes longer than a block.
      const float* sa_at = sa_row + (size_t)kb_lo * p.pitch;
      const float* sb_at = sb_row + kb_lo;
      const size_t step = p.pitch;
      int left = kb_hi - kb_lo;
      float sa[4] = {}, sb[4] = {};
      if (left >= 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sa[i] = ld_ordered(sa_at + i * step);
          sb[i] = ld_ordered(sb_at + i);
        }
      }
      while (left >= 4 && ok) {
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = sa[i] * sb[i];
        sa_at += 4 * step;
        sb_at += 4;
        left -= 4;
        if (left >= 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sa[i] = ld_ordered(sa_at + i * step);
            sb[i] = ld_ordered(sb_at + i);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (ok) block(s[i]);
      }
#pragma unroll 1
      for (; left > 0 && ok; --left, sa_at += step, ++sb_at) block(ld_ordered(sa_at) * ld_ordered(sb_at));
      if (!ok) {
        if (lane == 0) {
          *abort_flag = 1u;
          atomicCAS(p.status, 0, kStatusTimeout | 4);
        }
        break;
      }
      if (idle) continue;
      if (p.splits > 1) {   // left in the ring's memory, [column][lane]: nothing is loaded there any more
        const uint32_t sums = sbase + L::kOffRing + (uint32_t)(col0 * 128 + quad * 32 + lane) * 4;
#pragma unroll
        for (int i = 0; i < L::kPartCols; ++i)
          if (i < 32 || !tile.few) st_shared_f32(sums + i * 512, acc[i]);
        continue;
      }
#pragma unroll
      for (int c = 0; c < L::kPartCols / 32; ++c)
        if (c == 0 || !tile.few) store_piece(p, tile, acc + c * 32, part * (tile.few ? 1 : L::kPartCols / 32) + c, (int)rank, quad, lane, box);
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
      if (tile.tn <= 0) continue;
      // rows of this CTA: weights in boxes of 128 or 16, tokens in boxes of 128, 32 or 16
      const int wrows = tile.few ? 128 : tile.width >> 1;
      const int wrow = tile.g * p.n + tile.nt * 256 + (int)rank * wrows;
      const int tokens0 = tile.few ? tile.width >> 1 : (min(tile.tn, 128) + 31) & ~31;
      const int tokens1 = tile.few ? tile.width >> 1 : (max(tile.tn - 128, 0) + 31) & ~31;
      const int tokens = leader ? tokens0 : tokens1, trow = tile.row0 + (int)rank * (tile.few ? tokens0 : 128);
      const uint32_t bytes = (uint32_t)(2 * wrows + tokens0 + tokens1) * 128u;
      for (int kb = kb_lo; kb < kb_hi; ++kb) {
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
        if (tile.tn <= 0) continue;
        const uint32_t idesc = kIdescBase | ((uint32_t)(tile.width >> 3) << 17);
        const uint64_t adesc0 = tile.few ? wdesc0 : tdesc0, bdesc0 = tile.few ? tdesc0 : wdesc0;
        for (int kb = kb_lo; kb < kb_hi; ++kb) {
          ok = warp_wait(sbase + L::kBarFull + 8 * s, (bits >> s) & 1u, abort_flag, p.status, 3);
          if (!ok) break;
          bits ^= 1u << s;
          // all made ready before the wait: what lies between a free accumulator and the next product is on the
          // critical path
          const uint32_t at = (uint32_t)s * ((uint32_t)stage_bytes >> 4);   // descriptors count 16-byte units
          const uint64_t adesc = adesc0 + at, bdesc = bdesc0 + at;
          const uint32_t acc = tmem_base + slot * 256, full = sbase + L::kBarAccFull + 8 * slot, empty = sbase + L::kBarEmpty + 8 * s;
          ok = warp_wait(sbase + L::kBarAccEmpty + 8 * slot, parity, abort_flag, p.status, 2);
          if (!ok) break;
          tc_fence_after_sync();
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) tc_mma_f8_pair(acc, adesc + 2 * j, bdesc + 2 * j, idesc, j > 0 ? 1u : 0u);
            tc_commit_pair(full, both);
            tc_commit_pair(empty, both);
          }
          __syncwarp();
          s = (s + 1 == stages) ? 0 : s + 1;
          parity ^= slot;   // (two accumulators)
          slot ^= 1u;
        }
      }
    }
  }

  if (p.splits > 1) {
    cluster_sync();   // every pair's sums are in place
    Fp8Cursor cur;
    Fp8Tile tile;
    if (warp < L::kEpiWarps && cur.seek(p, ntiles, pair, tile) && tile.tn > 0) {
      const int quad = warp & 3;
      const uint32_t box = sbase + L::kOffBox + warp * L::kBoxBytes;
      const int pieces = tile.width >> 5;
      // lanes without a token are left out like the pairs' own warps left them out
      const bool there = tile.few || (int)rank * 128 + quad * 32 < tile.tn;
      for (int pc = share + p.splits * (warp >> 2); pc < pieces && there; pc += 2 * p.splits) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.0f;
        for (int s = 0; s < p.splits; ++s) {
          const uint32_t from = cluster_map_shared(sbase + L::kOffRing + (uint32_t)(pc * 4096 + quad * 32 + lane) * 4, 2 * s + rank);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] += ld_shared_cluster_f32(from + e * 512);
        }
        store_piece(p, tile, v, pc, (int)rank, quad, lane, box);
      }
    }
    __syncwarp();
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
  if (!b_q || !b_sf || (rows_total != 0 && (!a_q || !a_sf || !out))) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
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
  if (rows_total > 0x7ffffe00 || k > 0x7ffffe00) return fail(MSC_ERR_UNSUPPORTED, "rows=%d or k=%d is too large", rows_total, k);
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
  const int ctas = max_ctas > 0 && max_ctas < sms ? max_ctas : sms;
  const int room = ctas >= 2 ? ctas / 2 : 1;   // CTA pairs
  p.splits = 1;
  p.quarters_from = 0x7fffffff;
  long long units = max_tiles;                 // tiles, or clusters' pairs
  if (!group_rows) {
    const long long tiles = ((long long)rows_total + 255) / 256 * ntiles;
    const long long done = tiles / room * room;   // in full rounds
    units = tiles;
    // A share of K has 12 blocks at least: the sums' way through shared memory costs what a few blocks do
    // (64 x 2048 x 7168, four shares of 14: 22.6 us against 30.7; 16 x 7168 x 2048, two of 8: 18.4 against 16.4).
    while (p.splits < 4 && tiles * p.splits * 2 <= room && p.kblocks >= 24 * p.splits) p.splits *= 2;
    if (p.splits > 1) {
      units = tiles * p.splits;
    } else if (tiles > done && 4 * (tiles - done) <= room) {
      // A quarter to a pair (1024 x 5120 x 4096, 6 tiles in 24 quarters: 41.0 us against 45.1); where pairs would take
      // two of them nothing is gained (4101 x 7168 x 4096, 32 tiles: 133 us against 125).
      p.quarters_from = (int)done;
      units = done + 4 * (tiles - done);
    }
  }
  const int pairs = (int)(units < room ? units : room);
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(gemm_fp8_block_kernel), Fp8Smem::kAlloc)) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t lc = pdl_launch_config(2 * pairs, Fp8Smem::kThreads, Fp8Smem::kAlloc, static_cast<cudaStream_t>(stream), attr);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2u * (unsigned)p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1u;
  lc.numAttrs = 2;
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
