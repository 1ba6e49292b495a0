// FP8 matrix products with one fp32 scale per 128 columns of K, dense and over row-concatenated groups:
//
//   y[t, n] = row_scale[t] * sum_c sa[c, t] sb[n / 128, c] * sum_{k in block c} a[t, k] w[n, k]
//
// a, w e4m3; sa one fp32 scale per token and 128 columns, sb one per 128 x 128 block of the weights.
// The hardware's own block scales are powers of two (ue8m0), so the outer sum cannot stay in the
// tensor core: each K block of 128 is a product of its own in tensor memory, and the consumer warps add it,
// times its two scales, to sums in their registers (fp32 throughout).
//
// The weights are the MMA's M side (a CTA pair takes 256 weight rows, 128 per CTA, tensor-memory lane =
// weight row) and the tokens its N side, whose granularity of 32 makes a group of 272 rows cost 1.13
// tiles: a tile takes 256 tokens, the last one of a group up to 288.  A tile's tokens are up to three
// "subs" of up to 96, each an accumulator of its own; five accumulators rotate, so that some fill while
// others are read.  Four consumer warps belong to each sub; a warp holds 32 weight rows x 96 tokens of sums
// in registers and needs no other warp.
//
// Accumulators are read with the 16 x 256-bit form: a thread then has two neighbouring tokens of a weight
// row in neighbouring registers.  A quarter of the tokens meets each thread, so a token's scale is read
// from shared memory by a quarter of the lanes only (as pairs, for packed fp32 arithmetic), and the fragment is the one that
// stmatrix transposes: out rows are tokens.
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
  static constexpr int kSubs = 3;
  static constexpr int kSubTokens = 96;
  static constexpr int kTileTokens = kSubs * kSubTokens;   // most tokens of a tile
  static constexpr int kEpiWarps = 4 * kSubs;
  static constexpr int kThreads = (kEpiWarps + 4) * 32;   // whole warpgroups: two of the last four idle
  // Registers a thread: 128 at launch; the consumers need more than that, the others less.
  static constexpr int kConsumerRegs = 152, kOtherRegs = 56;
  static_assert(kEpiWarps * kConsumerRegs + 4 * kOtherRegs <= (kEpiWarps + 4) * 128, "the block was launched with no more");
  static constexpr int kMaxStages = 10;
  static constexpr int kSlots = 5;                 // accumulators
  static constexpr int kSlotCols = kSubTokens;
  static constexpr int kScales = 12;               // depth of a sub's ring of scales
  static constexpr int kScaleBytes = kSubTokens * 4;
  static constexpr int kBoxPitch = 80;             // a token's 32 16-bit columns, padded: no bank conflicts
  static constexpr int kBoxBytes = 32 * kBoxPitch;
  // barriers and flags | operand ring | scale rings | epilogue boxes
  static constexpr int kOffRing = 1024;
  static constexpr int kRing = 5 * (kW + kTileTokens * 64);
  static constexpr int kOffScale = kOffRing + kRing;
  static constexpr int kOffBox = kOffScale + kSubs * kScales * kScaleBytes;
  static constexpr int kTotal = kOffBox + kEpiWarps * kBoxBytes;
  static constexpr int kAlloc = kTotal + 1024;
  static_assert(kAlloc <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
  static_assert(kBoxBytes % 16 == 0 && kScaleBytes % 16 == 0, "bulk copies and vector accesses are 16-byte aligned");
  // barrier offsets
  static constexpr int kBarFull = 0;
  static constexpr int kBarEmpty = kBarFull + 8 * kMaxStages;
  static constexpr int kBarAccFull = kBarEmpty + 8 * kMaxStages;
  static constexpr int kBarAccEmpty = kBarAccFull + 8 * kSubs * kSlots;   // full: [sub][kSlots]; empty: per accumulator
  static constexpr int kBarScaleFull = kBarAccEmpty + 8 * kSlots;        // [sub][kScales]
  static constexpr int kBarScaleEmpty = kBarScaleFull + 8 * kSubs * kScales;
  static_assert(kBarScaleEmpty + 8 * kSubs * kScales <= 1000, "barriers and flags share the first 1024 bytes");
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

// Token tiles of a group: 256 each, the last one also taking a remainder of up to 32.
__device__ __forceinline__ int fp8_token_tiles(int rows) {
  if (rows <= 0) return 0;
  const int full = rows >> 8, rem = rows & 255;
  return full + ((rem == 0 || (rem <= 32 && full >= 1)) ? 0 : 1);
}

struct Fp8Tile {
  int g, nt;        // group, weight tile of 256 rows
  int row0, lead;   // first token row (a multiple of 4); rows of it that belong to somebody else
  int tn, units;    // tokens, in all and in units of 32
  __device__ __forceinline__ int subs() const { return min(units, Fp8Smem::kSubs); }
  __device__ __forceinline__ int width(int h) const { return (units + 2 - h) / 3 * 32; }   // tokens of sub h
  __device__ __forceinline__ int first(int h) const { return h == 0 ? 0 : h == 1 ? width(0) : width(0) + width(1); }
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
    tile.tn = (tt == fp8_token_tiles(rows) - 1) ? rows - tt * 256 : 256;
    tile.units = (tile.tn + 31) >> 5;
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

// 16 lanes x 8 N consecutive columns: r[4 j + 2 h + e] of thread t is lane t / 4 + 8 h, column
// 8 j + 2 (t % 4) + e.
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
               ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint64_t ld_shared_f32x2(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t pack_u32x2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float2 f32x2_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_16bit(float2 v, int out_type) {
  if (out_type == 0) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Fp8Smem::kThreads, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t48,
                      const __grid_constant__ CUtensorMap tmap_t32, const __grid_constant__ CUtensorMap tmap_t16,
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
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int ntiles = (p.n + 255) >> 8;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kMaxStages; ++s) {
      mbar_init(sbase + L::kBarFull + 8 * s, 1);
      mbar_init(sbase + L::kBarEmpty + 8 * s, 1);
    }
    for (int s = 0; s < L::kSubs * L::kSlots; ++s) mbar_init(sbase + L::kBarAccFull + 8 * s, 1);
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(sbase + L::kBarAccEmpty + 8 * s, 8);   // four warps of each CTA (used in the leader)
    }
    for (int s = 0; s < L::kSubs * L::kScales; ++s) {
      mbar_init(sbase + L::kBarScaleFull + 8 * s, 1);
      mbar_init(sbase + L::kBarScaleEmpty + 8 * s, 4);
    }
    *abort_flag = 0u;
    fence_barrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_t48);
    tma_prefetch_desc(&tmap_t32);
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
  const int stage_bytes = L::kW + (most > 256 ? L::kTileTokens : (most + 31) & ~31) * 64;
  const int stages = min(L::kRing / stage_bytes, L::kMaxStages);

  if (warp >= L::kEpiWarps) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kConsumerRegs));

  // (consumers first: with their branch last the compiler spilled 1.8 KB a thread)
  if (warp < L::kEpiWarps) {
    // ------------------------------ consumers (both CTAs) -----------------------
    Fp8Cursor cur;
    Fp8Tile tile;
    const int quad = warp & 3, sub = warp >> 2;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t box = sbase + L::kOffBox + warp * L::kBoxBytes;
    // Accumulators go round over all subs, barriers that announce them over this sub's own: a sub that sits
    // a tile out would otherwise meet a barrier any number of phases behind, where a parity says nothing.
    uint32_t seq = 0;                  // accumulators produced before this tile
    int af = 0;
    uint32_t af_parity = 0;
    int ss = 0;
    uint32_t sbits = 0;
    bool ok = true;
    for (int t = pair; ok; t += npairs) {
      if (!cur.seek(p, ntiles, t, tile)) break;
      const int subs = tile.subs();
      const uint32_t seq0 = seq + sub;
      seq += (uint32_t)(subs * p.kblocks);
      const int width = tile.width(sub);
      if (width == 0) continue;
      // weight blocks beyond the matrix (rows that are not stored) take the last block's scale
      const int nb = min(tile.nt * 2 + (int)rank, p.nblocks - 1);
      const float* sb_row = p.sfb + ((size_t)tile.g * p.nblocks + nb) * p.kblocks;
      float sb_lane = 0.0f;
      uint64_t acc[L::kSubTokens / 2];   // [16-token step][lane half][j][h]: pairs of tokens
#pragma unroll
      for (int i = 0; i < L::kSubTokens / 2; ++i) acc[i] = 0ull;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if ((kb & 31) == 0) sb_lane = kb + lane < p.kblocks ? ld_ordered(sb_row + kb + lane) : 0.0f;
        const float sb = __shfl_sync(0xffffffffu, sb_lane, kb & 31);
        const uint64_t sb2 = pack_u32x2(__float_as_uint(sb), __float_as_uint(sb));
        const int sslot = sub * L::kScales + ss;
        const uint32_t now = seq0 + (uint32_t)(subs * kb), slot = now % L::kSlots;
        ok = warp_wait(sbase + L::kBarScaleFull + 8 * sslot, (sbits >> ss) & 1u, abort_flag, p.status, 6) &&
             warp_wait(sbase + L::kBarAccFull + 8 * (sub * L::kSlots + af), af_parity, abort_flag, p.status, 4);
        if (!ok) break;
        if (++af == L::kSlots) {
          af = 0;
          af_parity ^= 1u;
        }
        sbits ^= 1u << ss;
        tc_fence_after_sync();
        const uint32_t tacc = tmem_base + lane_base + slot * L::kSlotCols;
        const uint32_t sc = sbase + L::kOffScale + sslot * L::kScaleBytes + (lane & 3) * 8;
        // steps of 16 tokens, the next one's accumulators on their way while one is added
        uint32_t d[2][2][8];
        tmem_ld_16x256b_x2(tacc, d[0][0]);
        tmem_ld_16x256b_x2(tacc + (16u << 16), d[0][1]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < L::kSubTokens / 16; ++c) {
          if (c * 16 < width) {
            if ((c + 1) * 16 < width) {
              tmem_ld_16x256b_x2(tacc + (c + 1) * 16, d[(c + 1) & 1][0]);
              tmem_ld_16x256b_x2(tacc + (c + 1) * 16 + (16u << 16), d[(c + 1) & 1][1]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint64_t s2 = f32x2_mul(ld_shared_f32x2(sc + c * 64 + j * 32), sb2);
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int i = c * 8 + hh * 4 + j * 2 + h;
                  acc[i] = f32x2_fma(pack_u32x2(d[c & 1][hh][4 * j + 2 * h], d[c & 1][hh][4 * j + 2 * h + 1]), s2, acc[i]);
                }
            }
            tmem_ld_wait();
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster((sbase + L::kBarAccEmpty + 8 * slot) & kLeaderMask);
          mbar_arrive(sbase + L::kBarScaleEmpty + 8 * sslot);
        }
        ss = (ss + 1 == L::kScales) ? 0 : ss + 1;
      }
      if (!ok) break;

      // ---- the sums leave: tokens [first, last) of the tile, this warp's 32 output columns -------------
      const int tok0 = tile.first(sub);
      const int col = tile.nt * 256 + (int)rank * 128 + quad * 32;
      if (col >= p.n) continue;
#pragma unroll
      for (int c = 0; c < L::kSubTokens / 16; ++c) {
        if (c * 16 < width) {
          const int tok_a = tok0 + c * 16 + (lane & 3) * 2;   // this thread's tokens: tok_a + 8 j + {0, 1}
          if (p.row_scale) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int row = tile.row0 + tok_a + j * 8;
              const float r0 = row < p.rows_total ? ld_ordered(p.row_scale + row) : 0.0f;
              const float r1 = row + 1 < p.rows_total ? ld_ordered(p.row_scale + row + 1) : 0.0f;
              const uint64_t r2 = pack_u32x2(__float_as_uint(r0), __float_as_uint(r1));
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int h = 0; h < 2; ++h) acc[c * 8 + hh * 4 + j * 2 + h] = f32x2_mul(acc[c * 8 + hh * 4 + j * 2 + h], r2);
            }
          }
          if (p.out_type == 1) {
            // a store instruction writes 8 neighbouring columns of 4 tokens: whole 32-byte sectors
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float2 v = f32x2_split(acc[c * 8 + hh * 4 + j * 2 + h]);
                  const int tok = tok_a + j * 8;
                  const int cc = col + hh * 16 + h * 8 + (lane >> 2);
                  float* dst = static_cast<float*>(p.out) + (size_t)(tile.row0 + tok) * p.n + cc;
                  if (cc < p.n) {
                    if (tok >= tile.lead && tok < tile.tn) dst[0] = v.x;
                    if (tok + 1 >= tile.lead && tok + 1 < tile.tn) dst[p.n] = v.y;
                  }
                }
          } else {
            const uint32_t part = box + (c & 1) * 16 * L::kBoxPitch;   // the halves of the box in turn
            if (c & 1) __syncwarp();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int b = 0; b < 4; ++b) w[b] = pack_16bit(f32x2_split(acc[c * 8 + (b >> 1) * 4 + j * 2 + (b & 1)]), p.out_type);
              stmatrix_x4_trans(part + (j * 8 + (lane & 7)) * L::kBoxPitch + (lane >> 3) * 16, w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int in = r * 8 + (lane >> 2), piece = lane & 3;
              const int tok = tok0 + c * 16 + in;
              uint4 v;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(part + in * L::kBoxPitch + piece * 16) : "memory");
              if (tok >= tile.lead && tok < tile.tn && col + piece * 8 < p.n)
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) +
                                          ((size_t)(tile.row0 + tok) * p.n + col + piece * 8) * 2) = v;
            }
          }
        }
      }
    }
  } else if (warp == kProducerWarp) {
    // ------------------------------ producer (both CTAs) ------------------------
    Fp8Cursor cur;
    Fp8Tile tile;
    uint32_t bits = 0;                 // parity per stage
    int s = 0;
    int ss[L::kSubs] = {};             // scale rings
    uint32_t sbits[L::kSubs] = {};
    bool ok = true;
    for (int t = pair; ok; t += npairs) {
      if (!cur.seek(p, ntiles, t, tile)) break;
      const int wrow = tile.g * p.n + tile.nt * 256 + (int)rank * 128;
      const uint32_t bytes = L::kW + (uint32_t)tile.units * (16 * 128);   // weights and half of the tokens
      for (int kb = 0; kb < p.kblocks && ok; ++kb) {
        ok = warp_wait(sbase + L::kBarEmpty + 8 * s, ((bits >> s) & 1u) ^ 1u, abort_flag, p.status, 1);
        if (!ok) break;
        bits ^= 1u << s;
        const uint32_t full = sbase + L::kBarFull + 8 * s;
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(full, 2 * bytes);
          uint32_t dst = sbase + L::kOffRing + s * stage_bytes;
          tma_load_2d_pair(dst, &tmap_w, full, kb * 128, wrow);
          dst += L::kW;
#pragma unroll
          for (int h = 0; h < L::kSubs; ++h) {
            const int rows = tile.width(h) >> 1;   // this CTA's: 0, 16, 32 or 48
            const int row = tile.row0 + tile.first(h) + (int)rank * rows;
            if (rows) tma_load_2d_pair(dst, rows == 48 ? &tmap_t48 : rows == 32 ? &tmap_t32 : &tmap_t16, full, kb * 128, row);
            dst += (uint32_t)rows * 128u;
          }
        }
        __syncwarp();
        s = (s + 1 == stages) ? 0 : s + 1;
#pragma unroll
        for (int h = 0; h < L::kSubs; ++h) {
          const int width = tile.width(h);
          if (width == 0 || !ok) continue;
          const int slot = h * L::kScales + ss[h];
          ok = warp_wait(sbase + L::kBarScaleEmpty + 8 * slot, ((sbits[h] >> ss[h]) & 1u) ^ 1u, abort_flag, p.status, 5);
          if (!ok) continue;
          sbits[h] ^= 1u << ss[h];
          const int row = tile.row0 + tile.first(h);
          const uint32_t sbytes = (uint32_t)min(width, p.pitch - row) * 4u;
          if (elect_one()) {
            mbar_arrive_expect_tx(sbase + L::kBarScaleFull + 8 * slot, sbytes);
            bulk_load_1d(sbase + L::kOffScale + slot * L::kScaleBytes, p.sfa + (size_t)kb * p.pitch + row, sbytes,
                         sbase + L::kBarScaleFull + 8 * slot);
          }
          __syncwarp();
          ss[h] = (ss[h] + 1 == L::kScales) ? 0 : ss[h] + 1;
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------ MMA issuer (leader only) --------------------
    if (leader) {
      Fp8Cursor cur;
      Fp8Tile tile;
      uint32_t bits = 0, slot = 0, slot_bits = 0;
      int s = 0, af[L::kSubs] = {};
      bool ok = true;
      const uint64_t wdesc0 = operand_desc_sw128(sbase + L::kOffRing);
      const uint64_t tdesc0 = operand_desc_sw128(sbase + L::kOffRing + L::kW);
      for (int t = pair; ok; t += npairs) {
        if (!cur.seek(p, ntiles, t, tile)) break;
        const int subs = tile.subs();
        for (int kb = 0; kb < p.kblocks && ok; ++kb) {
          ok = warp_wait(sbase + L::kBarFull + 8 * s, (bits >> s) & 1u, abort_flag, p.status, 3);
          if (!ok) break;
          bits ^= 1u << s;
          const uint32_t at = (uint32_t)s * ((uint32_t)stage_bytes >> 4);   // descriptors count 16-byte units
#pragma unroll
          for (int h = 0; h < L::kSubs; ++h) {
            if (h >= subs || !ok) continue;
            ok = warp_wait(sbase + L::kBarAccEmpty + 8 * slot, ((slot_bits >> slot) & 1u) ^ 1u, abort_flag, p.status, 2);
            if (!ok) continue;
            slot_bits ^= 1u << slot;
            tc_fence_after_sync();
            const int width = tile.width(h);
            const uint32_t idesc = kIdescBase | ((uint32_t)(width >> 3) << 17);
            const uint64_t wdesc = wdesc0 + at;
            const uint64_t tdesc = tdesc0 + at + (uint32_t)tile.first(h) * 4u;   // half of them, 128 bytes each
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma_f8_pair(tmem_base + slot * L::kSlotCols, wdesc + 2 * j, tdesc + 2 * j, idesc, j > 0 ? 1u : 0u);
              tc_commit_pair(sbase + L::kBarAccFull + 8 * (h * L::kSlots + af[h]), 3);
              if (h == subs - 1) tc_commit_pair(sbase + L::kBarEmpty + 8 * s, 3);
            }
            __syncwarp();
            af[h] = (af[h] + 1 == L::kSlots) ? 0 : af[h] + 1;
            slot = (slot + 1 == L::kSlots) ? 0u : slot + 1;
          }
          s = (s + 1 == stages) ? 0 : s + 1;
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
  const long long max_tiles = ((long long)rows_total / 256 + (group_rows ? 2LL * l : 1)) * ntiles;
  if (max_tiles > 0x7fff0000LL) return fail(MSC_ERR_UNSUPPORTED, "the problem has too many tiles");
  if (rows_total == 0) return MSC_OK;
  int* status = status_word();
  if (!status) return fail(MSC_ERR_CUDA, "status word unavailable on this device");

  CUtensorMap tw, t48, t32, t16;
  if (int rc = make_tmap_bytes_2d(&tw, b_q, (uint64_t)l * n, (uint64_t)k, 128)) return rc;
  if (int rc = make_tmap_bytes_2d(&t48, a_q, (uint64_t)rows_total, (uint64_t)k, 48)) return rc;
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
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, gemm_fp8_block_kernel, tw, t48, t32, t16, p));
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
