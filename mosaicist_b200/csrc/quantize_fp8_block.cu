// FP8 with one fp32 scale per block: activations in blocks of 1 x 128, weights of 128 x 128 (both HBM-bound).
//
//   s = max(amax / 448, 2^-126)     in fp32, amax the block's largest magnitude, NaNs left out
//   q = e4m3_rne(x / s)             the quotient rounded to fp32 first
// (structure of the reference's block-scaled FP8 quantiser, experiments/flashinfer-megamoe-sm90a/quant.py:47-75,
// with fp32 scales per 128).  The floor of the scale keeps x / s finite in a block of zeros.  An
// infinite element makes its block's scale infinite: infinities come out NaN, the others 0.  NaN stays NaN.
//
// The scales of activations are laid out by block column, (ceil(k / 128), rows rounded up to 4): what the
// product reads for a tile of rows and one K step is then one contiguous, 16-byte aligned piece.
#include "host_common.h"
#include "ptx.cuh"
#include "quantize_common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace msc {

constexpr int kMostOfASize = 0x7ffffe00;   // rounding a size up to a tile's stays within 32 bits
constexpr float kFp8Max = 448.0f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126

__device__ __forceinline__ float block_scale(float amax) { return fmaxf(__fdiv_rn(amax, kFp8Max), kLeastScale); }

// 16 values / s -> 16 bytes of e4m3.  The quotients are those of __fdiv_rn wherever they decide an e4m3
// value, at three instructions for two of them (div_rn_shared_rcp; the remainder is exact while s is well inside
// fp32's exponents, and quotients below 2^-10 round to zero whatever their last bit is).
__device__ __forceinline__ uint4 pack_e4m3_16(const float* v, float s) {
  const bool mid = s >= 1e-25f && s <= 1e25f;
  const float r = __frcp_rn(s);
  const uint64_t r2 = pair_f32(r, r), n2 = pair_f32(-s, -s);
  uint32_t w[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    float2 x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float a = v[4 * h + 2 * j], b = v[4 * h + 2 * j + 1];
      if (mid) {
        const uint64_t a2 = pair_f32(a, b);
        const uint64_t q2 = mul_f32x2(a2, r2);
        x[j] = unpair_f32(fma_f32x2(fma_f32x2(q2, n2, a2), r2, q2));
      } else {
        x[j] = make_float2(__fdiv_rn(a, s), __fdiv_rn(b, s));
      }
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(x[0], __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(x[1], __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight 16-bit or four 32-bit values of a 16-byte vector as fp32.
template <class T> struct Vec16;
template <> struct Vec16<__nv_bfloat16> {
  static constexpr int kPer = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  // largest magnitude, NaNs left out; two values an instruction
  static __device__ __forceinline__ float amax(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3]))));
    return fmaxf(fmaxf(0.0f, f.x), f.y);
  }
};
template <> struct Vec16<__half> {
  static constexpr int kPer = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float amax(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const float2 f = __half22float2(__hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3]))));
    return fmaxf(fmaxf(0.0f, f.x), f.y);
  }
};
template <> struct Vec16<float> {
  static constexpr int kPer = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float amax(const uint4& r) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(r.x)), fabsf(__uint_as_float(r.y))),
                 fmaxf(fmaxf(0.0f, fabsf(__uint_as_float(r.z))), fabsf(__uint_as_float(r.w))));
  }
};

struct RowBlockParams {
  const void* x;             // (rows, k), with SILU (rows, 2k) gate | up
  uint8_t* q;                // (rows, k)
  float* sf;                 // (kblocks, pitch)
  const int* group_offsets;  // [l] or null: every row
  const int* group_rows;     // [l]
  int l, rows, pitch, k, kblocks;
};

// ---- activations ---------------------------------------------------------------------------
// A CTA takes 8 rows, a warp one of them, and walks its share of the row's pieces of 512 columns with the next
// piece's loads in flight; a thread holds 16 values, 8 lanes share a block.  The 32 scales of a
// piece meet in shared memory and leave as 32-byte stretches of the column layout.
// Measured: gate | up of 16300 rows x 2048 bf16 in 64 groups with silu, 167 MB moved in 36 us, 4.6 TB/s, with half of the issue
// slots, half of DRAM and 48 % of the special-function pipe in use: 71 registers a thread leave three CTAs on an SM,
// so that latency is what bounds it.  Without silu (61 registers, four CTAs) 16384 x 7168 takes 68 to 76 us, 4.6 to 5.2
// TB/s, with 70 to 75 % of the issue slots in use; 16 rows x 7168 4.1 to 4.7 us, which is the launch.
template <class T, bool SILU>
__global__ void __launch_bounds__(256) quantize_fp8_rows_kernel(const RowBlockParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ float s_scale[2][8][4];
  __shared__ unsigned s_live;
  constexpr int kVecs = 16 / Vec16<T>::kPer;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * 8, row = row0 + warp;

  // the rows of the tile that take part: all of them, or those that some group owns
  unsigned live = row0 + 8 <= p.rows ? 0xffu : (1u << max(p.rows - row0, 0)) - 1u;
  if (p.group_offsets) {
    if (threadIdx.x == 0) s_live = 0u;
    __syncthreads();
    for (int g = threadIdx.x; g < p.l; g += 256) {
      const long long off = ld_ordered(p.group_offsets + g);
      const long long lo = max(off - row0, 0LL), hi = min(off + ld_ordered(p.group_rows + g) - row0, 8LL);
      if (off >= 0 && lo < hi) atomicOr(&s_live, ((1u << (int)hi) - 1u) & ~((1u << (int)lo) - 1u));
    }
    __syncthreads();
    live &= s_live;
  }
  if (live == 0 && row0 + 8 <= p.rows) return;   // (the last rows' tile also clears the scale columns behind them)
  const bool mine = (live >> warp) & 1u;
  const T* src = static_cast<const T*>(p.x) + (size_t)row * p.k * (SILU ? 2 : 1) + lane * 16;
  uint4 raw[kVecs * (SILU ? 2 : 1)];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < kVecs * (SILU ? 2 : 1); ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (mine && c * 512 + lane * 16 < p.k) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        raw[i] = ld_ordered(reinterpret_cast<const uint4*>(src + c * 512) + i);
        if (SILU) raw[kVecs * (SILU ? 1 : 0) + i] = ld_ordered(reinterpret_cast<const uint4*>(src + p.k + c * 512) + i);
      }
    }
  };
  const int pieces = (p.k + 511) >> 9;
  load(blockIdx.y);
  for (int c = blockIdx.y, buf = 0; c < pieces; c += gridDim.y, buf ^= 1) {
    float v[16], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if (!SILU) amax = fmaxf(amax, Vec16<T>::amax(raw[i]));
      Vec16<T>::unpack(raw[i], v + i * Vec16<T>::kPer);
    }
    if (SILU) {
      float up[16];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) Vec16<T>::unpack(raw[kVecs * (SILU ? 1 : 0) + i], up + i * Vec16<T>::kPer);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = silu_mul(v[i], up[i]);
      amax = amax_f32x16(v);
    }
    if (c + (int)gridDim.y < pieces) load(c + gridDim.y);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = block_scale(amax);
    if ((lane & 7) == 0) s_scale[buf][warp][lane >> 3] = s;
    const int col = c * 512 + lane * 16;
    if (mine && col < p.k) *reinterpret_cast<uint4*>(p.q + (size_t)row * p.k + col) = pack_e4m3_16(v, s);
    __syncthreads();
    if (threadIdx.x < 32) {
      const int kb = c * 4 + (threadIdx.x >> 3), r = threadIdx.x & 7;
      if (kb < p.kblocks) {
        if ((live >> r) & 1u) p.sf[(size_t)kb * p.pitch + row0 + r] = s_scale[buf][r][threadIdx.x >> 3];
        else if (row0 + r >= p.rows && row0 + r < p.pitch) p.sf[(size_t)kb * p.pitch + row0 + r] = 0.0f;
      }
    }
  }
}

// ---- dispatch of the routed layer ------------------------------------------------------------
// CTAs walk the tokens; a token's row is quantised once into shared memory and leaves for the row of every
// expert it is routed to as one bulk copy, the scales as words of their column layout.  Two row buffers
// alternate, so the copies of one token leave while the next is quantised.
struct Fp8DispatchParams {
  const __nv_bfloat16* tokens;   // (tokens, hidden)
  const int* ids;                // (tokens, topk)
  const float* weights;          // (tokens, topk)
  const int* rank;               // (tokens, topk)
  const int* group_offsets;      // (experts_local)
  uint8_t* q;                    // (rows_cap, hidden)
  float* sf;                     // (kblocks, pitch)
  float* row_weight;             // (rows_cap)
  int* row_token;                // (rows_cap)
  int* status;
  int hidden, kblocks, topk, expert_first, experts_local, rows_cap, pitch;
};

constexpr int kFp8MaxTopk = 64;

__global__ void __launch_bounds__(512) moe_permute_quantize_fp8_kernel(const Fp8DispatchParams p, int tokens) {
  grid_dependency_wait();
  grid_launch_dependents();
  extern __shared__ __align__(16) uint8_t row_smem[];   // 2 x ([hidden] values, [kblocks] scales)
  __shared__ int s_dest[2][kFp8MaxTopk];
  const int row_bytes = (p.hidden + 4 * p.kblocks + 15) & ~15;
  const int padded = (p.hidden + 127) & ~127;           // the eight lanes of a block stay together
  int it = 0;
  for (long long token = blockIdx.x; token < tokens; token += gridDim.x, ++it) {
    const int buf = it & 1;
    uint8_t* s_q = row_smem + buf * row_bytes;
    float* s_sf = reinterpret_cast<float*>(s_q + p.hidden);
    // the copies of the token before last have read this buffer; the last token's may still run
    if (threadIdx.x == 0) bulk_wait_group_read1();
    if ((int)threadIdx.x < p.topk) {
      const long long pair = token * p.topk + threadIdx.x;
      const int e = ld_ordered(p.ids + pair) - p.expert_first;
      int dest = -1;
      if (e >= 0 && e < p.experts_local) {
        dest = ld_ordered(p.group_offsets + e) + ld_ordered(p.rank + pair);
        if (dest < 0 || dest >= p.rows_cap) {
          dest = -1;
          atomicOr(reinterpret_cast<unsigned*>(p.status), kStatusRowsOverflow);
        } else {
          p.row_weight[dest] = ld_ordered(p.weights + pair);
          p.row_token[dest] = (int)token;
        }
      }
      s_dest[buf][threadIdx.x] = dest;
    }
    __syncthreads();
    for (int col = threadIdx.x * 16; col < padded; col += blockDim.x * 16) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.0f;
      if (col < p.hidden) load16_bf16(p.tokens + (size_t)token * p.hidden + col, v);
      float amax = amax_f32x16(v);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffu << (threadIdx.x & 24u), amax, o));
      const float s = block_scale(amax);
      if (col < p.hidden) *reinterpret_cast<uint4*>(s_q + col) = pack_e4m3_16(v, s);
      if ((threadIdx.x & 7) == 0) s_sf[col >> 7] = s;
    }
    fence_proxy_async_smem();
    __syncthreads();
    for (int k = 0; k < p.topk; ++k) {
      const int dest = s_dest[buf][k];
      if (dest < 0) continue;
      if (threadIdx.x == 0) bulk_store_1d(p.q + (size_t)dest * p.hidden, smem_u32(s_q), (uint32_t)p.hidden);
      for (int c = threadIdx.x; c < p.kblocks; c += blockDim.x) p.sf[(size_t)c * p.pitch + dest] = s_sf[c];
    }
    if (threadIdx.x == 0) bulk_commit_group();    // one group per token (empty ones count too)
  }
  if (threadIdx.x == 0) bulk_wait_group0();       // a kernel that starts early follows: the rows are in place
}

// ---- weights -------------------------------------------------------------------------------
// A CTA per 128 x 128 block, whose values stay in registers between the maximum and the quotients: a
// thread holds 64 of them in four row pieces of 16.  Four CTAs an SM keep enough loads in flight: 16 x 4096 x 7168 bf16
// in 239 us back to back, 5.9 TB/s of read and written bytes, 259 us with two (266 where results go to other memory in every
// call); fp32 values take twice the registers and two CTAs.
struct WeightBlockParams {
  const void* w;    // (l, n, k)
  uint8_t* q;       // (l, n, k)
  float* sf;        // (l, nblocks, kblocks)
  int n, k, nblocks, kblocks;
};

template <class T>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 4) quantize_fp8_weight_kernel(const WeightBlockParams p) {
  __shared__ float s_amax[8];
  constexpr int kVecs = 16 / Vec16<T>::kPer;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t g = blockIdx.z;
  const int col = blockIdx.x * 128 + (lane & 7) * 16;
  const int row0 = blockIdx.y * 128 + warp * 4 + (lane >> 3);   // then every 32 rows
  const T* src = static_cast<const T*>(p.w) + (g * p.n + row0) * p.k + col;
  uint4 raw[4][kVecs];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      raw[i][j] = (row0 + 32 * i < p.n && col < p.k) ? __ldg(reinterpret_cast<const uint4*>(src + (size_t)32 * i * p.k) + j)
                                                     : make_uint4(0u, 0u, 0u, 0u);
  float amax = 0.0f;
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kVecs; ++j) amax = fmaxf(amax, Vec16<T>::amax(raw[i][j]));
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (lane == 0) s_amax[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, s_amax[i]);
  const float s = block_scale(amax);
  uint8_t* dst = p.q + (g * p.n + row0) * p.k + col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) Vec16<T>::unpack(raw[i][j], v + j * Vec16<T>::kPer);
    if (row0 + 32 * i < p.n && col < p.k) *reinterpret_cast<uint4*>(dst + (size_t)32 * i * p.k) = pack_e4m3_16(v, s);
  }
  if (threadIdx.x == 0) p.sf[(g * p.nblocks + blockIdx.y) * p.kblocks + blockIdx.x] = s;
}

template <class T>
static int launch_rows(const RowBlockParams& p, bool silu, cudaStream_t stream) {
  const int sms = num_sms();
  if (sms <= 0) return fail(MSC_ERR_CUDA, "could not query the SM count");
  // As many CTAs per row as it takes to give every SM sixteen, of which three or four are resident: with up to 64 the pieces of
  // many rows lose their loads in flight (gate | up of 64 groups 52 us against 36), with 4 a middling number
  // of rows fills the SMs badly (4096 x 2048 9.7 us against 8.4).
  const int tiles = (p.rows + 7) / 8, pieces = (p.k + 511) / 512;
  const int split = std::max(1, std::min(pieces, (16 * sms + tiles - 1) / tiles));
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config(tiles, 256, 0, stream, attr);
  lc.gridDim.y = (unsigned)split;
  auto kern = silu ? quantize_fp8_rows_kernel<T, true> : quantize_fp8_rows_kernel<T, false>;
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, kern, p));
  return MSC_OK;
}

}  // namespace msc

extern "C" {

int msc_fp8_block_quantize(const void* x, int x_dtype, int silu, const int32_t* group_offsets, const int32_t* group_rows,
                           void* q, float* sf, int l, int rows, int k, void* stream) {
  using namespace msc;
  if (rows != 0 && (!x || !q || !sf)) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (!group_offsets != !group_rows) return fail(MSC_ERR_BAD_ARG, "group_offsets and group_rows come together");
  if (group_offsets && l <= 0) return fail(MSC_ERR_BAD_ARG, "l=%d must be positive with groups", l);
  if (rows < 0 || k <= 0) return fail(MSC_ERR_BAD_ARG, "rows=%d must not be negative, k=%d must be positive", rows, k);
  if (k % 16) return fail(MSC_ERR_BAD_ARG, "k=%d must be a multiple of 16", k);
  if (x_dtype < 0 || x_dtype > 2) return fail(MSC_ERR_UNSUPPORTED, "x_dtype must be 0 (bf16), 1 (f32) or 2 (f16), got %d", x_dtype);
  if (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(sf) % 4)
    return fail(MSC_ERR_BAD_ARG, "x and q must be 16-byte aligned, sf 4-byte aligned");
  if (rows > kMostOfASize || k > kMostOfASize) return fail(MSC_ERR_UNSUPPORTED, "rows=%d or k=%d exceeds %d", rows, k, kMostOfASize);
  if (rows == 0) return MSC_OK;
  RowBlockParams p;
  p.x = x; p.q = static_cast<uint8_t*>(q); p.sf = sf;
  p.group_offsets = group_offsets; p.group_rows = group_rows; p.l = l;
  p.rows = rows; p.pitch = (rows + 3) & ~3; p.k = k; p.kblocks = (k + 127) / 128;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == 0 ? launch_rows<__nv_bfloat16>(p, silu != 0, st)
         : x_dtype == 1 ? launch_rows<float>(p, silu != 0, st) : launch_rows<__half>(p, silu != 0, st);
}

int msc_moe_permute_quantize_fp8_block(const void* tokens_bf16, const int32_t* ids, const float* weights,
                                       const int32_t* rank, const int32_t* group_offsets, int tokens, int hidden,
                                       int topk, int expert_first, int experts_local, void* a_q, float* a_sf,
                                       float* row_weight, int32_t* row_token, int rows_cap, void* stream) {
  using namespace msc;
  if (!tokens_bf16 || !ids || !weights || !rank || !group_offsets || !a_q || !a_sf || !row_weight || !row_token)
    return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (tokens < 0 || topk <= 0 || experts_local <= 0 || rows_cap <= 0)
    return fail(MSC_ERR_BAD_ARG, "tokens must not be negative, topk, experts_local and rows_cap must be positive");
  if (rows_cap > kMostOfASize) return fail(MSC_ERR_UNSUPPORTED, "rows_cap=%d exceeds %d", rows_cap, kMostOfASize);
  if (hidden <= 0 || hidden % 16 || hidden > 200 * 1024) return fail(MSC_ERR_BAD_ARG, "hidden=%d must be a positive multiple of 16, two rows of which fit in shared memory", hidden);
  if (topk > kFp8MaxTopk) return fail(MSC_ERR_UNSUPPORTED, "topk=%d exceeds %d", topk, kFp8MaxTopk);
  if (reinterpret_cast<uintptr_t>(tokens_bf16) % 16 || reinterpret_cast<uintptr_t>(a_q) % 16)
    return fail(MSC_ERR_BAD_ARG, "tokens and a_q must be 16-byte aligned");
  for (const void* ptr : {static_cast<const void*>(ids), static_cast<const void*>(weights), static_cast<const void*>(rank),
                          static_cast<const void*>(group_offsets), static_cast<const void*>(a_sf), static_cast<const void*>(row_weight),
                          static_cast<const void*>(row_token)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4) return fail(MSC_ERR_BAD_ARG, "a pointer is not 4-byte aligned");
  Fp8DispatchParams p;
  p.tokens = static_cast<const __nv_bfloat16*>(tokens_bf16);
  p.ids = ids; p.weights = weights; p.rank = rank; p.group_offsets = group_offsets;
  p.q = static_cast<uint8_t*>(a_q); p.sf = a_sf; p.row_weight = row_weight; p.row_token = row_token;
  p.hidden = hidden; p.kblocks = (hidden + 127) / 128; p.topk = topk;
  p.expert_first = expert_first; p.experts_local = experts_local; p.rows_cap = rows_cap; p.pitch = (rows_cap + 3) & ~3;
  const int smem = 2 * ((hidden + 4 * p.kblocks + 15) & ~15);
  if (smem > 200 * 1024) return fail(MSC_ERR_UNSUPPORTED, "hidden=%d: two rows do not fit in shared memory", hidden);
  if (tokens == 0) return MSC_OK;
  p.status = status_word();
  if (!p.status) return fail(MSC_ERR_CUDA, "status word unavailable on this device");
  if (smem + (int)sizeof(int) * 2 * kFp8MaxTopk > 48 * 1024)   // (with its static arrays)
    if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(moe_permute_quantize_fp8_kernel), 200 * 1024)) return rc;
  const int sms = num_sms();
  if (sms <= 0) return fail(MSC_ERR_CUDA, "could not query the SM count");
  // enough CTAs to fill every SM, each walking its share of the tokens; wide CTAs for a few tokens, whose rows
  // are then one step long
  const int grid = std::min(tokens, 16 * sms), threads = tokens <= 2 * sms ? 512 : 128;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config(grid, threads, smem, static_cast<cudaStream_t>(stream), attr);
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, moe_permute_quantize_fp8_kernel, p, tokens));
  return MSC_OK;
}

int msc_fp8_block_quantize_weight(const void* w, int w_dtype, void* q, float* sf, int l, int n, int k, void* stream) {
  using namespace msc;
  if (!w || !q || !sf) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (l <= 0 || n <= 0 || k <= 0) return fail(MSC_ERR_BAD_ARG, "sizes must be positive");
  if (k % 16) return fail(MSC_ERR_BAD_ARG, "k=%d must be a multiple of 16", k);
  if (n > kMostOfASize || k > kMostOfASize) return fail(MSC_ERR_UNSUPPORTED, "n=%d or k=%d exceeds %d", n, k, kMostOfASize);
  if (w_dtype < 0 || w_dtype > 2) return fail(MSC_ERR_UNSUPPORTED, "w_dtype must be 0 (bf16), 1 (f32) or 2 (f16), got %d", w_dtype);
  if (reinterpret_cast<uintptr_t>(w) % 16 || reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(sf) % 4)
    return fail(MSC_ERR_BAD_ARG, "w and q must be 16-byte aligned, sf 4-byte aligned");
  WeightBlockParams p;
  p.w = w; p.q = static_cast<uint8_t*>(q); p.sf = sf;
  p.n = n; p.k = k; p.nblocks = (n + 127) / 128; p.kblocks = (k + 127) / 128;
  if (l > 65535 || p.nblocks > 65535) return fail(MSC_ERR_UNSUPPORTED, "l=%d or n=%d is too large for one launch", l, n);
  const dim3 grid((unsigned)p.kblocks, (unsigned)p.nblocks, (unsigned)l);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (w_dtype == 0) quantize_fp8_weight_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  else if (w_dtype == 1) quantize_fp8_weight_kernel<float><<<grid, 256, 0, st>>>(p);
  else quantize_fp8_weight_kernel<__half><<<grid, 256, 0, st>>>(p);
  MSC_CUDA_OK(cudaGetLastError());
  return MSC_OK;
}

}  // extern "C"
