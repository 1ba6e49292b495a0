// Routing of tokens to experts from router logits, and its gradient (latency- and issue-bound: a
// token is 1 KB of logits for 256 experts).
//
//   score_j = e^(x_j - max) / sum e^(x - max)   or   1 / (1 + e^(-x_j))
//   key_j   = score_j + bias_j                  the bias takes part in the choice only
//   a group's key is the sum of its best `group_top` keys; the best `topk_groups` groups take part
//   ids     = the best `topk` keys among them, in falling order, ties to the lower expert
//   w_i     = scale * score_i [ / sum of the chosen scores ]
//
// What a choice has to be.  The order of the keys is that of 64-bit arithmetic.  Without a bias and with
// groups judged by their best expert the order of the keys is the order of the logits, and nothing is
// rounded.  Otherwise the keys are computed in fp32, whose error is bounded (key_tolerance below); a
// token in which two keys that the result tells apart lie closer than that is chosen over again in 64
// bits (about one token in a thousand for 256 experts).
//
// Layout: a warp per token, the experts of a group spread over the lanes, 32 to a register slot, so that
// a group's maximum is one warp reduction (redux.sync) per slot; groups of fewer than 32 experts leave
// lanes idle.  A thread-wide maximum over the slots, one reduction and one minimum over the experts that
// hold it make a choice; 256 experts, top 8 of 4 of 8 groups take about 700 instructions per token.
//
// A logit of -inf or NaN, or a bias of -inf or NaN, bars its expert.  Where fewer than topk experts are
// left, the lowest barred ones fill up the ids (they stay distinct and in range) with weight 0.
#include "host_common.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace msc {

struct RouteParams {
  const void* logits;    // (tokens, experts)
  const float* bias;     // (experts) or null
  int* ids;              // (tokens, topk)
  float* weights;        // (tokens, topk)
  int tokens, experts, topk;
  int groups, topk_groups, group_top;   // groups = 1: no restriction
  int per, slots;        // experts and register slots of a group
  int base[32];          // lane 0's expert of every slot
  int renormalize;
  int by_score;          // keys are scores (+ bias), else logits
  float scale;
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// A NaN logit counts as -inf.
template <class T>
__device__ __forceinline__ float load_logit(const T* ptr) {
  const float v = as_float(ld_ordered(ptr));
  return v == v ? v : -INFINITY;
}

// Maximum over the warp; no operand is NaN.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// In the order of their bits (negative ones turned round), high words first: two reductions instead of five
// rounds of shuffles.  (-0 comes out below +0, which no comparison tells apart.)
__device__ __forceinline__ double warp_max(double v) {
  const long long bits = __double_as_longlong(v);
  const unsigned long long o = (unsigned long long)bits ^ ((unsigned long long)(bits >> 63) | 0x8000000000000000ull);
  const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(o >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(o >> 32) == hi ? (unsigned)o : 0u);
  const unsigned long long m = (unsigned long long)hi << 32 | lo;
  return __longlong_as_double((long long)(m ^ ((m >> 63) ? 0x8000000000000000ull : 0xffffffffffffffffull)));
}
// Every lane gets the same bits: the order of the additions is fixed.
template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// e^x to a relative 2^-22 + |x| 2^-24 (what feeds keys and sums; the weights take expf).
__device__ __forceinline__ float exp_fast(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(x, 1.4426950408889634f)));
  return e;
}

// e^(x - mx) where mx is the largest x: an infinite maximum leaves only the logits that equal it.
__device__ __forceinline__ float exp_below(float x, float mx) { return x == mx ? (x == -INFINITY ? 0.0f : 1.0f) : exp_fast(x - mx); }
__device__ __forceinline__ double exp_below(double x, double mx) { return x == mx ? (x == -INFINITY ? 0.0 : 1.0) : exp(x - mx); }
__device__ __forceinline__ float rcp_fast(float x) {   // one ulp
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp_fast(1.0f + exp_fast(-x)); }
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// What lane `k` is handed by the choice of the k-th expert.
struct Pick {
  int id = 0;
  bool barred = true;
};

// The groups that take part, a bit each.  `near`: whether the last that does and the first that does not are
// closer than `tol` (infinite differences of equal infinities come out NaN and count as near).
template <int PER, class F>
__device__ __forceinline__ uint32_t choose_groups(const RouteParams& p, const F (&key)[PER], F tol, int lane, bool& near) {
  const F kNone = -INFINITY;
  F strength = kNone;              // of group `lane`
  auto judge = [&](int g, F best, F second) {   // from every lane's best two keys of group g
    F sum = warp_max(best);
    if (p.group_top == 2) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, best == sum)) - 1;
      const F next = warp_max(lane == owner ? second : best);
      sum = (sum == kNone || next == kNone) ? kNone : sum + next;
    }
    if (lane == g) strength = sum;
  };
  if (p.slots == 1) {              // warp-uniform, as all of this
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < p.groups) judge(i, key[i], kNone);
  } else {
    F best = kNone, second = kNone;
    int j = 0, g = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (key[i] > best) {
        second = best;
        best = key[i];
      } else if (key[i] > second) {
        second = key[i];
      }
      if (++j == p.slots) {
        if (g < p.groups) judge(g, best, second);
        best = second = kNone;
        j = 0;
        ++g;
      }
    }
  }
  int ahead = 0;
  for (int o = 0; o < p.groups; ++o) {
    const F other = __shfl_sync(0xffffffffu, strength, o);
    ahead += (other > strength || (other == strength && o < lane)) ? 1 : 0;
  }
  const bool kept = lane < p.groups && ahead < p.topk_groups;
  const F weakest = -warp_max(kept ? -strength : kNone);
  const F left = warp_max(lane < p.groups && !kept ? strength : kNone);
  near = left != kNone && !(weakest - left > tol * (F)p.group_top);
  return __ballot_sync(0xffffffffu, kept);
}

template <int PER, class F>
__device__ __forceinline__ void bar_groups(const RouteParams& p, F (&key)[PER], uint32_t in) {
  int j = 0, g = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (!((in >> g) & 1u)) key[i] = -INFINITY;
    if (++j == p.slots) {
      j = 0;
      g = min(g + 1, 31);
    }
  }
}

// Chooses from key[slot] of every lane, whatever the keys.  `open`: bit per slot that holds an expert;
// base[slot]: its lane 0's expert.
template <int PER, class F>
__device__ __forceinline__ void choose_any(const RouteParams& p, F (&key)[PER], uint32_t open, const int* base, int lane, Pick& pick) {
  if (p.groups > 1) {
    bool near;
    bar_groups(p, key, choose_groups<PER, F>(p, key, (F)0, lane, near));
  }
  for (int k = 0; k < p.topk; ++k) {
    F m = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) m = key[i] > m ? key[i] : m;
    m = warp_max(m);
    int slot = -1;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == m && ((open >> i) & 1u)) slot = i;
    const int mine = slot < 0 ? 0x7fffffff : base[slot] + lane;
    const int won = __reduce_min_sync(0xffffffffu, mine);
    if (mine == won) {
      open &= ~(1u << slot);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i == slot) key[i] = -INFINITY;
    }
    if (lane == k) {
      pick.id = won;
      pick.barred = m == (F)-INFINITY;
    }
  }
}

// The same at a quarter of the instructions, for the usual case.  Every lane keeps its two best keys at hand and looks
// through its slots again only when both are gone (a lane that holds three of the best).  Returns false where
// the choice has to be made over again: two keys that it tells apart are closer than `tol` (CHECK), or
// fewer than topk experts are left.
template <int PER, bool CHECK>
__device__ __forceinline__ bool choose(const RouteParams& p, float (&key)[PER], float tol, const int* base, int lane, Pick& pick) {
  const float kNone = -INFINITY;
  if (p.groups > 1) {
    bool near;
    const uint32_t in = choose_groups<PER, float>(p, key, tol, lane, near);
    if (CHECK && near) return false;
    bar_groups(p, key, in);
  }
  float best, second;
  int best_at, second_at, best_id, second_id;
  uint32_t taken = 0;              // slots
  auto look = [&] {
    best = second = kNone;
    best_at = second_at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float v = (taken >> i) & 1u ? kNone : key[i];
      if (v > second) {
        const bool top = v > best;
        second = top ? best : v;
        second_at = top ? best_at : i;
        best = top ? v : best;
        best_at = top ? i : best_at;
      }
    }
    best_id = base[best_at] + lane;
    second_id = base[second_at] + lane;
  };
  look();
  bool fine = true;
  float before = INFINITY;
  for (int k = 0; k < p.topk; ++k) {
    const float m = warp_max(best);
    fine = fine && m != kNone;
    if (CHECK) {
      fine = fine && (k == 0 || before - m > tol);
      before = m;
    }
    const int mine = best == m ? best_id : 0x7fffffff;
    const int won = __reduce_min_sync(0xffffffffu, mine);
    if (mine == won) {
      taken |= 1u << best_at;
      best = second;
      best_at = second_at;
      best_id = second_id;
      second = kNone;
      if (best == kNone) look();
    }
    if (lane == k) pick.id = won;
  }
  if (CHECK) {                     // the best that is left
    const float m = warp_max(best);
    fine = fine && (m == kNone || before - m > tol);
  }
  pick.barred = false;
  return fine;
}

// The choice of a token in 64 bits.
template <int PER, bool SIGMOID, class T>
__device__ __noinline__ Pick choose_in_64_bits(const RouteParams& p, const T* row, uint32_t open, const int* base, int lane) {
  double key[PER];
  double mx = -INFINITY, sum = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = ((open >> i) & 1u) ? (double)load_logit(row + base[i] + lane) : -INFINITY;
    mx = fmax(mx, key[i]);
  }
  if (p.by_score) {
    if (!SIGMOID) {
      mx = warp_max(mx);
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += exp_below(key[i], mx);
      sum = warp_sum(sum);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double x = key[i];
      const double b = (p.bias && ((open >> i) & 1u)) ? (double)ld_ordered(p.bias + base[i] + lane) : 0.0;
      const double s = SIGMOID ? sigmoid(x) : sum > 0.0 ? exp_below(x, mx) / sum : 0.0;
      key[i] = (x == -INFINITY || b != b) ? -INFINITY : s + b;
    }
  }
  Pick pick;
  choose_any<PER, double>(p, key, open, base, lane, pick);
  return pick;
}

template <int PER, bool SIGMOID, class T>
__global__ void __launch_bounds__(128) moe_route_kernel(const RouteParams p) {
  __shared__ int base[32];
  if (threadIdx.x < 32) base[threadIdx.x] = p.base[threadIdx.x];
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long token = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.experts;

  float key[PER], b[PER];
  uint32_t open = 0;
  {
    int j = 0, g = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (g < p.groups && j * 32 + lane < p.per) open |= 1u << i;
      key[i] = ((open >> i) & 1u) ? load_logit(row + base[i] + lane) : -INFINITY;
      b[i] = (p.bias && ((open >> i) & 1u)) ? ld_ordered(p.bias + base[i] + lane) : 0.0f;
      if (++j == p.slots) {
        j = 0;
        ++g;
      }
    }
  }
  float mx = -INFINITY, sum = 0.0f;
  if (!SIGMOID && (p.by_score || !p.renormalize)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) mx = fmaxf(mx, key[i]);
    mx = warp_max(mx);
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += exp_below(key[i], mx);
    sum = warp_sum(sum);
  }
  Pick pick;
  bool fine;
  if (p.by_score) {
    const float inv = sum > 0.0f ? __fdividef(1.0f, sum) : 0.0f;
    float largest = 0.0f;   // magnitude of a key
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float x = key[i];
      const float s = SIGMOID ? sigmoid(x) : exp_below(x, mx) * inv;
      const float v = s + b[i];
      key[i] = (x == -INFINITY || v != v) ? -INFINITY : v;   // (a NaN is the bias')
      largest = fmaxf(largest, key[i] == -INFINITY ? 0.0f : fabsf(key[i]));
    }
    // What a key may be off by, twice.  Sigmoid: s (1 - s) (|x| 2^-24 + 2^-22) from the exponential, at
    // most 1.4e-7, the sum and the quotient 3 x 2^-24 s.  Softmax: 2^-22 + |x - max| 2^-24 of p from its
    // exponential (p |x - max| is at most 1/e of the largest p, which is `inv`), as much and up to 37
    // additions' 2^-24 from the sum, and the quotient: 51 x 2^-24.  Then the rounding of the key itself.
    const float tol = (SIGMOID ? 0x1p-20f : 0x1p-17f * inv) + 0x1p-22f * warp_max(largest);
    fine = choose<PER, true>(p, key, tol, base, lane, pick);
  } else {
    fine = choose<PER, false>(p, key, 0.0f, base, lane, pick);
  }
  if (!fine) pick = choose_in_64_bits<PER, SIGMOID, T>(p, row, open, base, lane);

  // the weights, lane k that of the k-th choice, from the logits again
  const bool there = lane < p.topk && !pick.barred;
  const float x = there ? load_logit(row + pick.id) : -INFINITY;
  float w;
  if (SIGMOID) {
    const float e = expf(-fabsf(x));
    w = x >= 0.0f ? __fdiv_rn(1.0f, 1.0f + e) : __fdiv_rn(e, 1.0f + e);
  } else {
    const float ref = p.renormalize ? warp_max(x) : mx;   // a common factor of the chosen ones cancels
    w = x == ref ? (x == -INFINITY ? 0.0f : 1.0f) : expf(x - ref);
    if (!p.renormalize) w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
  }
  if (!there) w = 0.0f;
  if (p.renormalize) {
    const float all = warp_sum(w);
    w = all > 0.0f ? __fdiv_rn(w, all) : 0.0f;
  }
  if (lane < p.topk) {
    p.ids[token * p.topk + lane] = pick.id;
    p.weights[token * p.topk + lane] = w * p.scale;
  }
}

// ---- gradient ------------------------------------------------------------------------------
// With w the forward's weights and g the gradient of them, A = sum g_i w_i over a token's choices:
//   softmax, renormalised   dx_i = w_i (g_i - A / scale)                     (chosen experts only)
//   softmax                 dx_j = [j chosen] w_j g_j - p_j A                (every expert)
//   sigmoid, renormalised   dx_i = w_i (1 - score_i) (g_i - A / scale)
//   sigmoid                 dx_i = w_i (1 - score_i) g_i
// A barred expert has weight 0, and so gradient 0.  A token's row is put together in shared memory and
// written in one pass; an id that occurs twice collects both shares, in the order of the choices.
struct RouteBackwardParams {
  const void* logits;         // (tokens, experts)
  const int* ids;             // (tokens, topk)
  const float* weights;       // (tokens, topk)
  const float* grad_weights;  // (tokens, topk)
  void* grad_logits;          // (tokens, experts)
  int tokens, experts, topk, renormalize;
  float inv_scale;
};

constexpr int kBackwardWarps = 4;

template <bool SIGMOID, class T>
__global__ void __launch_bounds__(32 * kBackwardWarps) moe_route_backward_kernel(const RouteBackwardParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  extern __shared__ float rows[];   // [warp][experts]
  const int lane = threadIdx.x & 31;
  const long long token = (long long)blockIdx.x * kBackwardWarps + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.experts;
  T* out = static_cast<T*>(p.grad_logits) + token * p.experts;
  float* mine = rows + (threadIdx.x >> 5) * p.experts;

  int id = -1 - lane;   // (lanes without a choice match nobody)
  float w = 0.0f, g = 0.0f;
  if (lane < p.topk) {
    const int e = ld_ordered(p.ids + token * p.topk + lane);
    if (e >= 0 && e < p.experts) {
      id = e;
      w = ld_ordered(p.weights + token * p.topk + lane);
      g = ld_ordered(p.grad_weights + token * p.topk + lane);
    }
  }
  if (w == 0.0f) g = 0.0f;   // an infinite gradient of a weight that does not move
  const float all = warp_sum(g * w);
  float c = w * (p.renormalize ? g - all * p.inv_scale : g);
  if (SIGMOID && id >= 0) c *= __fdiv_rn(1.0f, 1.0f + expf(load_logit(row + id)));

  if (!SIGMOID && !p.renormalize) {
    float mx = -INFINITY, sum = 0.0f;
    for (int e = lane; e < p.experts; e += 32) {
      mine[e] = load_logit(row + e);
      mx = fmaxf(mx, mine[e]);
    }
    mx = warp_max(mx);
    for (int e = lane; e < p.experts; e += 32) {
      mine[e] = exp_below(mine[e], mx);
      sum += mine[e];
    }
    sum = warp_sum(sum);
    const float f = sum > 0.0f ? -__fdiv_rn(all, sum) : 0.0f;
    for (int e = lane; e < p.experts; e += 32) mine[e] *= f;
  } else {
    for (int e = lane; e < p.experts; e += 32) mine[e] = 0.0f;
  }
  __syncwarp();
  const unsigned same = __match_any_sync(0xffffffffu, id);
  float total = 0.0f;
  for (int k = 0; k < p.topk; ++k) {
    const float ck = __shfl_sync(0xffffffffu, c, k);
    if ((same >> k) & 1u) total += ck;
  }
  if (id >= 0 && lane == __ffs(same) - 1) mine[id] += total;
  __syncwarp();
  for (int e = lane; e < p.experts; e += 32) out[e] = from_float<T>(mine[e]);
}

template <bool SIGMOID, class T>
static int launch_route(const RouteParams& p, cudaStream_t stream) {
  const int used = p.groups * p.slots;
  auto kern = used <= 2 ? moe_route_kernel<2, SIGMOID, T>
              : used <= 4 ? moe_route_kernel<4, SIGMOID, T>
              : used <= 8 ? moe_route_kernel<8, SIGMOID, T>
              : used <= 16 ? moe_route_kernel<16, SIGMOID, T> : moe_route_kernel<32, SIGMOID, T>;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config((p.tokens - 1) / 4 + 1, 128, 0, stream, attr);
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, kern, p));
  return MSC_OK;
}

template <bool SIGMOID, class T>
static int launch_route_backward(const RouteBackwardParams& p, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config((p.tokens - 1) / kBackwardWarps + 1, 32 * kBackwardWarps,
                                            kBackwardWarps * p.experts * (int)sizeof(float), stream, attr);
  auto kern = moe_route_backward_kernel<SIGMOID, T>;
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, kern, p));
  return MSC_OK;
}

template <class T>
static bool misaligned(const T* ptr, int bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes != 0; }

static int check_route(const void* logits, int dtype, int tokens, int experts, int topk, int score, float scale) {
  if (dtype < 0 || dtype > 2) return fail(MSC_ERR_UNSUPPORTED, "dtype must be 0 (bf16), 1 (f32) or 2 (f16), got %d", dtype);
  if (tokens < 0) return fail(MSC_ERR_BAD_ARG, "tokens=%d must not be negative", tokens);
  if (experts < 1 || experts > 1024) return fail(MSC_ERR_UNSUPPORTED, "experts=%d must be in [1, 1024]", experts);
  if (topk < 1 || topk > 32 || topk > experts) return fail(MSC_ERR_UNSUPPORTED, "topk=%d must be in [1, min(32, experts)]", topk);
  if (score != MSC_SCORE_SOFTMAX && score != MSC_SCORE_SIGMOID)
    return fail(MSC_ERR_UNSUPPORTED, "score must be MSC_SCORE_SOFTMAX or MSC_SCORE_SIGMOID, got %d", score);
  if (!(scale > 0.0f) || scale > 3.0e38f) return fail(MSC_ERR_BAD_ARG, "scale must be positive and finite");
  if (misaligned(logits, dtype == 1 ? 4 : 2)) return fail(MSC_ERR_BAD_ARG, "logits are not aligned to their type");
  return MSC_OK;
}

}  // namespace msc

extern "C" {

int msc_moe_route(const void* logits, int dtype, const float* bias, int32_t* ids, float* weights, int tokens,
                  int experts, int topk, const msc_route_cfg* cfg, void* stream) {
  using namespace msc;
  if (!logits || !ids || !weights || !cfg) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (int rc = check_route(logits, dtype, tokens, experts, topk, cfg->score, cfg->scale)) return rc;
  if (misaligned(bias, 4) || misaligned(ids, 4) || misaligned(weights, 4))
    return fail(MSC_ERR_BAD_ARG, "bias, ids and weights must be 4-byte aligned");
  const int groups = cfg->groups, chosen = cfg->topk_groups;
  if (groups < 1 || groups > 32 || experts % groups)
    return fail(MSC_ERR_UNSUPPORTED, "groups=%d must be in [1, 32] and divide experts=%d", groups, experts);
  if (chosen < 1 || chosen > groups) return fail(MSC_ERR_BAD_ARG, "topk_groups=%d must be in [1, groups=%d]", chosen, groups);
  const int per = experts / groups;
  if (cfg->group_top < 1 || cfg->group_top > 2 || cfg->group_top > per)
    return fail(MSC_ERR_UNSUPPORTED, "group_top=%d must be 1 or 2 and at most the %d experts of a group", cfg->group_top, per);
  if (topk > chosen * per)
    return fail(MSC_ERR_BAD_ARG, "topk=%d exceeds the %d experts of %d groups", topk, chosen * per, chosen);
  RouteParams p;
  p.logits = logits; p.bias = bias; p.ids = ids; p.weights = weights;
  p.tokens = tokens; p.experts = experts; p.topk = topk;
  const bool limited = chosen < groups;          // all groups taking part is no restriction
  p.groups = limited ? groups : 1;
  p.topk_groups = limited ? chosen : 1;
  p.group_top = cfg->group_top;
  p.per = experts / p.groups;
  p.slots = (p.per + 31) / 32;
  if (p.groups * p.slots > 32)
    return fail(MSC_ERR_UNSUPPORTED, "%d groups of %d experts: groups x (experts of a group / 32, rounded up) must be at most 32",
                groups, per);
  for (int i = 0; i < 32; ++i) p.base[i] = i / p.slots * p.per + i % p.slots * 32;
  p.renormalize = cfg->renormalize != 0;
  p.by_score = bias != nullptr || (limited && cfg->group_top == 2);
  p.scale = cfg->scale;
  if (tokens == 0) return MSC_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cfg->score == MSC_SCORE_SIGMOID)
    return dtype == 0 ? launch_route<true, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route<true, float>(p, st)
                                                                             : launch_route<true, __half>(p, st);
  return dtype == 0 ? launch_route<false, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route<false, float>(p, st)
                                                                            : launch_route<false, __half>(p, st);
}

int msc_moe_route_backward(const float* grad_weights, const void* logits, int dtype, const int32_t* ids,
                           const float* weights, void* grad_logits, int tokens, int experts, int topk, int score,
                           int renormalize, float scale, void* stream) {
  using namespace msc;
  if (!grad_weights || !logits || !ids || !weights || !grad_logits) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (int rc = check_route(logits, dtype, tokens, experts, topk, score, scale)) return rc;
  if (misaligned(grad_logits, dtype == 1 ? 4 : 2) || misaligned(ids, 4) || misaligned(weights, 4) || misaligned(grad_weights, 4))
    return fail(MSC_ERR_BAD_ARG, "a pointer is not aligned to its type");
  RouteBackwardParams p;
  p.logits = logits; p.ids = ids; p.weights = weights; p.grad_weights = grad_weights; p.grad_logits = grad_logits;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.renormalize = renormalize != 0;
  p.inv_scale = 1.0f / scale;
  if (tokens == 0) return MSC_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (score == MSC_SCORE_SIGMOID)
    return dtype == 0 ? launch_route_backward<true, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route_backward<true, float>(p, st)
                                                                                      : launch_route_backward<true, __half>(p, st);
  return dtype == 0 ? launch_route_backward<false, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route_backward<false, float>(p, st)
                                                                                     : launch_route_backward<false, __half>(p, st);
}

}  // extern "C"
