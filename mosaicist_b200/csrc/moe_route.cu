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
// rounded.  Otherwise the keys are computed in fp32, whose error is bounded (`tol` below); a token in which two
// keys that the result tells apart lie closer than that is looked at again in 64 bits (about one token in a
// thousand for 256 experts).
//
// Two layouts.  A warp per token, the experts of a group spread over the lanes, 32 to a register slot: a group's
// maximum is one warp reduction (redux.sync) per slot, and a thread-wide maximum over the slots, one reduction and
// one minimum over the experts that hold it make a choice.  That is the shortest way for a few tokens and serves up
// to 1024 experts, but 256 experts, top 8 of 4 of 8 groups take about 1330 instructions per token (533 by eight lanes), most of
// them the serial rounds of choosing.  From 1024 tokens on, and up to 256 experts, eight lanes per token share
// these rounds among four tokens (below).
//
// Neither is bound by memory: 8192 tokens of 256 fp32 logits are 8.9 MB, 1.4 us, and take 12 to 16 us with sigmoid, bias and
// 4 of 8 groups, by how many tokens lie close (21 a warp per token), 4.7 us for 128 bf16 experts without them; a warp
// per token takes 25 us for 8192 x 384 (top 8, sigmoid and bias), 20 for 8192 x 512 (top 10, softmax), 38 for 8192 x 256
// in 16 groups. 16 tokens take 2.3 to 4 us in a graph, 5.6 launched one by one.  What is left
// is the chain of one warp's steps (3 to 4 us) and, where keys lie close, the tokens that are looked at in 64 bits.
//
// A logit of -inf or NaN, or a bias of -inf or NaN, bars its expert.  Where fewer than topk experts are
// left, the lowest barred ones fill up the ids (they stay distinct and in range) with weight 0.
#include "host_common.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

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
  int sigmoid;           // else softmax
  int by_score;          // keys are scores (+ bias), else logits
  float scale;
  // eight lanes a token
  int lanes, chunk;      // lanes of a group, experts of a lane (the last lane of a group may have fewer)
  int per_inv, chunk_inv;   // ceil(2^16 / .): exact quotients of numbers below 256 by a multiplication
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

__device__ __forceinline__ float sigmoid_weight(float x) {
  const float e = expf(-fabsf(x));
  return x >= 0.0f ? __fdiv_rn(1.0f, 1.0f + e) : __fdiv_rn(e, 1.0f + e);
}
__device__ __forceinline__ float softmax_weight(float x, float ref) {
  return x == ref ? (x == -INFINITY ? 0.0f : 1.0f) : expf(x - ref);
}

// Sigmoids of small logits, e^x each to a relative e^-16 (two roundings), lose bits in fp32 below e^-87 and vanish below
// e^-104, where their share of the sum need not: their ratios are e^(x - best).  Above, what fp32 loses is less than
// 2^-126 of the sum.  In 64 bits they vanish too below -709.
__device__ __forceinline__ bool vanishing(float best) { return best < -16.0f && best >= -709.7827f; }

// A bit per slot in which this lane has an expert.
template <int PER>
__device__ __forceinline__ uint32_t open_slots(const RouteParams& p, int lane) {
  uint32_t open = 0;
  int j = 0, g = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (g < p.groups && j * 32 + lane < p.per) open |= 1u << i;
    if (++j == p.slots) {
      j = 0;
      ++g;
    }
  }
  return open;
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
  const uint32_t open = open_slots<PER>(p, lane);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = ((open >> i) & 1u) ? load_logit(row + base[i] + lane) : -INFINITY;
    b[i] = (p.bias && ((open >> i) & 1u)) ? ld_ordered(p.bias + base[i] + lane) : 0.0f;
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
    w = sigmoid_weight(x);
    if (p.renormalize) {
      const float best = warp_max(x);
      if (vanishing(best)) w = softmax_weight(x, best);
    }
  } else {
    w = softmax_weight(x, p.renormalize ? warp_max(x) : mx);   // a common factor of the chosen ones cancels
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

// ---- eight lanes a token ---------------------------------------------------------------------
// Up to 256 experts in 1, 2, 4 or 8 groups, topk <= 8: a warp takes four tokens, eight lanes each, and a lane
// up to 32 experts of one group.  A key is an unsigned word in the order of the keys, its lowest 8 bits
// 255 - expert, so that words are distinct and ties fall to the lower expert.  Lanes sort theirs in eights by
// networks, and three exchanges merge the best eight of the lanes; nothing branches.
//   Logits: the upper 24 bits of the fp32 number (all that a 16-bit logit has).
//   Scores: 23 bits of fixed point over [largest bias - 8, largest score + largest bias], or less where the
//   biases span less; a key below counts as the window's lower end.
// From this many tokens on.  A warp of four tokens takes longer than a warp of one (E = experts, us at 16 / 1024 /
// 2048 / 8192 tokens, eight lanes against a warp a token): E = 61 2.6 / 3.2 / 3.3 / 4.9 against 1.9 / 3.1 / 3.9 / 9.6;
// E = 128 2.4 / 2.7 / 2.8 / 4.8 against 2.3 / 3.2 / 4.1 / 11.3; E = 160 in groups 3.7 / 4.0 / 4.2 / 7.0 against
// 3.1 / 4.1 / 5.2 / 13.7.
constexpr int kOctetTokens = 1024;
constexpr int kOctetWarps = 2;
constexpr float kWindow = 8.0f, kUnits = 0x1p23f - 32.0f;

enum { kByLogit = 0, kBySoftmax = 1, kBySigmoid = 2 };   // what the keys are

template <int KEYS>
struct Word {
  // words below it are those of -inf: barred
  static constexpr uint32_t kLeast = KEYS == kByLogit ? 0x00800000u : 1u << 9;
  // `v`: a logit, or a place in the window, 2^23 + 1 .. 2^24 - 1 where it is not below it
  static __device__ __forceinline__ uint32_t of(float v, uint32_t low) {
    if (KEYS == kByLogit) {
      const uint32_t bits = __float_as_uint(v);
      return ((bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u)) & ~255u) | (low & 255u);
    }
    return v == -INFINITY ? 0u : (__float_as_uint(fmaxf(v, 0x1p23f + 1.0f)) << 9) | (low & 255u);
  }
  // The logit or at most 2^-15 of it less; the place less 2^24.
  static __device__ __forceinline__ float value(uint32_t word) {
    const uint32_t o = word & ~255u;
    if (word < kLeast) return -INFINITY;
    return KEYS == kByLogit ? __uint_as_float(o ^ ((int)o < 0 ? 0x80000000u : 0xffffffffu)) : __uint_as_float((o >> 9) | 0x4b000000u) - 0x1p24f;
  }
  static __device__ __forceinline__ bool below_window(uint32_t word) { return KEYS != kByLogit && word < 2u << 9; }
};
__device__ __forceinline__ void order(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
__device__ __forceinline__ void sort8(uint32_t* v) {   // falling (Batcher's odd-even merging)
  order(v[0], v[1]); order(v[2], v[3]); order(v[4], v[5]); order(v[6], v[7]);
  order(v[0], v[2]); order(v[1], v[3]); order(v[4], v[6]); order(v[5], v[7]);
  order(v[1], v[2]); order(v[5], v[6]);
  order(v[0], v[4]); order(v[1], v[5]); order(v[2], v[6]); order(v[3], v[7]);
  order(v[2], v[4]); order(v[3], v[5]);
  order(v[1], v[2]); order(v[3], v[4]); order(v[5], v[6]);
}
// v: the best eight of two falling lists; `left`: the best word that was dropped.
template <bool CHECK>
__device__ __forceinline__ void merge8(uint32_t* v, const uint32_t* with, uint32_t& left) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (CHECK) left = max(left, min(v[i], with[7 - i]));
    v[i] = max(v[i], with[7 - i]);
  }
#pragma unroll
  for (int d = 4; d; d >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & d)) order(v[i], v[i + d]);
}
template <class F>
__device__ __forceinline__ F octet_sum(F v) {
#pragma unroll
  for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float octet_max(float v) {
#pragma unroll
  for (int o = 4; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int PER, int KEYS, class T>
__global__ void __launch_bounds__(32 * kOctetWarps) moe_route_octets_kernel(const RouteParams p) {
  constexpr int kPitch = PER + 1, kTokenPitch = 8 * kPitch;   // the 32 lanes' k-th words lie in 32 banks
  constexpr bool kCheck = KEYS != kByLogit || sizeof(T) == 4;   // a 16-bit logit keeps all its bits in a word
  __shared__ float s_rows[kOctetWarps][4 * kTokenPitch];
  __shared__ float s_bias[KEYS == kByLogit ? 1 : kOctetWarps][kTokenPitch];
  __shared__ int s_some[kOctetWarps][32];
  using W = Word<KEYS>;
  __shared__ int base[32];
  base[threadIdx.x & 31] = p.base[threadIdx.x & 31];   // (every warp the same)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & 7, quad = lane >> 3;
  float* s_x = s_rows[warp];
  // where the logit of an expert lies in a token's row
  auto at = [&](int e) {
    const int g = (e * p.per_inv) >> 16, j = e - g * p.per;
    const int h = (j * p.chunk_inv) >> 16;
    return (g * p.lanes + h) * kPitch + (j - h * p.chunk);
  };
  const int group = sub / p.lanes, first = sub - group * p.lanes;        // this lane's
  const int e0 = group * p.per + first * p.chunk;
  const int count = min(max(p.per - first * p.chunk, 0), p.chunk);
  const float* list = s_x + quad * kTokenPitch + sub * kPitch;
  for (int i = count; i < PER; ++i) s_x[quad * kTokenPitch + sub * kPitch + i] = -INFINITY;
  grid_dependency_wait();
  grid_launch_dependents();
  const long long token0 = ((long long)blockIdx.x * kOctetWarps + warp) * 4;
  const T* rows = static_cast<const T*>(p.logits) + token0 * p.experts;
  const int tokens = (int)min(max(p.tokens - token0, 0LL), 4LL);         // of this warp
  for (int c = lane; c < p.experts; c += 128) {
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[i][q] = (c + 32 * i < p.experts && q < tokens) ? load_logit(rows + q * p.experts + c + 32 * i) : -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + 32 * i < p.experts) {
        const int to = at(c + 32 * i);
#pragma unroll
        for (int q = 0; q < 4; ++q) s_x[q * kTokenPitch + to] = v[i][q] + 0.0f;   // (-0 counts as 0)
      }
  }
  float spread = 0.0f;          // the biases' part of the window
  bool hopeless = false;
  if (KEYS != kByLogit) {       // biases less the largest one
    float b[8], most = p.bias ? -INFINITY : 0.0f, least = INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = lane + 32 * i;
      b[i] = e >= p.experts ? -INFINITY : p.bias ? ld_ordered(p.bias + e) : 0.0f;
      if (b[i] > -INFINITY) {   // (a NaN is not)
        most = fmaxf(most, b[i]);
        least = fminf(least, b[i]);
      } else {
        b[i] = -INFINITY;
      }
    }
    most = warp_max(most);
    least = -warp_max(-least);
    hopeless = !(fabsf(most) <= FLT_MAX);
    spread = fminf(most - least, kWindow);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.experts) s_bias[warp][at(lane + 32 * i)] = b[i] > -INFINITY ? fmaxf(b[i] - most, -1e20f) : b[i];
  }
  __syncwarp();
  if (tokens == 0) return;

  const bool softmax = KEYS == kBySoftmax || (KEYS == kByLogit && !p.sigmoid);
  float mx = -INFINITY, sum = 0.0f, inv = 0.0f;
  if (KEYS == kBySoftmax || (KEYS == kByLogit && softmax && !p.renormalize)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) mx = fmaxf(mx, list[i]);
    mx = octet_max(mx);
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += exp_below(list[i], mx);
    sum = octet_sum(sum);
    inv = sum > 0.0f ? __fdividef(1.0f, sum) : 0.0f;
  }
  const float top = KEYS == kBySoftmax && sum > 0.0f ? inv : 1.0f;       // the largest score there can be
  const float unit = __fdividef(kUnits, top + spread), end = 0x1p24f - 16.0f - top * unit;
  uint32_t word[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float x = list[i];
    float v = x;
    if (KEYS != kByLogit) {
      const float s = KEYS == kBySigmoid ? sigmoid(x) : exp_below(x, mx) * inv;
      v = x == -INFINITY ? -INFINITY : fmaf(s + s_bias[warp][sub * kPitch + i], unit, end);
    }
    word[i] = W::of(v, (uint32_t)(255 - e0 - i));
  }
  uint32_t left = 0;
  sort8(word);
#pragma unroll
  for (int b = 8; b < PER; b += 8) {
    sort8(word + b);
    merge8<kCheck>(word, word + b, left);
  }
  // What the difference of two keys may be off by, in units: that of the scores (as above), 2 from rounding
  // the bias' distance and the sum, 1 from the place itself.  Of two logits that differ in their words none is mistaken.
  const float tol = KEYS == kByLogit ? 0.0f : (KEYS == kBySigmoid ? 0x1p-20f : 0x1p-17f * inv) * unit + 4.0f;
  bool near = false, kept = true;      // this lane's group
  if (p.groups > 1) {
    uint32_t a = word[0], b = word[1];
    for (int o = 1; o < p.lanes; o <<= 1) {
      const uint32_t a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
      b = max(min(a, a2), max(b, b2));
      a = max(a, a2);
    }
    const float best = W::value(a), second = p.group_top == 2 ? W::value(b) : 0.0f;
    const float strength = (best == -INFINITY || second == -INFINITY) ? -INFINITY : best + second;
    int ahead = 0;
#pragma unroll
    for (int o = 0; o < 8; ++o) {
      const float other = __shfl_sync(0xffffffffu, strength, o, 8);
      if ((o & (p.lanes - 1)) == 0) ahead += (other > strength || (other == strength && o < sub - first)) ? 1 : 0;
    }
    kept = ahead < p.topk_groups;
    if (kCheck) {
      const float weakest = -octet_max(kept ? -strength : -INFINITY), out = octet_max(kept ? -INFINITY : strength);
      near = out != -INFINITY && !(weakest - out > tol * p.group_top);
      // (of a group that is kept for a key below the window nothing is known)
      const float unknown = octet_max(kept && strength != -INFINITY && W::below_window(p.group_top == 2 ? b : a) ? 1.0f : 0.0f);
      near = near || unknown > 0.0f;
    }
    if (!kept) {
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = 0;
      left = 0;
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    uint32_t with[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) with[i] = __shfl_xor_sync(0xffffffffu, word[i], o);
    if (kCheck) left = max(left, __shfl_xor_sync(0xffffffffu, left, o));
    merge8<kCheck>(word, with, left);
  }
  uint32_t mine = word[0];               // lane k has the k-th choice
#pragma unroll
  for (int i = 1; i < 8; ++i) mine = sub == i ? word[i] : mine;
  bool again = near || hopeless || (sub < p.topk && mine < W::kLeast);
  bool close = false;                    // only choices that are certain to be of the groups chosen
  if (kCheck) {
    const uint32_t following = __shfl_down_sync(0xffffffffu, mine, 1, 8);
    const float a = W::value(mine), b = W::value(sub == 7 ? left : following);
    if (sub < p.topk && b != -INFINITY) close = !(a - b > tol);
    if (KEYS == kBySoftmax) again = again || close;   // its 64-bit score takes every expert
  }
  Pick pick;
  pick.id = 255 - (int)(mine & 255u);
  pick.barred = false;
  uint32_t redo = __ballot_sync(0xffffffffu, again && quad < tokens);
  if (kCheck && KEYS != kBySoftmax) {
    uint32_t part = __ballot_sync(0xffffffffu, close && quad < tokens);
    while (part) {                       // of a token: what comes into question, a lane each, ranked in 64 bits
      const int q = (__ffs(part) - 1) >> 3;
      const uint32_t octet = 0xffu << (8 * q);
      part &= ~octet;
      if (redo & octet) continue;
      const float cut = __shfl_sync(0xffffffffu, W::value(mine), 8 * q + p.topk - 1) - 2.0f * tol;
      const bool in = __shfl_sync(0xffffffffu, (int)kept, 8 * q + sub) != 0;
      int n = 0;
#pragma unroll
      for (int i = 0; i < PER / 4; ++i) {
        const int slot = quad * (PER / 4) + i;
        const float x = s_x[q * kTokenPitch + sub * kPitch + slot];
        float v = x;
        if (KEYS != kByLogit && x != -INFINITY) {
          v = fmaf(sigmoid(x) + s_bias[warp][sub * kPitch + slot], unit, end);
          if (v != -INFINITY) v = fmaxf(v, 0x1p23f + 1.0f) - 0x1p24f;   // (a barred expert's is not lifted into the window)
        }
        const uint32_t who = __ballot_sync(0xffffffffu, in && v >= cut);
        const int place = n + __popc(who & ((1u << lane) - 1u));
        if (in && v >= cut && place < 32) s_some[warp][place] = e0 + slot;
        n += __popc(who);
      }
      __syncwarp();
      if (n < p.topk || n > 32) {
        redo |= octet;
      } else {
        const int e = s_some[warp][min(lane, n - 1)];
        double key = s_x[q * kTokenPitch + at(e)];
        if (KEYS != kByLogit) key = sigmoid(key) + (p.bias ? (double)ld_ordered(p.bias + e) : 0.0);
        int ahead = 0;
        for (int o = 0; o < n; ++o) {
          const double other = __shfl_sync(0xffffffffu, key, o);
          const int oe = __shfl_sync(0xffffffffu, e, o);
          ahead += (other > key || (other == key && oe < e)) ? 1 : 0;
        }
        __syncwarp();
        if (lane < n) s_some[warp][ahead] = e;
        __syncwarp();
        if (quad == q) pick.id = s_some[warp][sub];
      }
      __syncwarp();
    }
  }
  while (redo) {
    const int q = (__ffs(redo) - 1) >> 3;
    const Pick found = choose_in_64_bits<8, KEYS == kBySigmoid, T>(p, rows + q * p.experts, open_slots<8>(p, lane), base, lane);
    const int id = __shfl_sync(0xffffffffu, found.id, sub);
    const bool barred = __shfl_sync(0xffffffffu, (int)found.barred, sub) != 0;
    if (quad == q) {
      pick.id = id;
      pick.barred = barred;
    }
    redo &= ~(0xffu << (8 * q));
  }
  const bool there = sub < p.topk && !pick.barred && quad < tokens;
  const float x = there ? s_x[quad * kTokenPitch + at(pick.id)] : -INFINITY;
  float w;
  if (!softmax) {
    w = sigmoid_weight(x);
    if (p.renormalize) {
      const float best = octet_max(x);
      if (vanishing(best)) w = softmax_weight(x, best);
    }
  } else {
    w = softmax_weight(x, p.renormalize ? octet_max(x) : mx);   // a common factor of the chosen ones cancels
    if (!p.renormalize) w = sum > 0.0f ? __fdiv_rn(w, sum) : 0.0f;
  }
  if (!there) w = 0.0f;
  if (p.renormalize) {
    const float all = octet_sum(w);
    w = all > 0.0f ? __fdiv_rn(w, all) : 0.0f;
  }
  if (sub < p.topk && quad < tokens) {
    const long long to = (token0 + quad) * p.topk + sub;
    p.ids[to] = pick.id;
    p.weights[to] = w * p.scale;
  }
}

// ---- gradient ------------------------------------------------------------------------------
// With w the forward's weights and g the gradient of them, A = sum g_i w_i over a token's choices:
//   softmax, renormalised   dx_i = w_i (g_i - A / scale)                     (chosen experts only)
//   softmax                 dx_j = [j chosen] w_j g_j - p_j A                (every expert)
//   sigmoid, renormalised   dx_i = w_i (1 - score_i) (g_i - A / scale)
//   sigmoid                 dx_i = w_i (1 - score_i) g_i
// A barred expert has weight 0, and so gradient 0.  A warp per token; the row is written whole, then the chosen
// experts' elements over it.  Bound by the chain of a warp's loads, then of its reductions: 16383 tokens x 160 bf16, softmax as
// it is, take 7.6 to 7.8 us (10.5 MB, 1.6 us of traffic) with 31 % of the issue slots and 56 % of the warps in use, a
// warp waiting 9 issues for memory and 5 for shuffles per issue of its own; rows kept in shared memory took 10.1.
// 8192 x 256 fp32, chosen experts only, 4.4 us (5.0).  Eight warps a CTA: the same.
struct RouteBackwardParams {
  const void* logits;         // (tokens, experts)
  const int* ids;             // (tokens, topk)
  const float* weights;       // (tokens, topk)
  const float* grad_weights;  // (tokens, topk)
  void* grad_logits;          // (tokens, experts)
  int tokens, experts, topk, renormalize;
  float scale;
};

constexpr int kBackwardWarps = 4;

// PER > 0: softmax as it is, whose gradient every expert has a part of; the row stays in registers, 32 experts a slot.
// PER = 0: only the chosen experts have one.
template <int PER, bool SIGMOID, class T>
__global__ void __launch_bounds__(32 * kBackwardWarps) moe_route_backward_kernel(const RouteBackwardParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long token = (long long)blockIdx.x * kBackwardWarps + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.experts;
  T* out = static_cast<T*>(p.grad_logits) + token * p.experts;

  float v[PER > 0 ? PER : 1];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < p.experts ? load_logit(row + lane + 32 * i) : -INFINITY;
  int id = -1 - lane;   // (lanes without a choice match nobody)
  float w = 0.0f, g = 0.0f, x = -INFINITY;
  if (lane < p.topk) {
    const int e = ld_ordered(p.ids + token * p.topk + lane);
    if (e >= 0 && e < p.experts) {
      id = e;
      w = ld_ordered(p.weights + token * p.topk + lane);
      g = ld_ordered(p.grad_weights + token * p.topk + lane);
      if (SIGMOID || PER > 0) x = load_logit(row + e);
    }
  }
  if (w == 0.0f) g = 0.0f;   // an infinite gradient of a weight that does not move
  const float all = warp_sum(g * w);
  float c = w * (p.renormalize ? g - __fdiv_rn(all, p.scale) : g);
  if (SIGMOID && id >= 0) c *= __fdiv_rn(1.0f, 1.0f + expf(x));

  // an id that occurs twice collects both shares, in the order of the choices
  const unsigned same = __match_any_sync(0xffffffffu, id);
  float total = 0.0f;
  for (int k = 0; k < p.topk; ++k) {
    const float ck = __shfl_sync(0xffffffffu, c, k);
    if ((same >> k) & 1u) total += ck;
  }
  if (PER > 0) {
    float mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) mx = fmaxf(mx, v[i]);
    mx = warp_max(mx);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = exp_below(v[i], mx);
      sum += v[i];
    }
    sum = warp_sum(sum);
    const float f = sum > 0.0f ? -__fdiv_rn(all, sum) : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < p.experts) out[lane + 32 * i] = from_float<T>(v[i] * f);
    total += exp_below(x, mx) * f;
  } else {
    for (int e = lane; e < p.experts; e += 32) out[e] = from_float<T>(0.0f);
  }
  __syncwarp();              // (the chosen experts' come after what stands there)
  if (id >= 0 && lane == __ffs(same) - 1) out[id] = from_float<T>(total);
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

template <int KEYS, class T>
static int launch_octets(const RouteParams& p, cudaStream_t stream) {
  auto kern = p.chunk <= 8 ? moe_route_octets_kernel<8, KEYS, T>
              : p.chunk <= 16 ? moe_route_octets_kernel<16, KEYS, T>
              : p.chunk <= 24 ? moe_route_octets_kernel<24, KEYS, T> : moe_route_octets_kernel<32, KEYS, T>;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config((p.tokens - 1) / (4 * kOctetWarps) + 1, 32 * kOctetWarps, 0, stream, attr);
  MSC_CUDA_OK(cudaLaunchKernelEx(&lc, kern, p));
  return MSC_OK;
}

template <class T>
static int launch_route_of(RouteParams& p, cudaStream_t stream) {
  // (words have 8 bits for the expert; a lane's groups would not be its own if they were more than lanes)
  const bool eights = p.experts <= 256 && p.topk <= 8 && p.groups <= 8 && (p.groups & (p.groups - 1)) == 0;
  if (eights && p.tokens >= kOctetTokens) {
    p.lanes = 8 / p.groups;
    p.chunk = (p.per + p.lanes - 1) / p.lanes;
    p.per_inv = (0x10000 + p.per - 1) / p.per;
    p.chunk_inv = (0x10000 + p.chunk - 1) / p.chunk;
    return !p.by_score ? launch_octets<kByLogit, T>(p, stream)
           : p.sigmoid ? launch_octets<kBySigmoid, T>(p, stream) : launch_octets<kBySoftmax, T>(p, stream);
  }
  return p.sigmoid ? launch_route<true, T>(p, stream) : launch_route<false, T>(p, stream);
}

template <bool SIGMOID, class T>
static int launch_route_backward(const RouteBackwardParams& p, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t lc = pdl_launch_config((p.tokens - 1) / kBackwardWarps + 1, 32 * kBackwardWarps, 0, stream, attr);
  // (five slots rather than eight: 7.6 us against 7.8 to 7.9 for 72 to 160 experts of 16383 tokens; 8.2 for 192, 10.4 for 384)
  auto kern = SIGMOID || p.renormalize ? moe_route_backward_kernel<0, SIGMOID, T>
              : p.experts <= 64 ? moe_route_backward_kernel<2, false, T>
              : p.experts <= 160 ? moe_route_backward_kernel<5, false, T>
              : p.experts <= 256 ? moe_route_backward_kernel<8, false, T>
              : p.experts <= 512 ? moe_route_backward_kernel<16, false, T> : moe_route_backward_kernel<32, false, T>;
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
  if (!cfg || (tokens != 0 && (!logits || !ids || !weights))) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
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
  p.sigmoid = cfg->score == MSC_SCORE_SIGMOID;
  p.by_score = bias != nullptr || (limited && cfg->group_top == 2);
  p.scale = cfg->scale;
  if (tokens == 0) return MSC_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? launch_route_of<__nv_bfloat16>(p, st) : dtype == 1 ? launch_route_of<float>(p, st) : launch_route_of<__half>(p, st);
}

int msc_moe_route_backward(const float* grad_weights, const void* logits, int dtype, const int32_t* ids,
                           const float* weights, void* grad_logits, int tokens, int experts, int topk, int score,
                           int renormalize, float scale, void* stream) {
  using namespace msc;
  if (tokens != 0 && (!grad_weights || !logits || !ids || !weights || !grad_logits)) return fail(MSC_ERR_BAD_ARG, "NULL pointer");
  if (int rc = check_route(logits, dtype, tokens, experts, topk, score, scale)) return rc;
  if (misaligned(grad_logits, dtype == 1 ? 4 : 2) || misaligned(ids, 4) || misaligned(weights, 4) || misaligned(grad_weights, 4))
    return fail(MSC_ERR_BAD_ARG, "a pointer is not aligned to its type");
  RouteBackwardParams p;
  p.logits = logits; p.ids = ids; p.weights = weights; p.grad_weights = grad_weights; p.grad_logits = grad_logits;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.renormalize = renormalize != 0;
  p.scale = scale;
  if (tokens == 0) return MSC_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (score == MSC_SCORE_SIGMOID)
    return dtype == 0 ? launch_route_backward<true, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route_backward<true, float>(p, st)
                                                                                      : launch_route_backward<true, __half>(p, st);
  return dtype == 0 ? launch_route_backward<false, __nv_bfloat16>(p, st) : dtype == 1 ? launch_route_backward<false, float>(p, st)
                                                                                     : launch_route_backward<false, __half>(p, st);
}

}  // extern "C"
