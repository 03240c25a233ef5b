// Routing of tokens to experts, and its gradient.
//
//   score  s_e = softmax(x)_e or sigmoid(x_e); an expert whose logit is -inf
//          is closed: it has no score and is never picked
//   key    s_e + bias_e, or x_e itself without a bias (the same order)
//   groups value of a group = sum of its `group_best` largest s_e + bias_e;
//          only experts of the topk_groups best groups stay
//   picks  the topk largest keys, ties to the lowest index; a row with fewer
//          open experts gets index -1 and weight 0 behind them
//   weight scale * s_k / sum_j s_j, or scale * s_k
//
// Keys are formed and compared in 64 bits: two experts' keys often lie within
// a few units of the last place of a float, and the choice must not hang on
// the order in which a float sum was taken. CDNA4 runs 64-bit FMA at the
// vector rate of 32 bits, so this costs no extra pass over memory.
//
// A wave holds a token's row in registers, lane l the experts l, l + 64, ...
// (coalesced loads). A pick is an argmax over the wave: the high word of the
// order-preserving integer image of the key is maximised with DPP steps, and
// only when several lanes share it the low word and the index are.

#include <hip/hip_runtime.h>

#include "../device/primitives.h"
#include "expert_ops.h"

namespace uccl {
namespace ep {

namespace {

constexpr int kRouteWaves = 4;

template <typename T>
__device__ inline double load_logit(T const* p) {
  return static_cast<double>(static_cast<float>(*p));
}

// Integer image of a key: larger key, larger image; 0 is "not to be picked"
// (closed experts, NaN keys). -0 and 0 are one value.
__device__ inline uint64_t key_image(double k) {
  if (!(k > -INFINITY)) return 0;
  k += 0.0;
  uint64_t const b = __double_as_longlong(k);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

template <int kCtrl>
__device__ inline uint32_t dpp_max(uint32_t v) {
  // lanes without a source keep their own value
  uint32_t const o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
      static_cast<int>(v), static_cast<int>(v), kCtrl, 0xf, 0xf, false));
  return v > o ? v : o;
}

// Maximum over the 64 lanes, uniform. Row shifts of 1, 2, 4, 8, then the
// last lane of a row and of the lower half are broadcast onward.
__device__ inline uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x111>(v);
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142>(v);
  v = dpp_max<0x143>(v);
  return static_cast<uint32_t>(
      __builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

__device__ inline double wave_fmax(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmax(v, __shfl_xor(v, off));
  return v;
}

}  // namespace

template <typename T, int kPer, bool kSigmoid>
__global__ __launch_bounds__(kRouteWaves * 64) void k_route(
    RouteArgs a, int64_t* __restrict__ idx_out, float* __restrict__ w_out) {
  // keys of this wave's row, for the lanes that rank groups
  __shared__ double ranked[kRouteWaves][kPer * 64];
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const t = blockIdx.x * kRouteWaves + wave;
  if (t >= a.tokens) return;  // waves of a block share nothing
  T const* row = static_cast<T const*>(a.logits) + t * a.stride;

  double x[kPer];
  double top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int v = 0; v < kPer; ++v) {
    int const e = v * 64 + lane;
    x[v] = e < a.experts ? load_logit(row + e) : -INFINITY;
    nan |= x[v] != x[v];
    top = fmax(top, x[v]);
  }
  bool const spoiled_nan = __ballot(nan) != 0;

  bool const grouped = a.groups > 1;
  bool const by_score = a.bias != nullptr || grouped;
  double total = 1.0;
  bool spoiled = spoiled_nan;
  if (!kSigmoid) {
    top = wave_fmax(top);
    spoiled |= top == INFINITY;
    if (by_score || !a.renormalize) {
      double sum = 0.0;
#pragma unroll
      for (int v = 0; v < kPer; ++v)
        if (x[v] > -INFINITY) sum += exp(x[v] - top);
      total = wave_sum(sum);
    }
  }

  uint64_t key[kPer];
  uint64_t open_groups = ~0ull;
  int const group_size = a.experts / a.groups;
  if (by_score) {
#pragma unroll
    for (int v = 0; v < kPer; ++v) {
      int const e = v * 64 + lane;
      bool const open = x[v] > -INFINITY;
      double s = 0.0;
      if (open)
        s = kSigmoid ? 1.0 / (1.0 + exp(-x[v])) : exp(x[v] - top) / total;
      if (a.bias != nullptr && open) s += static_cast<double>(a.bias[e]);
      s = open ? s : -INFINITY;
      key[v] = key_image(a.bias != nullptr ? s : x[v]);
      if (grouped) ranked[wave][e] = s;
    }
  } else {
#pragma unroll
    for (int v = 0; v < kPer; ++v) key[v] = key_image(x[v]);
  }
  if (grouped) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    double first = -INFINITY, second = -INFINITY;
    if (lane < a.groups)
      for (int i = 0; i < group_size; ++i) {
        double const k = ranked[wave][lane * group_size + i];
        if (k > first) {
          second = first;
          first = k;
        } else if (k > second) {
          second = k;
        }
      }
    double value = first;
    if (a.group_best == 2 && second > -INFINITY) value += second;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      double const o = __shfl(value, g);
      rank += o > value || (o == value && g < lane);
    }
    open_groups = __ballot(lane < a.groups && rank < a.topk_groups);
#pragma unroll
    for (int v = 0; v < kPer; ++v) {
      int const e = v * 64 + lane;
      if (e < a.experts && !((open_groups >> (e / group_size)) & 1))
        key[v] = 0;
    }
  }

  int picked = -1;  // lane k: the k-th pick
  for (int k = 0; k < a.topk; ++k) {
    uint64_t best = key[0];
    int at = 0;
#pragma unroll
    for (int v = 1; v < kPer; ++v)
      if (key[v] > best) {
        best = key[v];
        at = v;
      }
    uint32_t const hi = static_cast<uint32_t>(best >> 32);
    uint32_t const top_hi = wave_max(hi);
    if (top_hi == 0) break;  // every open key's image has its high word set
    uint64_t who = __ballot(hi == top_hi);
    int e = at * 64 + lane;
    if (__popcll(who) > 1) {
      uint32_t const lo = static_cast<uint32_t>(best);
      uint32_t const top_lo = wave_max(hi == top_hi ? lo : 0);
      bool const tied = hi == top_hi && lo == top_lo;
      uint32_t const first =
          ~wave_max(tied ? ~static_cast<uint32_t>(e) : 0);
      who = __ballot(tied && static_cast<uint32_t>(e) == first);
    }
    int const winner = __builtin_ctzll(who);
    int const chosen = __builtin_amdgcn_readlane(e, winner);
    if (lane == k) picked = chosen;
#pragma unroll
    for (int v = 0; v < kPer; ++v)
      if (v * 64 + lane == chosen) key[v] = 0;
  }

  double s = 0.0;
  if (picked >= 0) {
    double const xk = load_logit(row + picked);
    s = kSigmoid ? 1.0 / (1.0 + exp(-xk)) : exp(xk - top) / total;
  }
  if (a.renormalize) {
    double const sum = wave_sum(s);
    s = sum > 0.0 ? s / sum : 0.0;
  }
  if (lane < a.topk) {
    int64_t const o = static_cast<int64_t>(t) * a.topk + lane;
    idx_out[o] = picked;
    w_out[o] = spoiled ? NAN : static_cast<float>(s * a.scale);
  }
}

// Gradient of the logits. With r_k = s_k / sum s, g the weights' gradient:
//   softmax, renormalised:  scale r_k (g_k - sum_j g_j r_j)
//   sigmoid, renormalised:  scale r_k (g_k - sum_j g_j r_j)(1 - s_k)
//   softmax:                scale p_e (G_e - sum_k g_k p_k), G_e the g of e
//   sigmoid:                scale g_k s_k (1 - s_k)
// Lane k works out what pick k adds; then each lane gathers, for its experts,
// what the picks add: no atomics, and an index that occurs twice adds twice.
template <typename T, int kPer, bool kSigmoid>
__global__ __launch_bounds__(kRouteWaves * 64) void k_route_grad(
    RouteArgs a, float const* __restrict__ gw,
    int64_t const* __restrict__ idx, T* __restrict__ grad) {
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const t = blockIdx.x * kRouteWaves + wave;
  if (t >= a.tokens) return;
  T const* row = static_cast<T const*>(a.logits) + t * a.stride;

  int e_k = -1;
  double g = 0.0, x_k = -INFINITY;
  if (lane < a.topk) {
    int64_t const o = static_cast<int64_t>(t) * a.topk + lane;
    int64_t const e = idx[o];
    if (e >= 0 && e < a.experts) {
      e_k = static_cast<int>(e);
      g = gw[o];
      x_k = load_logit(row + e_k);
    }
  }
  bool const dense = !kSigmoid && !a.renormalize;
  double x[kPer];
  double top = x_k, total = 1.0;
  if (dense) {
    top = -INFINITY;
#pragma unroll
    for (int v = 0; v < kPer; ++v) {
      int const e = v * 64 + lane;
      x[v] = e < a.experts ? load_logit(row + e) : -INFINITY;
      top = fmax(top, x[v]);
    }
  }
  if (!kSigmoid) top = wave_fmax(top);
  if (dense) {
    total = 0.0;
#pragma unroll
    for (int v = 0; v < kPer; ++v)
      if (x[v] != -INFINITY) total += exp(x[v] - top);
    total = wave_sum(total);
  }
  double s = 0.0;
  if (e_k >= 0 && x_k != -INFINITY)
    s = kSigmoid ? 1.0 / (1.0 + exp(-x_k)) : exp(x_k - top) / total;

  double add, inner = 0.0;
  if (a.renormalize) {
    double const sum = wave_sum(s);
    double const r = sum != 0.0 ? s / sum : 0.0;
    inner = wave_sum(g * r);
    add = a.scale * r * (g - inner);
    if (kSigmoid) add *= 1.0 - s;
  } else if (kSigmoid) {
    add = a.scale * g * s * (1.0 - s);
  } else {
    inner = wave_sum(g * s);
    add = a.scale * g * s;
  }

  double acc[kPer];
#pragma unroll
  for (int v = 0; v < kPer; ++v)
    acc[v] = dense && x[v] != -INFINITY
                 ? -a.scale * inner * (exp(x[v] - top) / total)
                 : 0.0;
  for (int k = 0; k < a.topk; ++k) {
    int const e = __builtin_amdgcn_readlane(e_k, k);
    double const more = __shfl(add, k);
    if (e < 0) continue;
#pragma unroll
    for (int v = 0; v < kPer; ++v)
      if (v * 64 + lane == e) acc[v] += more;
  }
  T* out = grad + static_cast<int64_t>(t) * a.experts;
#pragma unroll
  for (int v = 0; v < kPer; ++v) {
    int const e = v * 64 + lane;
    if (e < a.experts) out[e] = static_cast<T>(static_cast<float>(acc[v]));
  }
}

namespace {

template <typename F>
void by_size(int experts, F&& f) {
  if (experts <= 64) f(std::integral_constant<int, 1>{});
  else if (experts <= 128) f(std::integral_constant<int, 2>{});
  else if (experts <= 256) f(std::integral_constant<int, 4>{});
  else if (experts <= 512) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}

template <typename F>
void by_elem(Elem e, F&& f) {
  if (e == Elem::kF32) f(float{});
  else if (e == Elem::kBF16) f(__hip_bfloat16{});
  else f(__half{});
}

}  // namespace

void launch_route(RouteArgs const& a, int64_t* idx, float* weights,
                  hipStream_t s) {
  int const grid = (a.tokens + kRouteWaves - 1) / kRouteWaves;
  by_elem(a.elem, [&](auto t) {
    using T = decltype(t);
    by_size(a.experts, [&](auto per) {
      constexpr int kPer = decltype(per)::value;
      if (a.sigmoid)
        k_route<T, kPer, true>
            <<<grid, kRouteWaves * 64, 0, s>>>(a, idx, weights);
      else
        k_route<T, kPer, false>
            <<<grid, kRouteWaves * 64, 0, s>>>(a, idx, weights);
    });
  });
}

void launch_route_grad(RouteArgs const& a, float const* grad_weights,
                       int64_t const* idx, void* grad, hipStream_t s) {
  int const grid = (a.tokens + kRouteWaves - 1) / kRouteWaves;
  by_elem(a.elem, [&](auto t) {
    using T = decltype(t);
    by_size(a.experts, [&](auto per) {
      constexpr int kPer = decltype(per)::value;
      if (a.sigmoid)
        k_route_grad<T, kPer, true><<<grid, kRouteWaves * 64, 0, s>>>(
            a, grad_weights, idx, static_cast<T*>(grad));
      else
        k_route_grad<T, kPer, false><<<grid, kRouteWaves * 64, 0, s>>>(
            a, grad_weights, idx, static_cast<T*>(grad));
    });
  });
}

}  // namespace ep
}  // namespace uccl
