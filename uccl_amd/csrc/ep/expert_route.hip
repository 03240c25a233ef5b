// Routing of tokens to experts, and its gradient.
//
//   score  s_e = softmax(x)_e or sigmoid(x_e); an expert whose logit is -inf
//          is closed: it has no score and is never picked
//   rank   s_e + bias_e, or x_e itself without a bias (the same order)
//   groups value of a group = sum of its `group_best` largest s_e + bias_e;
//          only experts of the topk_groups best groups stay
//   picks  the topk largest ranks, ties to the lowest index; a row with fewer
//          open experts gets index -1 and weight 0 behind them
//   weight scale * s_k / sum_j s_j, or scale * s_k
//
// Ranks with a bias or groups are formed and compared in 64 bits: two experts'
// ranks often lie within a few units of the last place of a float, and the
// choice must not hang on the order in which a float sum was taken. CDNA4 runs
// 64-bit FMA at the vector rate of 32 bits, so this costs no extra pass over
// memory. Without them the logits are compared as they are.
//
// A token's row lies in the registers of 64 or 16 lanes, neighbouring experts
// in a lane. 64 lanes are the shorter way for a token (what counts while the
// card has idle waves), 16 take a third of the instructions (what counts when
// it has not): four tokens share a wave, and a maximum over a row of 16 lanes
// is four DPP rotations. A pick is an argmax over the row: the high word of an
// order-preserving integer image of the rank is maximised first, the rest only
// among the lanes that share it.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "expert_ops.h"

namespace uccl {
namespace ep {

namespace {

constexpr int kRouteWaves = 4;

// --- reductions over a token's lanes, the result in all of them ------------

template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(old), static_cast<int>(v),
                                  kCtrl, kRows, 0xf, false));
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ double dpp(double old, double v) {
  uint2 const o = __builtin_bit_cast(uint2, old),
              w = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, make_uint2(dpp<kCtrl, kRows>(o.x, w.x),
                                               dpp<kCtrl, kRows>(o.y, w.y)));
}
__device__ __forceinline__ uint32_t lane63(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ double lane63(double v) {
  uint2 const w = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, make_uint2(lane63(w.x), lane63(w.y)));
}

// 16 lanes: rotations in a row. 64: shifts by 1, 2, 4, 8 in a row, then the
// last lane of a row, and of the lower half, is handed on; lanes without a
// source see `none`.
template <int kLanes, typename V, typename F>
__device__ __forceinline__ V over_row(V v, V none, F&& f) {
  if constexpr (kLanes == 16) {
    v = f(v, dpp<0x128>(v, v));
    v = f(v, dpp<0x124>(v, v));
    v = f(v, dpp<0x122>(v, v));
    return f(v, dpp<0x121>(v, v));
  } else {
    v = f(v, dpp<0x111>(none, v));
    v = f(v, dpp<0x112>(none, v));
    v = f(v, dpp<0x114>(none, v));
    v = f(v, dpp<0x118>(none, v));
    v = f(v, dpp<0x142, 0xa>(none, v));
    v = f(v, dpp<0x143, 0xc>(none, v));
    return lane63(v);
  }
}
template <int kLanes>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  return over_row<kLanes>(v, 0u, [](uint32_t a, uint32_t b) {
    return a > b ? a : b;
  });
}
template <int kLanes>
__device__ __forceinline__ double row_max(double v) {
  return over_row<kLanes>(v, -static_cast<double>(INFINITY),
                          [](double a, double b) { return fmax(a, b); });
}
template <int kLanes>
__device__ __forceinline__ double row_sum(double v) {
  return over_row<kLanes>(v, 0.0, [](double a, double b) { return a + b; });
}

// Integer images of ranks: larger rank, larger image; 0 is "not to be picked"
// (closed experts, NaN ranks), and every other image has a bit of its high
// word set. -0 and 0 are one value.
__device__ __forceinline__ uint64_t image(double k) {
  if (!(k > -static_cast<double>(INFINITY))) return 0;
  uint64_t const b = __double_as_longlong(k + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t image(float k) {
  if (!(k > -INFINITY)) return 0;
  uint32_t const b = __builtin_bit_cast(uint32_t, k + 0.f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_image(uint32_t i) {
  return __builtin_bit_cast(float, (i >> 31) ? i & 0x7fffffffu : ~i);
}

template <bool kSigmoid>
__device__ __forceinline__ double score_of(double x, double top,
                                           double total) {
  if constexpr (kSigmoid) return 1.0 / (1.0 + exp(-x));
  return exp(x - top) / total;
}

template <typename T, int kPer>
using Vec = T __attribute__((ext_vector_type(kPer)));

// kPer neighbouring logits of a row; `whole`: rows of kLanes * kPer experts
// that start at multiples of kPer.
template <typename T, int kPer>
__device__ __forceinline__ void load_logits(float (&x)[kPer], T const* row,
                                            int at, int experts, bool whole) {
  if (whole) {
    if constexpr (kPer == 1) {
      x[0] = static_cast<float>(row[at]);
    } else {
      auto const v = *reinterpret_cast<Vec<T, kPer> const*>(row + at);
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = static_cast<float>(v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      x[i] = at + i < experts ? static_cast<float>(row[at + i]) : -INFINITY;
  }
}

}  // namespace

// kRanked: ranks are scores plus bias, or groups are chosen by scores.
template <typename T, int kLanes, int kPer, bool kSigmoid, bool kRanked>
__global__ __launch_bounds__(kRouteWaves * 64) void k_route(
    RouteArgs a, int64_t* __restrict__ idx_out, float* __restrict__ w_out) {
  constexpr int kTokens = 64 / kLanes;  // of a wave
  constexpr double kInf = INFINITY;
  __shared__ double ranked[kRanked ? kRouteWaves : 1]
                          [kRanked ? kTokens : 1][kRanked ? kLanes * kPer : 1];
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const sub = lane % kLanes, mine = lane / kLanes;
  int const token = (blockIdx.x * kRouteWaves + wave) * kTokens + mine;
  if (token - mine >= a.tokens) return;  // waves of a block share nothing
  // lanes behind the last token go along with it
  int const t = token < a.tokens ? token : a.tokens - 1;
  T const* const row = static_cast<T const*>(a.logits) + t * a.stride;
  int const e0 = sub * kPer;

  float x[kPer];
  load_logits<T, kPer>(x, row, e0, a.experts, a.whole);
  float bias[kRanked ? kPer : 1];
  if constexpr (kRanked) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      bias[i] = a.bias ? a.bias[min(e0 + i, a.experts - 1)] : 0.f;
  }
  double top = 0.0, total = 1.0;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) nan |= x[i] != x[i];
  uint64_t const row_lanes =
      (kLanes == 64 ? ~0ull : (1ull << (kLanes & 63)) - 1) << mine * kLanes;
  bool spoiled = (__ballot(nan) & row_lanes) != 0;
  if constexpr (!kSigmoid) {
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) most = fmaxf(most, x[i]);
    top = row_max<kLanes>(static_cast<double>(most));
    spoiled |= top == kInf;
    if (kRanked || !a.renormalize) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        sum += x[i] > -INFINITY ? exp(x[i] - top) : 0.0;
      total = row_sum<kLanes>(sum);
    }
  }

  // ranks: of 64 bits, or the logit and the index in one word
  uint64_t key[kPer];
  double s[kRanked ? kPer : 1];
  if constexpr (kRanked) {
    bool const grouped = a.groups > 1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int const e = e0 + i;
      bool const open = x[i] > -INFINITY;  // also not NaN
      // worked out for closed ones, too: without a branch the exponentials
      // of a lane's experts overlap
      double const score = score_of<kSigmoid>(x[i], top, total);
      s[i] = open ? score : 0.0;
      double const rank = open ? s[i] + bias[i] : -kInf;
      key[i] = image(a.bias != nullptr ? rank : static_cast<double>(x[i]));
      if (grouped) ranked[wave][mine][e] = rank == rank ? rank : -kInf;
    }
    if (grouped) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      // 2^n lanes for a group; each takes the best two of its share
      int const size = a.experts / a.groups;
      int const log_each = 31 - __builtin_clz(kLanes / a.groups);
      int const each = 1 << log_each, g_mine = sub >> log_each;
      double first = -kInf, second = -kInf;
      auto add = [&](double f1, double f2) {
        second = fmax(fmin(first, f1), fmax(second, f2));
        first = fmax(first, f1);
      };
      if (g_mine < a.groups)
        for (int i = sub & (each - 1); i < size; i += each)
          add(ranked[wave][mine][g_mine * size + i], -kInf);
      for (int by = 1; by < each; by <<= 1) {
        double const f1 = __shfl_xor(first, by), f2 = __shfl_xor(second, by);
        add(f1, f2);
      }
      double value = first;
      if (a.group_best == 2 && second > -kInf) value += second;
      int before = 0;  // groups ahead of this lane's
      for (int g = 0; g < a.groups; ++g) {
        double const o = __shfl(value, (g << log_each) + mine * kLanes);
        before += o > value || (o == value && g < g_mine);
      }
      uint64_t const open_groups =
          __ballot(g_mine < a.groups && before < a.topk_groups) >>
          mine * kLanes;
      float const by_size = 1.f / static_cast<float>(size);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        // exact: e + 1/2 is far from the next multiple for its rounding
        int const g =
            min(static_cast<int>((static_cast<float>(e0 + i) + 0.5f) * by_size),
                a.groups - 1);
        if (!((open_groups >> (g << log_each)) & 1)) key[i] = 0;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      uint32_t const hi = image(x[i]);
      key[i] = hi ? static_cast<uint64_t>(hi) << 32 |
                        ~static_cast<uint32_t>(e0 + i)
                  : 0;
    }
  }

  int picked = -1;  // lane `sub` of a token's: pick number `sub`
  double s_picked = 0.0;
  for (int k = 0; k < a.topk; ++k) {
    uint64_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < kPer; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    uint32_t const hi = static_cast<uint32_t>(best >> 32);
    uint32_t const lo = static_cast<uint32_t>(best);
    uint32_t const top_hi = row_max<kLanes>(hi);
    if (__ballot(top_hi != 0) == 0) break;
    bool cand = hi == top_hi;
    int chosen = e0 + at;
    uint64_t who = __ballot(cand);
    if constexpr (kRanked) {
      if (__popcll(who) > kTokens) {
        uint32_t const top_lo = row_max<kLanes>(cand ? lo : 0);
        cand &= lo == top_lo;
        uint32_t const first = row_max<kLanes>(
            cand ? ~static_cast<uint32_t>(chosen) : 0);
        cand &= ~static_cast<uint32_t>(chosen) == first;
        who = __ballot(cand);
      }
    } else {
      if (__popcll(who) > kTokens) {
        cand &= lo == row_max<kLanes>(cand ? lo : 0);
        who = __ballot(cand);
      }
    }
    // every row with an open expert has one candidate left
    int const winner =
        __builtin_ctzll((who & row_lanes) | 0x8000000000000000ull);
    if constexpr (kLanes == 64) {
      chosen = __builtin_amdgcn_readlane(
          chosen, __builtin_amdgcn_readfirstlane(winner));
      if constexpr (kRanked) {
        double sk = s[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) sk = at == i ? s[i] : sk;
        uint2 const w = __builtin_bit_cast(uint2, sk);
        int const from = __builtin_amdgcn_readfirstlane(winner);
        sk = __builtin_bit_cast(
            double,
            make_uint2(__builtin_amdgcn_readlane(static_cast<int>(w.x), from),
                       __builtin_amdgcn_readlane(static_cast<int>(w.y), from)));
        if (sub == k) s_picked = sk;
      }
    } else {
      chosen = __shfl(chosen, winner);
    }
    bool const open = top_hi != 0;
    if (sub == k && open) {
      picked = chosen;
      if constexpr (!kRanked) s_picked = from_image(top_hi);  // the logit
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (open && e0 + i == chosen) key[i] = 0;
  }

  // weights: lanes below topk
  if constexpr (!kRanked || kLanes != 64) {
    if (picked >= 0) {
      double const xk =
          kRanked ? static_cast<double>(static_cast<float>(row[picked]))
                  : s_picked;
      s_picked = score_of<kSigmoid>(xk, top, total);
    }
  }
  if (picked < 0) s_picked = 0.0;
  if (a.renormalize) {
    double const sum = row_sum<kLanes>(s_picked);
    s_picked = sum > 0.0 ? s_picked / sum : 0.0;
  }
  if (sub < a.topk && token < a.tokens) {
    int64_t const o = static_cast<int64_t>(t) * a.topk + sub;
    idx_out[o] = picked;
    w_out[o] = spoiled ? NAN : static_cast<float>(s_picked * a.scale);
  }
}

// Gradient of the logits. With r_k = s_k / sum s, g the weights' gradient:
//   softmax, renormalised:  scale r_k (g_k - sum_j g_j r_j)
//   sigmoid, renormalised:  scale r_k (g_k - sum_j g_j r_j)(1 - s_k)
//   softmax:                scale p_e (G_e - sum_k g_k p_k), G_e the g of e
//   sigmoid:                scale g_k s_k (1 - s_k)
// Lane k works out what pick k adds; then each lane gathers, for its experts,
// what the picks add: no atomics, and an index that occurs twice adds twice.
template <typename T, int kLanes, int kPer, bool kSigmoid>
__global__ __launch_bounds__(kRouteWaves * 64) void k_route_grad(
    RouteArgs a, float const* __restrict__ gw,
    int64_t const* __restrict__ idx, T* __restrict__ grad) {
  constexpr int kTokens = 64 / kLanes;
  constexpr double kInf = INFINITY;
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const sub = lane % kLanes, mine = lane / kLanes;
  int const token = (blockIdx.x * kRouteWaves + wave) * kTokens + mine;
  if (token - mine >= a.tokens) return;
  int const t = token < a.tokens ? token : a.tokens - 1;
  T const* const row = static_cast<T const*>(a.logits) + t * a.stride;
  int const e0 = sub * kPer;

  int e_k = -1;
  double g = 0.0, x_k = -kInf;
  if (sub < a.topk) {
    int64_t const o = static_cast<int64_t>(t) * a.topk + sub;
    int64_t const e = idx[o];
    if (e >= 0 && e < a.experts) {
      e_k = static_cast<int>(e);
      g = gw[o];
      x_k = static_cast<float>(row[e_k]);
    }
  }
  bool const dense = !kSigmoid && !a.renormalize;
  float x[kPer];
  double top = x_k, total = 1.0;
  if (dense) {
    load_logits<T, kPer>(x, row, e0, a.experts, a.whole);
    top = -kInf;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = fmax(top, x[i]);
  }
  if (!kSigmoid) top = row_max<kLanes>(top);
  if (dense) {
    total = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      total += x[i] != -INFINITY ? exp(x[i] - top) : 0.0;
    total = row_sum<kLanes>(total);
  }
  double s = 0.0;
  if (e_k >= 0 && x_k != -kInf) s = score_of<kSigmoid>(x_k, top, total);

  double add, inner = 0.0;
  if (a.renormalize) {
    double const sum = row_sum<kLanes>(s);
    double const r = sum != 0.0 ? s / sum : 0.0;
    inner = row_sum<kLanes>(g * r);
    add = a.scale * r * (g - inner);
    if (kSigmoid) add *= 1.0 - s;
  } else if (kSigmoid) {
    add = a.scale * g * s * (1.0 - s);
  } else {
    inner = row_sum<kLanes>(g * s);
    add = a.scale * g * s;
  }

  double acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    acc[i] = dense && x[i] != -INFINITY
                 ? -a.scale * inner * (exp(x[i] - top) / total)
                 : 0.0;
  for (int k = 0; k < a.topk; ++k) {
    int const e = __shfl(e_k, mine * kLanes + k);
    double const more = __shfl(add, mine * kLanes + k);
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += e == e0 + i ? more : 0.0;
  }
  if (token >= a.tokens) return;
  T* const out = grad + static_cast<int64_t>(t) * a.experts + e0;
  if (a.whole_out) {
    if constexpr (kPer == 1) {
      out[0] = static_cast<T>(static_cast<float>(acc[0]));
    } else {
      Vec<T, kPer> v;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        v[i] = static_cast<T>(static_cast<float>(acc[i]));
      *reinterpret_cast<Vec<T, kPer>*>(out) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (e0 + i < a.experts)
        out[i] = static_cast<T>(static_cast<float>(acc[i]));
  }
}

namespace {

// 16 lanes for a token where the row and the picks fit and where 64 would
// need more than 4 waves on each of the card's 1024 vector units; more than 32
// where a lane would hold 16 ranks of 64 bits. Measured in us, 64 / 16 lanes:
//   tokens                              2048         4096         8192
//     128 experts, top 8, bf16        4.0 / 5.5    5.1 / 5.6    7.5 / 6.3
//       gradient                      3.2 / 3.6    4.1 / 3.7    6.0 / 4.2
//     256 experts, ranked, 8 groups   7.4 / 13.4  10.6 / 13.7  17.5 / 18.9
//   tokens                             16384        65536
//     128 experts, top 8, bf16       12.4 / 8.8   42.4 / 25.8
//       gradient                      9.8 / 6.0   31.9 / 17.8
//     256 experts, ranked, 8 groups  29.5 / 31.4   105 / 94
// One token of the last takes 5.7: a chain of 8 picks, a few reductions each.
// 4096 tokens read and write 4.6 MB, 0.9 us of a copy; what bounds them is
// the 64-bit exponentials and the picks' reductions.
constexpr int kWideTokens = 4096, kWideRanked = 32768;

template <typename T, int kLanes, int kPer>
void set_whole(RouteArgs& a, void const* grad) {
  constexpr int kBytes = kPer * static_cast<int>(sizeof(T));
  bool const full = a.experts == kLanes * kPer;
  a.whole = full && reinterpret_cast<uintptr_t>(a.logits) % kBytes == 0 &&
            a.stride % kPer == 0;
  a.whole_out = full && reinterpret_cast<uintptr_t>(grad) % kBytes == 0;
}

template <typename T, typename F>
void by_size(RouteArgs const& a, F&& f) {
  auto const call = [&](auto lanes, auto per) { f(T{}, lanes, per); };
#define UCCL_ROUTE(lanes, per)                       \
  call(std::integral_constant<int, lanes>{},         \
       std::integral_constant<int, per>{})
  int const e = a.experts;
  bool const ranked = a.bias != nullptr || a.groups > 1;
  int const wide = ranked && e > 128 ? kWideRanked : kWideTokens;
  if (a.tokens > wide && e <= 256 && a.topk <= 16 && a.groups <= 16) {
    if (e <= 16) UCCL_ROUTE(16, 1);
    else if (e <= 32) UCCL_ROUTE(16, 2);
    else if (e <= 64) UCCL_ROUTE(16, 4);
    else if (e <= 128) UCCL_ROUTE(16, 8);
    else UCCL_ROUTE(16, 16);
  } else {
    if (e <= 64) UCCL_ROUTE(64, 1);
    else if (e <= 128) UCCL_ROUTE(64, 2);
    else if (e <= 256) UCCL_ROUTE(64, 4);
    else if (e <= 512) UCCL_ROUTE(64, 8);
    else UCCL_ROUTE(64, 16);
  }
#undef UCCL_ROUTE
}

template <typename F>
void by_kind(RouteArgs const& a, F&& f) {
  if (a.elem == Elem::kF32) by_size<float>(a, f);
  else if (a.elem == Elem::kBF16) by_size<__bf16>(a, f);
  else by_size<_Float16>(a, f);
}

template <int kLanes>
int grid_of(RouteArgs const& a) {
  constexpr int kTokens = kRouteWaves * (64 / kLanes);
  return (a.tokens + kTokens - 1) / kTokens;
}

}  // namespace

void launch_route(RouteArgs const& args, int64_t* idx, float* weights,
                  hipStream_t s) {
  by_kind(args, [&](auto t, auto lanes, auto per) {
    using T = decltype(t);
    constexpr int kLanes = decltype(lanes)::value, kPer = decltype(per)::value;
    RouteArgs a = args;
    set_whole<T, kLanes, kPer>(a, nullptr);
    int const grid = grid_of<kLanes>(a);
    bool const ranked = a.bias != nullptr || a.groups > 1;
    auto const go = [&](auto sigmoid, auto with_ranks) {
      k_route<T, kLanes, kPer, decltype(sigmoid)::value,
              decltype(with_ranks)::value>
          <<<grid, kRouteWaves * 64, 0, s>>>(a, idx, weights);
    };
    if (a.sigmoid && ranked) go(std::true_type{}, std::true_type{});
    else if (a.sigmoid) go(std::true_type{}, std::false_type{});
    else if (ranked) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
  });
}

void launch_route_grad(RouteArgs const& args, float const* grad_weights,
                       int64_t const* idx, void* grad, hipStream_t s) {
  by_kind(args, [&](auto t, auto lanes, auto per) {
    using T = decltype(t);
    constexpr int kLanes = decltype(lanes)::value, kPer = decltype(per)::value;
    RouteArgs a = args;
    set_whole<T, kLanes, kPer>(a, grad);
    int const grid = grid_of<kLanes>(a);
    if (a.sigmoid)
      k_route_grad<T, kLanes, kPer, true><<<grid, kRouteWaves * 64, 0, s>>>(
          a, grad_weights, idx, static_cast<T*>(grad));
    else
      k_route_grad<T, kLanes, kPer, false><<<grid, kRouteWaves * 64, 0, s>>>(
          a, grad_weights, idx, static_cast<T*>(grad));
  });
}

}  // namespace ep
}  // namespace uccl
