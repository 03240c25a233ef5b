// Compute operators of an expert layer over the EP slot arrays: routing,
// the experts' matrix products, their weight gradient, and the gated
// activation between two products. The launchers check nothing: shapes,
// strides, alignment and limits are checked in bindings/expert_ops.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace uccl {
namespace ep {

enum class Elem : int { kF8 = 0, kBF16 = 1, kF16 = 2, kF32 = 3 };

constexpr int kMaxRouteExperts = 1024;  // a wave holds a row, 16 a lane
constexpr int kMaxRouteTopk = 64;       // one lane for each pick
constexpr int kMaxRouteGroups = 64;     // one bit of a lane mask each
constexpr int kMaxSlotExperts = 1024;   // experts, and experts * sources:
constexpr int kMaxSlotCells = 2048;     // their row counts are held in LDS

// Rows of a slot array [experts, sources * length, cols]: source r of
// expert e has counts[e * sources + r] valid rows from r * length on.
// counts == nullptr: all rows are valid. Kernels clamp a count into
// [0, length], so no value of it leads out of the array.
struct SlotRows {
  int const* counts;
  int experts;
  int sources;
  int length;
};

struct RouteArgs {
  void const* logits;  // [tokens, experts], rows `stride` elements apart
  int64_t stride;
  Elem elem;  // kF32 | kBF16 | kF16
  int tokens, experts, topk;
  bool sigmoid;       // else softmax
  float const* bias;  // [experts] or nullptr
  int groups, topk_groups, group_best;
  bool renormalize;
  float scale;
  // set by the launchers: rows can be read, the gradient's be written, a
  // lane's experts at a time
  bool whole, whole_out;
};
void launch_route(RouteArgs const& a, int64_t* idx, float* weights,
                  hipStream_t s);
// grad: [tokens, experts] of `a.elem`, dense.
void launch_route_grad(RouteArgs const& a, float const* grad_weights,
                       int64_t const* idx, void* grad, hipStream_t s);

// One operand or result of a grouped product; strides in elements.
struct Mat {
  void* p;
  int64_t expert_stride;
  int64_t row_stride;
};

struct MatmulArgs {
  SlotRows rows;
  Mat x;    // [experts, slots, k]
  Mat w;    // [experts, n, k], or [experts, k, n] where w_turned
  Mat out;  // [experts, slots, n]
  bool w_turned;
  int n, k;
  Elem elem;      // of x and w
  Elem out_elem;  // kBF16 | kF16 | kF32
  // 8-bit only: scales [experts, slots, k/128] and [experts, ceil(n/128),
  // k/128], dense in their last dimension
  Mat x_scales, w_scales;
  int expected_rows;  // rows an expert is expected to have; picks the tile
  bool precise;  // 8-bit only: sums of 32 bits, and any out_elem
};
void launch_expert_matmul(MatmulArgs const& a, hipStream_t s);

struct WeightGradArgs {
  SlotRows rows;
  Mat grad;  // [experts, slots, n]
  Mat x;     // [experts, slots, k]
  Mat out;   // [experts, n, k]
  int n, k;
  Elem elem;
  Elem out_elem;
};
void launch_expert_weight_grad(WeightGradArgs const& a, hipStream_t s);

struct SwigluArgs {
  SlotRows rows;
  Mat h;    // [experts, slots, 2 * cols]
  Mat out;  // [experts, slots, cols], kF8 with scales or h's type
  Mat scales;
  Mat grad_out;  // gradient pass only: [experts, slots, cols]
  int cols;
  Elem elem;  // of h
  bool quantize;
};
void launch_expert_swiglu(SwigluArgs const& a, hipStream_t s);
// out: [experts, slots, 2 * cols]
void launch_expert_swiglu_grad(SwigluArgs const& a, hipStream_t s);

}  // namespace ep
}  // namespace uccl
