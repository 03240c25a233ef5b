// Gated activation between two expert products, and its gradient.
//
//   v = silu(a) b, a the first half of a row's columns, b the second
//   to 8 bits: s = max|v| / 448 over each 128 columns (1 if all are 0),
//              q = the e4m3 value nearest to v / s, ties to even
//   gradient: da = g b sig(a) (1 + a (1 - sig(a))), db = g silu(a)
//
// Bound by memory: every value is read and written once, 16 bytes a lane.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../core/log.h"
#include "../device/primitives.h"
#include "expert_ops.h"

namespace uccl {
namespace ep {

using namespace uccl::device;

namespace {

__device__ __forceinline__ int clamp_count(SlotRows const& r, int i) {
  return r.counts ? min(max(r.counts[i], 0), r.length) : r.length;
}

__device__ __forceinline__ double silu_mul(double a, double b) {
  return a / (1.0 + exp(-a)) * b;
}

}  // namespace

// Grid: (cells = experts * sources, row chunks). One wave takes a row at a
// time.
template <typename T, bool kQuantize>
__global__ __launch_bounds__(256) void k_swiglu(SwigluArgs a) {
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const cell = blockIdx.x;
  int const e = cell / a.rows.sources, src = cell % a.rows.sources;
  int const valid = clamp_count(a.rows, cell);
  for (int i = blockIdx.y * 4 + wave; i < valid; i += gridDim.y * 4) {
    int64_t const slot = static_cast<int64_t>(src) * a.rows.length + i;
    T const* row = static_cast<T const*>(a.h.p) + e * a.h.expert_stride +
                   slot * a.h.row_stride;
    if constexpr (kQuantize) {
      __hip_fp8_e4m3* out = static_cast<__hip_fp8_e4m3*>(a.out.p) +
                            e * a.out.expert_stride + slot * a.out.row_stride;
      float* scales = static_cast<float*>(a.scales.p) +
                      e * a.scales.expert_stride + slot * a.scales.row_stride;
      for (int g = 0; g < a.cols / 128; ++g) {
        double v[2];
        double most = 0.0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          int const c = g * 128 + lane * 2 + j;
          v[j] = silu_mul(static_cast<float>(row[c]),
                          static_cast<float>(row[a.cols + c]));
          most = fmax(most, fabs(v[j]));
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
          most = fmax(most, __shfl_xor(most, off));
        float const scale = most > 0.0 ? static_cast<float>(most / 448.0) : 1.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          double const y = v[j] / scale;
          int ex;
          frexp(y, &ex);
          double const step = ldexp(1.0, max(ex - 4, -9));
          out[g * 128 + lane * 2 + j] =
              __hip_fp8_e4m3(static_cast<float>(rint(y / step) * step));
        }
        if (lane == 0) scales[g] = scale;
      }
    } else {
      T* out = static_cast<T*>(a.out.p) + e * a.out.expert_stride +
               slot * a.out.row_stride;
      for (int c = lane; c < a.cols; c += 64) {
        float const x = static_cast<float>(row[c]);
        float const b = static_cast<float>(row[a.cols + c]);
        out[c] = static_cast<T>(x / (1.f + expf(-x)) * b);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_swiglu_grad(SwigluArgs a) {
  int const wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int const cell = blockIdx.x;
  int const e = cell / a.rows.sources, src = cell % a.rows.sources;
  int const valid = clamp_count(a.rows, cell);
  for (int i = blockIdx.y * 4 + wave; i < valid; i += gridDim.y * 4) {
    int64_t const slot = static_cast<int64_t>(src) * a.rows.length + i;
    T const* row = static_cast<T const*>(a.h.p) + e * a.h.expert_stride +
                   slot * a.h.row_stride;
    T const* gr = static_cast<T const*>(a.grad_out.p) +
                  e * a.grad_out.expert_stride + slot * a.grad_out.row_stride;
    T* out = static_cast<T*>(a.out.p) + e * a.out.expert_stride +
             slot * a.out.row_stride;
    for (int c = lane; c < a.cols; c += 64) {
      float const x = static_cast<float>(row[c]);
      float const b = static_cast<float>(row[a.cols + c]);
      float const g = static_cast<float>(gr[c]);
      float const sig = 1.f / (1.f + expf(-x));
      out[c] = static_cast<T>(g * b * sig * (1.f + x * (1.f - sig)));
      out[a.cols + c] = static_cast<T>(g * x * sig);
    }
  }
}

namespace {

dim3 row_grid(SlotRows const& r) {
  int const cells = r.experts * r.sources;
  return dim3(cells, std::max(1, std::min((r.length + 3) / 4, 4096 / cells)));
}

}  // namespace

void launch_expert_swiglu(SwigluArgs const& a, hipStream_t s) {
  dim3 const grid = row_grid(a.rows);
  if (a.elem == Elem::kBF16) {
    if (a.quantize)
      k_swiglu<__hip_bfloat16, true><<<grid, 256, 0, s>>>(a);
    else
      k_swiglu<__hip_bfloat16, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (a.quantize)
      k_swiglu<__half, true><<<grid, 256, 0, s>>>(a);
    else
      k_swiglu<__half, false><<<grid, 256, 0, s>>>(a);
  }
}

void launch_expert_swiglu_grad(SwigluArgs const& a, hipStream_t s) {
  dim3 const grid = row_grid(a.rows);
  if (a.elem == Elem::kBF16)
    k_swiglu_grad<__hip_bfloat16><<<grid, 256, 0, s>>>(a);
  else
    k_swiglu_grad<__half><<<grid, 256, 0, s>>>(a);
}

}  // namespace ep
}  // namespace uccl
