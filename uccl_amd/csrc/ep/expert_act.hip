// Gated activation between two expert products, and its gradient.
//
//   v = silu(a) b, a the first half of a row's columns, b the second
//   to 8 bits: s = max|v| / 448 over each 128 columns (1 where that is 0 as a
//              float), q = the e4m3 value nearest to v / s, ties to even
//   gradient: da = g b sig(a) (1 + a (1 - sig(a))), db = g silu(a)
//
// Every value is read and written once, 16 bytes a lane and load; a wave takes
// 512 columns of a row, or several rows of fewer columns. 16 bits are bound by
// memory: 16384 rows of 2048 columns, 48 us, 4.2 TB/s, and 74 us, 4.5 TB/s, for
// the gradient. 8 bits are bound by the vector units, about 39 instructions a
// value: 32768 rows of 2048 columns, 111 us, 3.0 TB/s.
//
// The exponential is taken of -|a| / 2 and used twice, w = exp(-|a| / 2): for
// a < 0 sig(a) = w w / (1 + w w), and the factors of a product take one w
// each, so nothing overflows, and no product above 6e-36 is lost to an
// underflow on the way (w ends at a = -174.6, where a |b| of 1e36 and more
// would still give a normal one).
//
// 8 bits: scales and values are those of exact arithmetic, whatever the last
// bits of a float exponential are. Only the largest |v| of a group is worked
// out in 64 bits, and values that lie so close to the middle between two 8-bit
// values that 32 bits do not decide; groups whose largest |v| is outside
// 1e-20 .. 1e30, or that have a below -85, entirely.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "expert_ops.h"

namespace uccl {
namespace ep {

namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));
template <typename T>
using x8 = T __attribute__((ext_vector_type(8)));

constexpr int kUnit = 8;  // columns of a lane

// How a wave's lanes lie on the rows of a cell: 64 lanes on 512 columns of a
// row, or several rows of fewer columns.
struct Part {
  int rows;   // rows that a wave takes together
  int lanes;  // lanes of a row
  int parts;  // waves' shares of a row
};

__host__ __device__ inline Part part_of(int cols) {
  int const units = cols / kUnit;
  if (units < 64) return {64 / units, units, 1};
  return {1, 64, (units + 63) / 64};
}

struct Share {
  int at;   // row of the cell
  int col;  // first column
  bool on;  // whether the lane has work
};

// Takes this wave through its shares of the cell's valid rows, kShares at a
// time: parts of a row next to each other, or rows where a row is one share.
// load(shares) asks for a turn's data while work(shares, data) is at the turn
// before. blockIdx: cell, rows, parts. All lanes of a wave call both together.
template <int kShares, bool kSplit, typename Load, typename Work>
__device__ __forceinline__ void each_share(SlotRows const& r, int cols,
                                           Load&& load, Work&& work) {
  Part const p = kSplit ? Part{1, 64, 0} : part_of(cols);
  int const lane = threadIdx.x & 63;
  int const cell = blockIdx.x;
  int const valid =
      r.counts ? min(max(r.counts[cell], 0), r.length) : r.length;
  int const row = kSplit ? 0 : lane / p.lanes;
  int const in_row = lane - row * p.lanes;
  int const waves = gridDim.y * (blockDim.x >> 6);
  int const part = kSplit ? blockIdx.z * kShares : 0;
  int64_t const stride = static_cast<int64_t>(waves) * p.rows;
  int64_t const turn = kSplit ? stride : stride * kShares;
  struct Shares {
    Share s[kShares];
  };
  auto shares_at = [&](int64_t first) {
    Shares t;
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
      int64_t const begin = first + (kSplit ? 0 : k * stride) + row;
      t.s[k].at = begin < valid ? static_cast<int>(begin) : valid;
      t.s[k].col = ((part + (kSplit ? k : 0)) * 64 + in_row) * kUnit;
      t.s[k].on = row < p.rows && t.s[k].at < valid && t.s[k].col < cols;
    }
    return t;
  };
  int64_t first = (blockIdx.y * static_cast<int64_t>(blockDim.x >> 6) +
                   __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) *
                  p.rows;
  if (first >= valid) return;
  Shares now = shares_at(first);
  auto data = load(now.s);
  for (;;) {
    first += turn;
    Shares const next = shares_at(first);
    auto const more = load(next.s);
    work(now.s, data);
    if (first >= valid) break;
    now = next;
    data = more;
  }
}

// First row of the block's cell.
__device__ __forceinline__ char* cell_of(Mat const& m, SlotRows const& r,
                                         int size) {
  int const e = blockIdx.x / r.sources;
  int const source = blockIdx.x - e * r.sources;
  return static_cast<char*>(m.p) +
         (e * m.expert_stride +
          static_cast<int64_t>(source) * r.length * m.row_stride) *
             size;
}
__device__ __forceinline__ char* row_at(char* cell, Mat const& m, int at,
                                        int size) {
  return cell + static_cast<int64_t>(at) * m.row_stride * size;
}

template <typename T>
__device__ __forceinline__ x8<T> load8(char const* row, int col) {
  return reinterpret_cast<x8<T> const*>(row)[col / kUnit];
}
template <typename T>
__device__ __forceinline__ f32x8 floats(x8<T> v) {
  return __builtin_convertvector(v, f32x8);
}
// Past the caches, where results would take the place of what is still to be
// read: 16384 rows of 2048 columns, 49 -> 47 us, gradient 84 -> 74 us. (Loads
// past the caches cost 10%.)
template <typename T>
__device__ __forceinline__ void store8(char* row, int col, f32x8 v) {
  __builtin_nontemporal_store(__builtin_convertvector(v, x8<T>),
                              reinterpret_cast<x8<T>*>(row) + col / kUnit);
}

// exp(-|a| / 2), good to about a unit in the last place: the part of the
// exponent that its product lost is put back.
__device__ __forceinline__ float half_exp(float a) {
  // log2(e) / 2, in two parts
  constexpr float kHigh = 0.72134752f, kLow = 9.629815e-9f;
  // Beyond -1000 the exponential is 0 as well, and an infinite a would leave
  // inf - inf in the lost part. (A NaN is lost here, but every result has a
  // as a factor, too.)
  float const x = fmaxf(-fabsf(a), -1000.f);
  float const h = x * kHigh;
  float const l = fmaf(x, kLow, fmaf(x, kHigh, -h));
  float const e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, l * 0.69314718f, e);
}

struct Gate {
  float w;     // 1, or exp(a / 2) where a < 0
  float norm;  // 1 / (1 + exp(-|a|)); sig(a) = w w norm
};
__device__ __forceinline__ Gate gate_of(float a) {
  float const e = half_exp(a);
  return {a < 0.f ? e : 1.f, __builtin_amdgcn_rcpf(fmaf(e, e, 1.f))};
}

__device__ __forceinline__ float silu_mul(float a, float b) {
  Gate const g = gate_of(a);
  return (a * g.w) * g.norm * (g.w * b);
}

__device__ __forceinline__ double silu_mul_exact(float a, float b) {
  double const x = a;
  return x / (1.0 + exp(-x)) * static_cast<double>(b);
}

// Nearest 8-bit value to y, given back as a float, ties to even.
__device__ __forceinline__ float nearest_exact(double y) {
  int e;
  (void)frexp(y, &e);
  double const step = ldexp(1.0, max(e - 4, -9));
  double const r = rint(y / step) * step;
  return static_cast<float>(r > 448.0 ? 448.0 : r < -448.0 ? -448.0 : r);
}

// Largest of the 16 lanes of a group, in all of them: rotations in a DPP row.
template <int kBy>
__device__ __forceinline__ int rotated(int v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + kBy, 0xf, 0xf, false);
}
template <int kBy = 8>
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, __builtin_bit_cast(
                   float, rotated<kBy>(__builtin_bit_cast(int, v))));
  if constexpr (kBy > 1) v = group_max<kBy / 2>(v);
  return v;
}
template <int kBy = 8>
__device__ __forceinline__ double group_max(double v) {
  int2 const w = __builtin_bit_cast(int2, v);
  v = fmax(v, __builtin_bit_cast(
                  double, make_int2(rotated<kBy>(w.x), rotated<kBy>(w.y))));
  if constexpr (kBy > 1) v = group_max<kBy / 2>(v);
  return v;
}

// Whether one of the values is below -85: among negative values, the order of
// the bits. A negative NaN counts too.
template <typename T>
__device__ __forceinline__ bool ends_exp(x8<T> v) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x8 const bits = __builtin_bit_cast(u16x8, v);
  u16x4 const four = __builtin_elementwise_max(
      __builtin_shufflevector(bits, bits, 0, 1, 2, 3),
      __builtin_shufflevector(bits, bits, 4, 5, 6, 7));
  u16x2 const two = __builtin_elementwise_max(
      __builtin_shufflevector(four, four, 0, 1),
      __builtin_shufflevector(four, four, 2, 3));
  constexpr unsigned short kEnd =
      __builtin_bit_cast(unsigned short, static_cast<T>(-85.f));
  return two[0] > kEnd || two[1] > kEnd;
}

// Four values as 8-bit ones, each times `by`.
__device__ __forceinline__ unsigned to_8bit(float a, float b, float c, float d,
                                            float by) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * by, b * by, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c * by, d * by, v, true);
}

// The j-th of 16 values, of two lots of 8.
template <typename T>
__device__ __forceinline__ float pick(x8<T> const (&v)[2], int j) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  i32x4 const p = __builtin_bit_cast(i32x4, v[0]),
              q = __builtin_bit_cast(i32x4, v[1]);
  int r = p[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) r = (j >> 1) == k ? (k < 4 ? p[k] : q[k - 4]) : r;
  auto const half =
      static_cast<unsigned short>(static_cast<unsigned>(r) >> (j & 1) * 16);
  return static_cast<float>(__builtin_bit_cast(T, half));
}

}  // namespace

template <typename T, bool kSplit>
__global__ __launch_bounds__(256) void k_swiglu(SwigluArgs a) {
  char* const h_cell = cell_of(a.h, a.rows, sizeof(T));
  char* const out_cell = cell_of(a.out, a.rows, sizeof(T));
  struct Data {
    x8<T> x, b;
  };
  auto load = [&](Share const (&s)[1]) {
    Data d{};
    if (s[0].on) {
      char const* const h = row_at(h_cell, a.h, s[0].at, sizeof(T));
      d.x = load8<T>(h, s[0].col);
      d.b = load8<T>(h, a.cols + s[0].col);
    }
    return d;
  };
  each_share<1, kSplit>(a.rows, a.cols, load, [&](Share const (&s)[1],
                                                  Data const& d) {
    if (!s[0].on) return;
    f32x8 const x = floats<T>(d.x), b = floats<T>(d.b);
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = silu_mul(x[j], b[j]);
    store8<T>(row_at(out_cell, a.out, s[0].at, sizeof(T)), s[0].col, v);
  });
}

// Two shares at a time, so that one pass in 64 bits serves both: each lane
// brings the largest of its values, if that may be its group's largest.
template <typename T, bool kSplit>
__global__ __launch_bounds__(256) void k_swiglu_quant(SwigluArgs a) {
  constexpr int kShares = 2;
  char* const h_cell = cell_of(a.h, a.rows, sizeof(T));
  char* const out_cell = cell_of(a.out, a.rows, 1);
  char* const scale_cell = cell_of(a.scales, a.rows, 4);
  struct Data {
    x8<T> x[kShares], b[kShares];
  };
  auto load = [&](Share const (&s)[kShares]) {
    Data d{};
#pragma unroll
    for (int k = 0; k < kShares; ++k)
      if (s[k].on) {
        char const* const h = row_at(h_cell, a.h, s[k].at, sizeof(T));
        d.x[k] = load8<T>(h, s[k].col);
        d.b[k] = load8<T>(h, a.cols + s[k].col);
      }
    return d;
  };
  each_share<kShares, kSplit>(a.rows, a.cols, load,
                              [&](Share const (&s)[kShares], Data const& raw) {
    // a group's 128 columns are 16 neighbouring lanes, all of them on or off
    f32x8 v[kShares];
    // v in 32 bits, good to 70 parts in 2^24 for a down to -85: 64 of the
    // exponential (its argument is rounded, up to 45, and so is log2(e) in
    // it, 0.22 |a|) and one of each operation more. Groups with a below -85,
    // where the exponential ends, or whose largest |v| is far from 1 are
    // `wild`: nothing of them is decided in 32 bits.
    bool wild[kShares];
    float limit[kShares];         // below it, no value is its group's largest
    float top_x[kShares], top_b[kShares];  // where this lane's largest is
    unsigned open = 0;  // shares with a lane's largest to work out
    unsigned left = 0;  // further values, when one does not do
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
      f32x8 const x = floats<T>(raw.x[k]), b = floats<T>(raw.b[k]);
      float most = -1.f, second = -1.f;
      top_x[k] = top_b[k] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float const e = __builtin_amdgcn_exp2f(x[j] * -1.44269504f);
        v[k][j] = x[j] * b[j] * __builtin_amdgcn_rcpf(1.f + e);
        float const size = fabsf(v[k][j]);
        bool const more = size > most;
        top_x[k] = more ? x[j] : top_x[k];
        top_b[k] = more ? b[j] : top_b[k];
        second = __builtin_amdgcn_fmed3f(second, size, most);
        most = fmaxf(most, size);
      }
      float const group =
          group_max(ends_exp<T>(raw.x[k]) ? INFINITY : most);
      wild[k] = !(group >= 1e-20f && group <= 1e30f);
      limit[k] = group * (1.f - 0x1p-15f);
      if (s[k].on) {
        if (!wild[k] && most >= limit[k]) open |= 1u << k;
        if (wild[k] || second >= limit[k]) left |= 0xffu << (k * 8);
      }
    }
    double exact[kShares] = {};
    while (open) {
      int const k = __builtin_ctz(open);
      open &= open - 1;
      double const size = fabs(silu_mul_exact(k ? top_x[1] : top_x[0],
                                              k ? top_b[1] : top_b[0]));
      exact[0] = fmax(exact[0], k ? 0.0 : size);
      exact[1] = fmax(exact[1], k ? size : 0.0);
    }
    while (left) {
      int const j = __builtin_ctz(left);
      left &= left - 1;
      double const size =
          fabs(silu_mul_exact(pick<T>(raw.x, j), pick<T>(raw.b, j)));
      exact[0] = fmax(exact[0], j < 8 ? size : 0.0);
      exact[1] = fmax(exact[1], j < 8 ? 0.0 : size);
    }
    // Scaled values are known to 96 parts in 2^24: the error above, and that
    // of the scaling. Where a value less 2^-17 of it and the value and 2^-17
    // of it become the same 8-bit value, it is that one; else 32 bits do not
    // decide.
    constexpr float kNear = 0x1p-17f;
    unsigned values[kShares][2];
    float scale[kShares];
    unsigned near = 0;
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
      double const largest = group_max(exact[k]);
      // the quotient by 448, rounded once: a product with 1 / 448, corrected
      double q = largest * (1.0 / 448.0);
      q = fma(fma(-448.0, q, largest), 1.0 / 448.0, q);
      scale[k] = static_cast<float>(largest < INFINITY ? q : largest);
      // also where the largest is not 0 but its 448th part rounds to 0: the
      // group's values then are 0, not quotients by 0
      if (!(scale[k] > 0.f)) scale[k] = 1.f;
      float const inverse = __builtin_amdgcn_rcpf(scale[k]);
      unsigned differ[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        auto const scaled = [&](float by) {
          return to_8bit(v[k][d * 4], v[k][d * 4 + 1], v[k][d * 4 + 2],
                         v[k][d * 4 + 3], by);
        };
        values[k][d] = scaled(inverse * (1.f - kNear));
        differ[d] = values[k][d] ^ scaled(inverse * (1.f + kNear));
      }
      if (s[k].on && ((differ[0] | differ[1]) != 0 || wild[k])) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((differ[j / 4] >> (j % 4 * 8) & 0xffu) || wild[k])
            near |= 1u << (k * 8 + j);
      }
    }
    while (near) {
      int const j = __builtin_ctz(near);
      near &= near - 1;
      float const y =
          nearest_exact(silu_mul_exact(pick<T>(raw.x, j), pick<T>(raw.b, j)) /
                        (j < 8 ? scale[0] : scale[1]));
      unsigned const place = 0xffu << (j & 3) * 8;
      unsigned const value = to_8bit(y, y, y, y, 1.f) & place;
#pragma unroll
      for (int k = 0; k < kShares; ++k)
#pragma unroll
        for (int d = 0; d < 2; ++d)
          if ((j >> 2) == k * 2 + d)
            values[k][d] = (values[k][d] & ~place) | value;
    }
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
      if (!s[k].on) continue;
      char* const out = row_at(out_cell, a.out, s[k].at, 1);
      *reinterpret_cast<uint2*>(out + s[k].col) = make_uint2(values[k][0], values[k][1]);
      if ((threadIdx.x & 15) == 0)
        reinterpret_cast<float*>(
            row_at(scale_cell, a.scales, s[k].at, 4))[s[k].col / 128] =
            scale[k];
    }
  });
}

template <typename T, bool kSplit>
__global__ __launch_bounds__(256) void k_swiglu_grad(SwigluArgs a) {
  char* const h_cell = cell_of(a.h, a.rows, sizeof(T));
  char* const g_cell = cell_of(a.grad_out, a.rows, sizeof(T));
  char* const out_cell = cell_of(a.out, a.rows, sizeof(T));
  struct Data {
    x8<T> x, b, g;
  };
  auto load = [&](Share const (&s)[1]) {
    Data d{};
    if (s[0].on) {
      char const* const h = row_at(h_cell, a.h, s[0].at, sizeof(T));
      d.x = load8<T>(h, s[0].col);
      d.b = load8<T>(h, a.cols + s[0].col);
      d.g = load8<T>(row_at(g_cell, a.grad_out, s[0].at, sizeof(T)),
                     s[0].col);
    }
    return d;
  };
  each_share<1, kSplit>(a.rows, a.cols, load, [&](Share const (&s)[1],
                                                  Data const& d) {
    if (!s[0].on) return;
    int const col = s[0].col;
    f32x8 const x = floats<T>(d.x), b = floats<T>(d.b), g = floats<T>(d.g);
    f32x8 da, db;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      Gate const t = gate_of(x[j]);
      float const gn = (g[j] * t.w) * t.norm;
      float const sig = t.w * t.w * t.norm;
      db[j] = gn * (t.w * x[j]);
      da[j] = gn * (t.w * b[j]) * fmaf(x[j], 1.f - sig, 1.f);
    }
    char* const out = row_at(out_cell, a.out, s[0].at, sizeof(T));
    store8<T>(out, col, da);
    store8<T>(out, a.cols + col, db);
  });
}

namespace {

// At most kMost blocks, of 4 waves with a row or more each: few enough that
// a wave has rows to load ahead of, enough to fill the card. The host does not
// know the counts; a block without rows ends at once.
constexpr int64_t kMost = 4096;
dim3 share_grid(SwigluArgs const& a, int shares) {
  Part const p = part_of(a.cols);
  int64_t const cells = static_cast<int64_t>(a.rows.experts) * a.rows.sources;
  int64_t const z = p.parts > 1 ? (p.parts + shares - 1) / shares : 1;
  int64_t const rows = (a.rows.length + p.rows - 1) / p.rows;
  int64_t const y = std::min(std::max<int64_t>(1, kMost / (cells * z)),
                             (rows + 3) / 4);
  return dim3(static_cast<unsigned>(cells), static_cast<unsigned>(y),
              static_cast<unsigned>(z));
}

// f(T{}, whether a row has several shares)
template <typename F>
void by_kind(SwigluArgs const& a, F&& f) {
  auto const split = [&](auto t) {
    if (part_of(a.cols).parts > 1)
      f(t, std::true_type{});
    else
      f(t, std::false_type{});
  };
  if (a.elem == Elem::kBF16)
    split(__bf16{});
  else
    split(_Float16{});
}

}  // namespace

void launch_expert_swiglu(SwigluArgs const& a, hipStream_t s) {
  dim3 const grid = share_grid(a, a.quantize ? 2 : 1);
  by_kind(a, [&](auto t, auto split) {
    if (a.quantize)
      k_swiglu_quant<decltype(t), decltype(split)::value>
          <<<grid, 256, 0, s>>>(a);
    else
      k_swiglu<decltype(t), decltype(split)::value><<<grid, 256, 0, s>>>(a);
  });
}

void launch_expert_swiglu_grad(SwigluArgs const& a, hipStream_t s) {
  dim3 const grid = share_grid(a, 1);
  by_kind(a, [&](auto t, auto split) {
    k_swiglu_grad<decltype(t), decltype(split)::value>
        <<<grid, 256, 0, s>>>(a);
  });
}

}  // namespace ep
}  // namespace uccl
