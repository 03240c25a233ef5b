// The experts' matrix products over slot arrays, and their weight gradient.
//
//   product        y[m, n]  = sum_k x[m, k] w[n, k]
//     8 bit:       y[m, n]  = sum_b sx[m, b] sw[n / 128, b]
//                             sum_{k in block b} qx[m, k] qw[n, k]
//   turned weights (k and n swapped in memory) give the rows' gradient
//   weight gradient  dw[n, k] = sum_m g[m, n] x[m, k], over the valid rows
//
// One kernel computes D[p, q] = sum_c P[p, c] Q[q, c] tile by tile with MFMA
// 16x16 instructions; a lane then holds 4 consecutive p of one q, so p is the
// contiguous dimension of the result: P = w, Q = x for a product, P = x^T,
// Q = g^T for the weight gradient.
//
// The tile's operands go from memory to LDS in steps of 128 bytes (direct
// operands, contiguous along c) or 64 rows (turned operands, contiguous along
// p or q; read back through the transposing LDS load), double-buffered, by
// loads that write LDS without passing registers. Each lane forms its own
// address, so the valid rows of all sources are gathered on the way: a tile
// is full of valid rows wherever they lie.
//
// Rows behind an expert's last are never read: tiles are cut from the number
// of valid rows, lanes behind the last row load it again, and lanes behind
// the end of the contraction load from a page of zeros.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../core/log.h"
#include "../device/primitives.h"
#include "expert_ops.h"

// The loads below list m0 as clobbered, which is what tells the compiler that
// they set it; it warns for every such listing of a reserved register.
#pragma clang diagnostic ignored "-Winline-asm"

namespace uccl {
namespace ep {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kStep = 128;  // bytes of the contraction in a stage, a row

// 16 bytes of zeros: where lanes behind the contraction's end load from.
__device__ const int4 zero_page = {0, 0, 0, 0};

// Load 16 (4) bytes of each lane from its own address to LDS at `lds` + lane
// * 16 (* 4). The instruction has no register result; the caller waits with
// wait_loads() and a barrier before the LDS is read.
__device__ __forceinline__ void lds_load16(void const* g, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
      :
      : "v"(g), "s"(lds)
      : "memory", "m0");
}
__device__ __forceinline__ void lds_load4(void const* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(g), "s"(lds)
               : "memory", "m0");
}

// Every load to LDS of this wave has landed, every LDS read of it is done,
// and so for the other waves of the block.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_addr(void const* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)p));
}

__device__ __forceinline__ int clamp_count(SlotRows const& r, int i) {
  return r.counts ? min(max(r.counts[i], 0), r.length) : r.length;
}

__device__ __forceinline__ int rows_of(SlotRows const& r, int e) {
  int n = 0;
  for (int s = 0; s < r.sources; ++s) n += clamp_count(r, e * r.sources + s);
  return n;
}

// Slot of the i-th valid row of expert e; i < rows_of(e).
__device__ __forceinline__ int slot_of(SlotRows const& r, int e, int i) {
  i = max(i, 0);
  for (int s = 0; s < r.sources; ++s) {
    int const n = clamp_count(r, e * r.sources + s);
    if (i < n) return s * r.length + i;
    i -= n;
  }
  return 0;
}

struct GemmArgs {
  SlotRows rows;
  char const* p;
  char const* q;
  char* out;
  // bytes
  int64_t p_expert, p_row, q_expert, q_row, out_expert, out_row;
  int np;       // extent of p
  int nq;       // extent of q (weight gradient only; else the valid rows)
  int depth;    // contraction in elements (product only)
  char const* q_scales;
  char const* p_scales;
  int64_t qs_expert, qs_row, ps_expert, ps_row;  // bytes
};

enum class Mode { kProduct, kProductTurned, kWeightGrad };

template <Elem kElem>
__device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c) {
  if constexpr (kElem == Elem::kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
        0);
}

__device__ __forceinline__ f32x4 mfma8(i32x8 a, i32x8 b) {
  f32x4 const zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0,
                                                          0, 0, 0);
}

template <Elem kOut>
__device__ __forceinline__ void store4(char* at, f32x4 v, int n, bool wide) {
  using T = std::conditional_t<
      kOut == Elem::kF32, float,
      std::conditional_t<kOut == Elem::kBF16, __hip_bfloat16, __half>>;
  T* o = reinterpret_cast<T*>(at);
  if (wide) {
    struct alignas(4 * sizeof(T)) Four {
      T v[4];
    } four;
#pragma unroll
    for (int j = 0; j < 4; ++j) four.v[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Four*>(o) = four;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) o[j] = static_cast<T>(v[j]);
  }
}

// Tiles BP x BQ, WP x WQ waves, two stages.
template <Mode kMode, Elem kElem, Elem kOut, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(WP* WQ * 64, 2) void k_expert_gemm(GemmArgs a) {
  constexpr bool kWGrad = kMode == Mode::kWeightGrad;
  constexpr bool kPTurned = kMode != Mode::kProduct;
  constexpr bool kQTurned = kWGrad;
  constexpr bool k8 = kElem == Elem::kF8;
  constexpr int kSize = k8 ? 1 : 2;
  constexpr int kDepth = kStep / kSize;  // contraction elements of a stage
  constexpr int kWaves = WP * WQ, kThreads = kWaves * 64;
  constexpr int TP = BP / WP / 16, TQ = BQ / WQ / 16;  // 16x16 tiles of a wave
  constexpr int kPBytes = BP * kStep, kQBytes = BQ * kStep;
  constexpr int kScaleBytes = k8 ? BQ * 4 : 0;
  constexpr int kStage = kPBytes + kQBytes + kScaleBytes;
  constexpr int kPLoads = kPBytes / 1024 / kWaves;
  constexpr int kQLoads = kQBytes / 1024 / kWaves;
  static_assert(kPLoads * 1024 * kWaves == kPBytes, "P loads");
  static_assert(kQLoads * 1024 * kWaves == kQBytes, "Q loads");
  static_assert(!k8 || 128 % (BP / WP) == 0, "a wave stays in a scale block");

  __shared__ __attribute__((aligned(1024))) char stages[2 * kStage];
  __shared__ int tile_end[kWGrad ? 1 : kMaxSlotExperts];
  __shared__ int slots[kWGrad ? 2 * kDepth : BQ];

  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const lane = threadIdx.x & 63;
  int const wp = wave % WP, wq = wave / WP;
  uint32_t const lds0 = lds_addr(stages);

  // --- tiles of all experts ------------------------------------------------
  int const tiles_p = (a.np + BP - 1) / BP;
  int total;
  if constexpr (kWGrad) {
    total = a.rows.experts * tiles_p * ((a.nq + BQ - 1) / BQ);
  } else {
    for (int e = threadIdx.x; e < a.rows.experts; e += kThreads)
      tile_end[e] = (rows_of(a.rows, e) + BQ - 1) / BQ * tiles_p;
    __syncthreads();
    if (wave == 0) {
      int carry = 0;
      for (int e0 = 0; e0 < a.rows.experts; e0 += 64) {
        int v = e0 + lane < a.rows.experts ? tile_end[e0 + lane] : 0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          int const o = __shfl_up(v, off);
          if (lane >= off) v += o;
        }
        if (e0 + lane < a.rows.experts) tile_end[e0 + lane] = carry + v;
        carry += __shfl(v, 63);
      }
    }
    __syncthreads();
    total = tile_end[a.rows.experts - 1];
  }

  // Blocks are handed to the 8 XCDs in turn; each XCD gets a contiguous run
  // of tiles, so that the blocks that share an L2 share operands.
  int const per_xcd = (total + 7) / 8;
  int const xcd = blockIdx.x & 7;
  for (int i = blockIdx.x >> 3; i < per_xcd; i += gridDim.x >> 3) {
    int const tile = xcd * per_xcd + i;
    if (tile >= total) break;

    // --- which tile --------------------------------------------------------
    int e, local, tiles_q, valid;
    if constexpr (kWGrad) {
      tiles_q = (a.nq + BQ - 1) / BQ;
      e = tile / (tiles_p * tiles_q);
      local = tile % (tiles_p * tiles_q);
      valid = rows_of(a.rows, e);
    } else {
      int lo = 0, hi = a.rows.experts - 1;  // first e with tile < tile_end[e]
      while (lo < hi) {
        int const mid = (lo + hi) >> 1;
        if (tile < tile_end[mid]) hi = mid;
        else lo = mid + 1;
      }
      e = lo;
      int const begin = e ? tile_end[e - 1] : 0;
      local = tile - begin;
      tiles_q = (tile_end[e] - begin) / tiles_p;
      valid = rows_of(a.rows, e);
    }
    e = __builtin_amdgcn_readfirstlane(e);
    // four rows of tiles at a time, so that tiles near in order share both
    // operands
    int const band = local / (4 * tiles_p) * 4;
    int const in_band = local - band * tiles_p;
    int const high = min(4, tiles_q - band);
    int const q0 = (band + in_band % high) * BQ;
    int const p0 = in_band / high * BP;

    __syncthreads();  // slots and stages of the last tile are no longer read
    if constexpr (!kWGrad) {
      for (int j = threadIdx.x; j < BQ; j += kThreads)
        slots[j] = slot_of(a.rows, e, min(q0 + j, valid - 1));
    } else {
      if (threadIdx.x < kDepth && threadIdx.x < valid)
        slots[threadIdx.x] = slot_of(a.rows, e, threadIdx.x);
    }
    __syncthreads();

    // --- loads of a stage --------------------------------------------------
    char const* const pe = a.p + e * a.p_expert;
    char const* const qe = a.q + e * a.q_expert;
    int const depth = kWGrad ? valid : a.depth;
    int const steps = (depth + kDepth - 1) / kDepth;
    char const* const zeros = reinterpret_cast<char const*>(&zero_page);

    // Direct operand: a row of 128 bytes, 16-byte chunk c at place c ^ (row &
    // 7). Turned operand: a row of B * 2 bytes, chunk c at place c ^ turn(row).
    auto turn = [](int row) { return ((row & 3) | ((row >> 1) & 4)) << 1; };

    char const* p_at[kPLoads];
    char const* q_at[kQLoads];
#pragma unroll
    for (int j = 0; j < kPLoads; ++j) {
      int const at = (wave * kPLoads + j) * 64 + lane;
      if constexpr (!kPTurned) {
        int const row = at >> 3, c = (at & 7) ^ (row & 7);
        p_at[j] = pe + static_cast<int64_t>(min(p0 + row, a.np - 1)) * a.p_row +
                  c * 16;
      } else {
        int const row = at / (BP / 8), c = (at % (BP / 8)) ^ turn(row);
        // a chunk behind the last column gives results that are not stored
        int const col = min(p0 + c * 8, a.np - 8);
        p_at[j] = pe + static_cast<int64_t>(kWGrad ? 0 : row) * a.p_row +
                  static_cast<int64_t>(col) * 2;
      }
    }
#pragma unroll
    for (int j = 0; j < kQLoads; ++j) {
      int const at = (wave * kQLoads + j) * 64 + lane;
      if constexpr (!kQTurned) {
        int const row = at >> 3, c = (at & 7) ^ (row & 7);
        q_at[j] = qe + static_cast<int64_t>(slots[row]) * a.q_row + c * 16;
      } else {
        int const row = at / (BQ / 8), c = (at % (BQ / 8)) ^ turn(row);
        int const col = min(q0 + c * 8, a.nq - 8);
        q_at[j] = qe + static_cast<int64_t>(col) * 2;
      }
    }
    char const* s_at = nullptr;
    if constexpr (k8) {
      int const row = (wave % (BQ / 64)) * 64 + lane;
      s_at = a.q_scales + e * a.qs_expert +
             static_cast<int64_t>(slots[row]) * a.qs_row;
    }

    auto load_stage = [&](int step) {
      uint32_t const base = lds0 + (step & 1) * kStage;
#pragma unroll
      for (int j = 0; j < kPLoads; ++j) {
        int const at = (wave * kPLoads + j) * 64 + lane;
        char const* g;
        if constexpr (!kPTurned) {
          int const c = (at & 7) ^ ((at >> 3) & 7);
          int const left = a.depth * kSize - step * kStep - c * 16;
          g = left > 0 ? p_at[j] + static_cast<int64_t>(step) * kStep : zeros;
        } else {
          int const row = step * kDepth + at / (BP / 8);
          if constexpr (kWGrad)
            g = row < depth
                    ? p_at[j] + static_cast<int64_t>(
                                    slots[(step & 1) * kDepth +
                                          at / (BP / 8)]) *
                                    a.p_row
                    : zeros;
          else
            g = row < depth ? p_at[j] + static_cast<int64_t>(step) * kDepth *
                                            a.p_row
                            : zeros;
        }
        lds_load16(g, base + (wave * kPLoads + j) * 1024);
      }
#pragma unroll
      for (int j = 0; j < kQLoads; ++j) {
        int const at = (wave * kQLoads + j) * 64 + lane;
        char const* g;
        if constexpr (!kQTurned) {
          int const c = (at & 7) ^ ((at >> 3) & 7);
          int const left = a.depth * kSize - step * kStep - c * 16;
          g = left > 0 ? q_at[j] + static_cast<int64_t>(step) * kStep : zeros;
        } else {
          int const row = step * kDepth + at / (BQ / 8);
          g = row < depth
                  ? q_at[j] + static_cast<int64_t>(
                                  slots[(step & 1) * kDepth + at / (BQ / 8)]) *
                                  a.q_row
                  : zeros;
        }
        lds_load16(g, base + kPBytes + (wave * kQLoads + j) * 1024);
      }
      if constexpr (k8)
        lds_load4(s_at + static_cast<int64_t>(step) * 4,
                  base + kPBytes + kQBytes + (wave % (BQ / 64)) * 256);
    };

    // --- the product -------------------------------------------------------
    f32x4 acc[TP][TQ];
#pragma unroll
    for (int i2 = 0; i2 < TP; ++i2)
#pragma unroll
      for (int j = 0; j < TQ; ++j) acc[i2][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    float const* p_scale = nullptr;
    if constexpr (k8) {
      int const block =
          min(p0 + wp * (BP / WP), a.np - 1) / 128;  // uniform in a wave
      p_scale = reinterpret_cast<float const*>(
          a.p_scales + e * a.ps_expert + block * a.ps_row);
    }

    // Operand fragment of 16 rows (or columns) from `row0`: 16 bits, the
    // 32 contraction elements of half `h`; lane l has row l % 16, elements
    // (l / 16) * 8 on. Both operands use the same order of the contraction.
    auto direct16 = [&](char const* tile_at, int row0, int h) {
      int const row = row0 + (lane & 15);
      int const c = (h * 4 + (lane >> 4)) ^ (row & 7);
      return *reinterpret_cast<i32x4 const*>(tile_at + row * kStep + c * 16);
    };
    auto turned16 = [&](char const* tile_at, int width, int col0, int h) {
      i16x4 v[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        int const row = h * 32 + (lane >> 4) * 8 + g * 4 + ((lane >> 2) & 3);
        int const col = col0 + (lane & 3) * 4;
        int const c = (col >> 3) ^ turn(row);
        v[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)(
                tile_at + row * width * 2 + c * 16 + (col & 7) * 2));
      }
      i16x8 const both = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5,
                                                 6, 7);
      return __builtin_bit_cast(i32x4, both);
    };
    auto direct8 = [&](char const* tile_at, int row0) {
      int const row = row0 + (lane & 15);
      int const c = (lane >> 4) * 2;
      i32x4 const lo = *reinterpret_cast<i32x4 const*>(
          tile_at + row * kStep + ((c ^ (row & 7)) * 16));
      i32x4 const hi = *reinterpret_cast<i32x4 const*>(
          tile_at + row * kStep + (((c + 1) ^ (row & 7)) * 16));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    if (steps > 0) load_stage(0);
    for (int step = 0; step < steps; ++step) {
      if constexpr (kWGrad) {
        // slots of the next stage, behind the same barrier as its loads
        int const next = (step + 1) * kDepth + static_cast<int>(threadIdx.x);
        if (threadIdx.x < kDepth && next < depth)
          slots[((step + 1) & 1) * kDepth + threadIdx.x] =
              slot_of(a.rows, e, next);
      }
      stage_barrier();
      if (step + 1 < steps) load_stage(step + 1);
      char const* const pt = stages + (step & 1) * kStage;
      char const* const qt = pt + kPBytes;
      if constexpr (k8) {
        float const sw = p_scale[step];
        float const* const sx = reinterpret_cast<float const*>(qt + kQBytes);
        i32x8 pf[TP];
#pragma unroll
        for (int i2 = 0; i2 < TP; ++i2)
          pf[i2] = direct8(pt, wp * (BP / WP) + i2 * 16);
#pragma unroll
        for (int j = 0; j < TQ; ++j) {
          int const row = wq * (BQ / WQ) + j * 16;
          i32x8 const qf = direct8(qt, row);
          float const s = sx[row + (lane & 15)] * sw;
#pragma unroll
          for (int i2 = 0; i2 < TP; ++i2) {
            f32x4 const d = mfma8(pf[i2], qf);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i2][j][r] = fmaf(d[r], s, acc[i2][j][r]);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          i32x4 pf[TP];
#pragma unroll
          for (int i2 = 0; i2 < TP; ++i2) {
            int const at = wp * (BP / WP) + i2 * 16;
            pf[i2] = kPTurned ? turned16(pt, BP, at, h) : direct16(pt, at, h);
          }
#pragma unroll
          for (int j = 0; j < TQ; ++j) {
            int const at = wq * (BQ / WQ) + j * 16;
            i32x4 const qf =
                kQTurned ? turned16(qt, BQ, at, h) : direct16(qt, at, h);
#pragma unroll
            for (int i2 = 0; i2 < TP; ++i2)
              acc[i2][j] = mfma16<kElem>(pf[i2], qf, acc[i2][j]);
          }
        }
      }
    }

    // --- results -----------------------------------------------------------
    constexpr int kOutSize = kOut == Elem::kF32 ? 4 : 2;
    bool const wide = a.np % 4 == 0 && a.out_row % (4 * kOutSize) == 0 &&
                      a.out_expert % (4 * kOutSize) == 0 &&
                      reinterpret_cast<uintptr_t>(a.out) % (4 * kOutSize) == 0;
    int const end_q = kWGrad ? a.nq : valid;
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
      int const in_q = wq * (BQ / WQ) + j * 16 + (lane & 15);
      if (q0 + in_q >= end_q) continue;
      int64_t const row = kWGrad ? q0 + in_q : slots[in_q];
      char* const o = a.out + e * a.out_expert + row * a.out_row;
#pragma unroll
      for (int i2 = 0; i2 < TP; ++i2) {
        int const p = p0 + wp * (BP / WP) + i2 * 16 + (lane >> 4) * 4;
        if (p < a.np)
          store4<kOut>(o + static_cast<int64_t>(p) * kOutSize, acc[i2][j],
                       a.np - p, wide);
      }
    }
  }
}

int compute_units() {
  int dev = 0, n = 0;
  UCCL_CHECK_HIP(hipGetDevice(&dev));
  UCCL_CHECK_HIP(
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
  return n;
}

template <Mode kMode, Elem kElem, Elem kOut, int BP, int BQ, int WP, int WQ>
void launch_tiles(GemmArgs const& a, int blocks_per_cu, hipStream_t s) {
  int64_t const tiles_p = (a.np + BP - 1) / BP;
  int64_t const q = kMode == Mode::kWeightGrad
                        ? a.nq
                        : static_cast<int64_t>(a.rows.sources) * a.rows.length;
  int64_t const most = a.rows.experts * tiles_p * ((q + BQ - 1) / BQ);
  int64_t grid = std::min<int64_t>(most, compute_units() * blocks_per_cu);
  grid = (grid + 7) / 8 * 8;
  k_expert_gemm<kMode, kElem, kOut, BP, BQ, WP, WQ>
      <<<static_cast<int>(grid), WP * WQ * 64, 0, s>>>(a);
}

template <Mode kMode, Elem kElem, Elem kOut>
void launch_sized(GemmArgs const& a, int expected_rows, hipStream_t s) {
  int64_t const tiles = static_cast<int64_t>(a.rows.experts) *
                        ((a.np + 255) / 256) * ((expected_rows + 255) / 256);
  if (tiles >= compute_units())
    launch_tiles<kMode, kElem, kOut, 256, 256, 4, 2>(a, 1, s);
  else
    launch_tiles<kMode, kElem, kOut, 128, 128, 2, 2>(a, 2, s);
}

template <Mode kMode, Elem kElem>
void by_out(GemmArgs const& a, Elem out, int expected_rows, hipStream_t s) {
  if (out == Elem::kBF16)
    launch_sized<kMode, kElem, Elem::kBF16>(a, expected_rows, s);
  else if (out == Elem::kF16)
    launch_sized<kMode, kElem, Elem::kF16>(a, expected_rows, s);
  else if constexpr (kElem != Elem::kF8)
    launch_sized<kMode, kElem, Elem::kF32>(a, expected_rows, s);
}

}  // namespace

void launch_expert_matmul(MatmulArgs const& m, hipStream_t s) {
  int const size = m.elem == Elem::kF8 ? 1 : 2;
  int const out_size = m.out_elem == Elem::kF32 ? 4 : 2;
  GemmArgs a{};
  a.rows = m.rows;
  a.p = static_cast<char const*>(m.w.p);
  a.p_expert = m.w.expert_stride * size;
  a.p_row = m.w.row_stride * size;
  a.q = static_cast<char const*>(m.x.p);
  a.q_expert = m.x.expert_stride * size;
  a.q_row = m.x.row_stride * size;
  a.out = static_cast<char*>(m.out.p);
  a.out_expert = m.out.expert_stride * out_size;
  a.out_row = m.out.row_stride * out_size;
  a.np = m.n;
  a.depth = m.k;
  if (m.elem == Elem::kF8) {
    a.p_scales = static_cast<char const*>(m.w_scales.p);
    a.ps_expert = m.w_scales.expert_stride * 4;
    a.ps_row = m.w_scales.row_stride * 4;
    a.q_scales = static_cast<char const*>(m.x_scales.p);
    a.qs_expert = m.x_scales.expert_stride * 4;
    a.qs_row = m.x_scales.row_stride * 4;
    by_out<Mode::kProduct, Elem::kF8>(a, m.out_elem, m.expected_rows, s);
  } else if (m.elem == Elem::kBF16) {
    if (m.w_turned)
      by_out<Mode::kProductTurned, Elem::kBF16>(a, m.out_elem,
                                                m.expected_rows, s);
    else
      by_out<Mode::kProduct, Elem::kBF16>(a, m.out_elem, m.expected_rows, s);
  } else {
    if (m.w_turned)
      by_out<Mode::kProductTurned, Elem::kF16>(a, m.out_elem,
                                               m.expected_rows, s);
    else
      by_out<Mode::kProduct, Elem::kF16>(a, m.out_elem, m.expected_rows, s);
  }
}

void launch_expert_weight_grad(WeightGradArgs const& w, hipStream_t s) {
  int const out_size = w.out_elem == Elem::kF32 ? 4 : 2;
  GemmArgs a{};
  a.rows = w.rows;
  a.p = static_cast<char const*>(w.x.p);
  a.p_expert = w.x.expert_stride * 2;
  a.p_row = w.x.row_stride * 2;
  a.q = static_cast<char const*>(w.grad.p);
  a.q_expert = w.grad.expert_stride * 2;
  a.q_row = w.grad.row_stride * 2;
  a.out = static_cast<char*>(w.out.p);
  a.out_expert = w.out.expert_stride * out_size;
  a.out_row = w.out.row_stride * out_size;
  a.np = w.k;
  a.nq = w.n;
  if (w.elem == Elem::kBF16)
    by_out<Mode::kWeightGrad, Elem::kBF16>(a, w.out_elem, w.n, s);
  else
    by_out<Mode::kWeightGrad, Elem::kF16>(a, w.out_elem, w.n, s);
}

}  // namespace ep
}  // namespace uccl
