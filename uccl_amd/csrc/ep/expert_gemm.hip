// The experts' matrix products over slot arrays, and their weight gradient.
//
//   product        y[m, n]  = sum_k x[m, k] w[n, k]
//     8 bit:       y[m, n]  = sum_b sx[m, b] sw[n / 128, b]
//                             sum_{k in block b} qx[m, k] qw[n, k]
//   turned weights (k and n swapped in memory) give the rows' gradient
//   weight gradient  dw[n, k] = sum_m g[m, n] x[m, k], over the valid rows
//
// One kernel computes D[p, q] = sum_c P[p, c] Q[q, c] tile by tile with MFMA
// 16x16 instructions; a lane then holds consecutive p of one q, so p is the
// contiguous dimension of the result: P = w, Q = x for a product, P = x^T,
// Q = g^T for the weight gradient.
//
// A tile's operands go from memory to LDS in steps of 128 bytes (direct
// operands, contiguous along c) or 64 rows (turned operands, contiguous along
// p or q; read back through the transposing LDS load), in two stages, by
// loads that write LDS without passing registers. Each lane forms its own
// address, so the valid rows of all sources are gathered on the way: a tile
// is full of valid rows wherever they lie.
//
// Rows behind an expert's last are never read: tiles are cut from the number
// of valid rows, lanes behind the last row load it again, and lanes behind
// the end of the contraction load from a page of zeros.
//
// What bounds a large product is LDS: a step of a 256 x 256 tile brings 64 KB
// in and gives 192 KB to the waves, 2048 clocks of the 128 bytes it moves in
// each, and the same 2048 clocks the matrix units are busy. 16384 rows of 8
// experts, bf16, calls in a stream on several cards, the slowest of which is 7%
// behind the fastest: product 7168 x 4096 805 us, 1.20 PFLOP/s, its row
// gradient 815 to 885 us, weight gradient 4096 x 7168 865 to 924 us, 1.04 to
// 1.11 PFLOP/s; 32768 rows, 4096 x 7168, 8 bits: 906 to 969 us, 1.99 to 2.12
// PFLOP/s. (The library reaches 1.40 and 2.73 on dense products of 8192 cubed,
// on the fastest 1.55 and 3.10.) Products of few rows are bound by the
// weights' bytes: 1024 rows of 32 experts, 4096 x 7168, 8 bits: 175 to 179 us,
// 5.4 TB/s, bf16: 322 us, 5.9 TB/s.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../core/log.h"
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
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;  // bytes of the contraction in a stage, a row

// 16 bytes of zeros: where lanes behind the contraction's end load from.
__device__ const int4 zero_page = {0, 0, 0, 0};

// --- loads to LDS ----------------------------------------------------------
// Each lane loads 16 bytes from its own address to LDS at `lds` + lane * 16;
// load n of a group to n KiB behind that, and n KiB behind its offset.
// Where `on` is 0 it loads nothing. The branch is inside the statement so that
// it does not cut the block that the compiler schedules.
#define LDS_LOAD_GROUP(loads, last, ...)                                      \
  asm volatile("s_cmp_eq_u32 %1, 0\n\ts_cbranch_scc1 1f\n\t"                  \
               "s_mov_b32 m0, %2\n\ts_nop 0\n\t" loads "\n1:"                 \
               :                                                              \
               : "s"(base), "s"(on), "s"(lds), "n"(last), __VA_ARGS__         \
               : "memory", "m0", "scc")
template <int kCount>
__device__ __forceinline__ void lds_load_group(int on, char const* base,
                                               uint32_t const* off,
                                               uint32_t lds) {
  static_assert(kCount == 1 || kCount == 2 || kCount == 4, "loads of a group");
  if constexpr (kCount == 1)
    LDS_LOAD_GROUP("global_load_lds_dwordx4 %4, %0", 0, "v"(off[0]));
  else if constexpr (kCount == 2)
    LDS_LOAD_GROUP(
        "global_load_lds_dwordx4 %4, %0\n\t"
        "global_load_lds_dwordx4 %5, %0 offset:%3",
        1024, "v"(off[0]), "v"(off[1]));
  else
    LDS_LOAD_GROUP(
        "global_load_lds_dwordx4 %4, %0\n\t"
        "global_load_lds_dwordx4 %5, %0 offset:1024\n\t"
        "global_load_lds_dwordx4 %6, %0 offset:2048\n\t"
        "global_load_lds_dwordx4 %7, %0 offset:%3",
        3 * 1024, "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]));
}
#undef LDS_LOAD_GROUP
__device__ __forceinline__ void lds_load16(char const* g, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
      :
      : "v"(g), "s"(lds)
      : "memory", "m0");
}
// 4 bytes a lane, where `on` is not 0.
__device__ __forceinline__ void lds_load4(int on, char const* g,
                                          uint32_t lds) {
  asm volatile(
      "s_cmp_eq_u32 %2, 0\n\ts_cbranch_scc1 1f\n\ts_mov_b32 m0, %1\n\t"
      "s_nop 0\n\tglobal_load_lds_dword %0, off\n1:"
      :
      : "v"(g), "s"(lds), "s"(on)
      : "memory", "m0", "scc");
}

// This wave's LDS reads are done and its loads and stores have landed, all
// but the last `left` (0, kMore or kMost; uniform); and so for the other waves
// of the block.
template <int kMore, int kMost>
__device__ __forceinline__ void stage_barrier(int left) {
  asm volatile(
      "s_cmp_lt_i32 %2, %1\n\ts_cbranch_scc0 2f\n\t"
      "s_cmp_lt_i32 %2, %0\n\ts_cbranch_scc0 1f\n\t"
      "s_waitcnt vmcnt(0)\n1:\n\ts_waitcnt vmcnt(%0)\n2:\n\t"
      "s_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_barrier" ::"n"(kMore),
      "n"(kMost), "s"(left)
      : "memory", "scc");
}

__device__ __forceinline__ uint32_t lds_addr(void const* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)p));
}
template <typename T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *reinterpret_cast<__attribute__((address_space(3))) T const*>(at);
}
__device__ __forceinline__ i16x4 lds_read_turned(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      reinterpret_cast<__attribute__((address_space(3))) i16x4*>(at));
}

__device__ __forceinline__ int uniform(int v) {
  return __builtin_amdgcn_readfirstlane(v);
}

// -1 where a < b, else 0, for uniform operands: a condition that stays in
// scalar registers, where the statements above want it.
__device__ __forceinline__ int before(int a, int b) {
  int r;
  asm("s_cmp_lt_i32 %1, %2\n\ts_cselect_b32 %0, -1, 0"
      : "=s"(r)
      : "s"(a), "s"(b)
      : "scc");
  return r;
}

template <int kAt, int kEnd, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (kAt < kEnd) {
    f(std::integral_constant<int, kAt>{});
    unrolled<kAt + 1, kEnd>(f);
  }
}

struct GemmArgs {
  SlotRows rows;
  char const* p;
  char const* q;
  char* out;
  // bytes
  int64_t p_expert, p_row, q_expert, q_row, out_expert, out_row;
  int np;     // extent of p
  int nq;     // extent of q (weight gradient only; else the valid rows)
  int depth;  // contraction in elements (product only)
  bool near;  // a lane's addresses in a stage lie within 32 bits
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

// The sum of 128 products of 8 bits. The unit aligns the products to the
// largest before it adds them and drops what lies below: on bytes of all
// magnitudes that costs up to 8.4e-5 of sum |products|, on normal data 1.4e-5
// of the result, whichever of its 8-bit instructions is used. It is taken all
// the same where the caller does not ask for more: results have 16 bits, whose
// own rounding is 3 times that (float16, such bytes) to 140 times (bfloat16,
// normal data), and sums of 32 bits (Sums::k32) take the product of 32768 rows
// from 903 to 1717 us.
__device__ __forceinline__ f32x4 mfma8(i32x8 a, i32x8 b) {
  f32x4 const zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0,
                                                          0, 0, 0);
}

// 8-bit values in 16 bits, which hold them exactly, four lots of 8: the same
// sum in 32 bits. Any order of the values serves that both operands share.
struct Wide {
  i32x4 v[4];
};
__device__ __forceinline__ Wide widened(i32x8 r) {
  Wide w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w.v[i / 2][i % 2 * 2] = __builtin_bit_cast(
        int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r[i], 1.f, false));
    w.v[i / 2][i % 2 * 2 + 1] = __builtin_bit_cast(
        int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r[i], 1.f, true));
  }
  return w;
}
__device__ __forceinline__ f32x4 mfma_wide(Wide const& a, Wide const& b) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) d = mfma16<Elem::kF16>(a.v[i], b.v[i], d);
  return d;
}

// How the sum over a block of 128 8-bit values is held.
enum class Sums { kUnit, k32 };

template <Elem kOut>
using OutType = std::conditional_t<
    kOut == Elem::kF32, float,
    std::conditional_t<kOut == Elem::kBF16, __bf16, _Float16>>;

// Store 8 results of a row, or the first n of them. 16 bytes at a time at any
// address: this target allows it, and a row of odd length starts anywhere.
template <Elem kOut>
__device__ __forceinline__ void store8(char* at, f32x4 a, f32x4 b) {
  using T = OutType<kOut>;
  T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = static_cast<T>(j < 4 ? a[j % 4] : b[j % 4]);
  __builtin_memcpy(at, v, sizeof(v));
}
template <Elem kOut>
__device__ __forceinline__ void store_few(char* at, f32x4 a, f32x4 b, int n) {
  using T = OutType<kOut>;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n)
      reinterpret_cast<T*>(at)[j] = static_cast<T>(j < 4 ? a[j % 4] : b[j % 4]);
}

// --- the valid rows of all experts, in LDS ---------------------------------
struct RowTable {
  int end[kMaxSlotCells];        // [expert][source]: valid rows up to there
  int tile_end[kMaxSlotExperts];  // tiles of rows up to and with the expert
};

__device__ __forceinline__ void fill_table(RowTable& t, SlotRows const& r,
                                           int tile_rows) {
  int const cells = r.experts * r.sources;
  for (int i = threadIdx.x; i < cells; i += blockDim.x)
    t.end[i] = r.counts ? min(max(r.counts[i], 0), r.length) : r.length;
  __syncthreads();
  for (int e = threadIdx.x; e < r.experts; e += blockDim.x) {
    int n = 0;
    for (int s = 0; s < r.sources; ++s) {
      n += t.end[e * r.sources + s];
      t.end[e * r.sources + s] = n;
    }
    t.tile_end[e] = (n + tile_rows - 1) / tile_rows;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    int const lane = threadIdx.x;
    int carry = 0;
    for (int e0 = 0; e0 < r.experts; e0 += 64) {
      int v = e0 + lane < r.experts ? t.tile_end[e0 + lane] : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        int const o = __shfl_up(v, off);
        if (lane >= off) v += o;
      }
      if (e0 + lane < r.experts) t.tile_end[e0 + lane] = carry + v;
      carry += __shfl(v, 63);
    }
  }
  __syncthreads();
}

__device__ __forceinline__ int valid_rows(RowTable const& t, SlotRows const& r,
                                          int e) {
  return t.end[(e + 1) * r.sources - 1];
}

// Slot of the i-th valid row of expert e, i below valid_rows().
__device__ __forceinline__ int slot_of(RowTable const& t, SlotRows const& r,
                                       int e, int i) {
  int begin = 0;
  for (int s = 0; s < r.sources; ++s) {
    int const end = t.end[e * r.sources + s];
    if (i < end) return s * r.length + i - begin;
    begin = end;
  }
  return 0;
}

struct Tile {
  int e, p0, q0;
  int valid;  // rows of the expert
};

// Tiles are counted expert by expert; in an expert, four rows of tiles at a
// time, so that tiles near in order share both operands.
template <Mode kMode, int BP, int BQ>
__device__ __forceinline__ Tile find_tile(GemmArgs const& a,
                                          RowTable const& t, int tile,
                                          int tiles_p) {
  int e, local, tiles_q;
  if constexpr (kMode == Mode::kWeightGrad) {
    tiles_q = (a.nq + BQ - 1) / BQ;
    e = tile / (tiles_p * tiles_q);
    local = tile - e * tiles_p * tiles_q;
  } else {
    int const row = tile / tiles_p;  // counted over all experts
    int lo = 0, hi = a.rows.experts - 1;  // first e with row < tile_end[e]
    while (lo < hi) {
      int const mid = (lo + hi) >> 1;
      if (row < t.tile_end[mid]) hi = mid;
      else lo = mid + 1;
    }
    e = lo;
    int const begin = e ? t.tile_end[e - 1] : 0;
    tiles_q = t.tile_end[e] - begin;
    local = tile - begin * tiles_p;
  }
  int const band = local / (4 * tiles_p) * 4;
  int const in_band = local - band * tiles_p;
  int const high = min(4, tiles_q - band);
  Tile r;
  r.e = uniform(e);
  r.q0 = uniform((band + in_band % high) * BQ);
  r.p0 = uniform(in_band / high * BP);
  r.valid = uniform(valid_rows(t, a.rows, e));
  return r;
}

template <int kH>
__device__ __forceinline__ i32x4 half(i32x8 v) {
  return __builtin_shufflevector(v, v, kH * 4, kH * 4 + 1, kH * 4 + 2,
                                 kH * 4 + 3);
}

// Tiles BP x BQ, WP x WQ waves of TP x TQ MFMA tiles, two stages.
//
// Places in LDS. Direct operands: a row of 128 bytes, its 16-byte chunk c at
// place c ^ f(row), f taken from the row bits in which the 16 rows that a wave
// reads together differ, so that these reads fall into different banks. Turned
// operands: a row of the contraction, chunk c at place c ^ ((row & 3) << 2).
// Q comes in two halves, of the first and the last half of each wave's rows.
//
// P rows are given to MFMA rows so that a lane's results of two tiles are 8
// consecutive p: row m of tile i is p = 32 (i / 2) + 8 (m / 4) + 4 (i % 2) +
// m % 4 of the wave's 64.
template <Mode kMode, Elem kElem, Elem kOut, int BP, int BQ, int WP, int WQ,
          bool kFar, Sums kSums>
__global__ __launch_bounds__(WP* WQ * 64, 2) void k_expert_gemm(GemmArgs a) {
  constexpr bool kWGrad = kMode == Mode::kWeightGrad;
  constexpr bool kPTurned = kMode != Mode::kProduct;
  constexpr bool kQTurned = kWGrad;
  constexpr bool k8 = kElem == Elem::kF8;
  constexpr bool kWide = k8 && kSums == Sums::k32;
  constexpr int kSize = k8 ? 1 : 2;
  constexpr int kDepth = kStep / kSize;  // contraction elements of a stage
  constexpr int kWaves = WP * WQ, kThreads = kWaves * 64;
  constexpr int RP = BP / WP, RQ = BQ / WQ;  // rows of a wave
  constexpr int TP = RP / 16, TQ = RQ / 16, kT = TP * TQ;
  constexpr int kPBytes = BP * kStep, kQBytes = BQ * kStep;
  constexpr int kStage = kPBytes + kQBytes;
  constexpr int kPLoads = kPBytes / 1024 / kWaves;  // of a wave and stage
  constexpr int kQLoads = kQBytes / 1024 / kWaves;
  constexpr int kHalf = kQLoads / 2;
  constexpr int kLoads = kPLoads + kQLoads;
  static_assert(kPLoads * 1024 * kWaves == kPBytes, "P loads");
  static_assert(kHalf * 2048 * kWaves == kQBytes, "Q loads");
  constexpr int kOutSize = kOut == Elem::kF32 ? 4 : 2;
  constexpr int kStores = kT * kOutSize / 4;  // of a whole tile
  static_assert(kLoads + kStores < 64, "vmcnt");
  static_assert(TP == 4 && TQ % 4 == 0, "places and stores");
  static_assert(!k8 || (128 % RP == 0 && BQ <= kThreads), "scales");
  // turned rows
  constexpr int kPPitch = BP * 2, kQPitch = BQ;

  __shared__ __attribute__((aligned(1024))) char stages[2 * kStage];
  __shared__ float q_scale[k8 ? 4 : 1][k8 ? BQ : 1];
  __shared__ float p_scale[k8 ? 4 : 1][k8 ? 64 : 1];
  __shared__ RowTable table;
  // rows of a tile: of the last, whose results are stored, of this one and of
  // the next; weight gradient: rows of a stage, kNoted stages in a ring
  constexpr int kNoted = 8;
  __shared__ int slots[kWGrad ? kNoted : 3][kWGrad ? kDepth : BQ];
  __shared__ uint32_t p_rows[kWGrad ? kNoted : 1][kWGrad ? kDepth : 1];
  __shared__ uint32_t q_rows[kWGrad ? kNoted : 1][kWGrad ? kDepth : 1];

  int const wave = uniform(threadIdx.x >> 6);
  int const lane = threadIdx.x & 63;
  int const wp = wave % WP, wq = wave / WP;
  uint32_t const lds0 = lds_addr(stages);

  int const tiles_p = (a.np + BP - 1) / BP;
  fill_table(table, a.rows, kWGrad ? 1 : BQ);
  int const total =
      uniform(kWGrad ? a.rows.experts * tiles_p * ((a.nq + BQ - 1) / BQ)
                     : table.tile_end[a.rows.experts - 1] * tiles_p);
  // Blocks are handed to the 8 XCDs in turn. Each round of tiles, the last one
  // too, is cut into one run for each XCD, so that the blocks that share an L2
  // share operands, all XCDs have work, and all of the card works on
  // neighbouring tiles, whose operands stay in the last-level cache.
  auto tile_of = [&](int first) {  // of the round that begins there, or total
    int const round = min(total - first, static_cast<int>(gridDim.x));
    int const run = (round + 7) >> 3, i = blockIdx.x >> 3;
    int const t = (blockIdx.x & 7) * run + i;
    return i < run && t < round ? first + t : total;
  };
  int first = 0, tile = tile_of(0);
  if (tile >= total) return;

  // --- this lane's part of the loads ---------------------------------------
  // P: loads wave * kPLoads on of the stage's; Q: wave * kHalf on of a half's.
  auto p_row = [&](int j) {
    int const at = (wave * kPLoads + j) * 64 + lane;
    return kPTurned ? at / (kPPitch / 16) : at >> 3;
  };
  auto p_chunk = [&](int j) {
    int const at = (wave * kPLoads + j) * 64 + lane, row = p_row(j);
    if (kPTurned) return (at % (kPPitch / 16)) ^ ((row & 3) << 2);
    return (at & 7) ^ (((row >> 1) & 1) | (((row >> 3) & 3) << 1));
  };
  auto q_row = [&](int j) {  // in the half
    int const at = (wave * kHalf + j % kHalf) * 64 + lane;
    return kQTurned ? at / (kQPitch / 16) : at >> 3;
  };
  auto q_chunk = [&](int j) {
    int const at = (wave * kHalf + j % kHalf) * 64 + lane, row = q_row(j);
    if (kQTurned)
      return (at % (kQPitch / 16)) ^ (((row & 3) << 2) & (kQPitch / 16 - 1));
    return (at & 7) ^ ((row >> 1) & 7);
  };
  char const* const zeros = reinterpret_cast<char const*>(&zero_page);
  // row (or column) of the tile that place r of half h belongs to
  auto q_of = [&](int h, int r) {
    return r / (RQ / 2) * RQ + h * (RQ / 2) + r % (RQ / 2);
  };

  // Of the tile that is loaded. Loads of whole stages take 32-bit offsets from
  // a base that moves along the contraction. Up to four loads share an LDS
  // address: load n of a group lands n KiB behind it, and reads n KiB behind
  // its offset, which is that much lower; kBias keeps it above 0.
  constexpr uint32_t kBias = 4096;
  constexpr int kGroup = kPLoads / 2;
  Tile from{};
  int from_turn = 0;
  char const* p_base = nullptr;
  char const* q_base = nullptr;
  uint32_t p_off[kPLoads], q_off[kQLoads];
  char const* scale_at = nullptr;
  int steps = 0, whole = 0, depth = 0;

  // offsets of a tile's first stage
  auto set_tile = [&](Tile const& t, int turn) {
    from = t;
    from_turn = turn;
    depth = kWGrad ? t.valid : a.depth;
    steps = uniform((depth + kDepth - 1) / kDepth);
    whole = uniform(a.near ? depth / kDepth : 0);
    p_base = a.p + t.e * a.p_expert - kBias;
    p_base += kPTurned ? static_cast<int64_t>(t.p0) * 2
                       : static_cast<int64_t>(t.p0) * a.p_row;
    q_base = a.q + t.e * a.q_expert - kBias;
    if constexpr (kQTurned) q_base += static_cast<int64_t>(t.q0) * 2;
    uint32_t const p_pitch = static_cast<uint32_t>(a.p_row);
    uint32_t const q_pitch = static_cast<uint32_t>(a.q_row);
#pragma unroll
    for (int j = 0; j < kPLoads; ++j) {
      uint32_t const at = kBias - j % kGroup * 1024;
      if constexpr (!kPTurned)
        p_off[j] = min(p_row(j), a.np - 1 - t.p0) * p_pitch + p_chunk(j) * 16 +
                   at;
      else  // columns behind the last give results that are not stored
        p_off[j] = (kWGrad ? 0 : p_row(j) * p_pitch) +
                   min(p_chunk(j) * 8, a.np - 8 - t.p0) * 2 + at;
    }
#pragma unroll
    for (int j = 0; j < kQLoads; ++j) {
      uint32_t const at = kBias - j % kHalf * 1024;
      if constexpr (!kQTurned)
        q_off[j] = slots[turn][q_of(j / kHalf, q_row(j))] * q_pitch +
                   q_chunk(j) * 16 + at;
      else
        q_off[j] = min(q_of(j / kHalf, q_chunk(j) * 8), a.nq - 8 - t.q0) * 2 +
                   at;
    }
    if constexpr (k8) {
      if (wave < BQ / 64) {
        scale_at = a.q_scales + t.e * a.qs_expert +
                   static_cast<int64_t>(slots[turn][threadIdx.x % BQ]) *
                       a.qs_row;
      } else {
        int const block =
            min(t.p0 + min(lane, BP / 128 - 1) * 128, a.np - 1) / 128;
        scale_at = a.p_scales + t.e * a.ps_expert + block * a.ps_row;
      }
    }
  };

  uint32_t const my_p = lds0 + wave * kPLoads * 1024;
  uint32_t const my_q = lds0 + kPBytes + wave * kHalf * 1024;
  // Weight gradient: where a stage's rows begin.
  uint32_t p_at[kWGrad ? kPLoads : 1], q_at[kWGrad ? kQLoads : 1];
  auto find_rows = [&](int step) __attribute__((always_inline)) {
    if constexpr (kWGrad) {
#pragma unroll
      for (int j = 0; j < kPLoads; ++j)
        p_at[j] = p_off[j] + p_rows[step % kNoted][p_row(j)];
#pragma unroll
      for (int j = 0; j < kQLoads; ++j)
        q_at[j] = q_off[j] + q_rows[step % kNoted][q_row(j)];
    }
  };
  // Loads of stage `step`: parts 0 and 1 are P, 2 and 3 the halves of Q.
  // Barriers count on this order.
  auto load_near = [&](auto n, int on, int step)
                       __attribute__((always_inline)) {
    constexpr int part = decltype(n)::value;
    uint32_t const buf = (step & 1) * kStage;
    if constexpr (part < 2) {
      uint32_t const* const off = kWGrad ? p_at : p_off;
      lds_load_group<kGroup>(on, p_base, off + part * kGroup,
                             my_p + buf + part * kGroup * 1024);
      if constexpr (part == 1 && !kPTurned) p_base += kStep;
      if constexpr (part == 1 && kPTurned && !kWGrad)
        p_base += kDepth * a.p_row;
    } else {
      uint32_t const* const off = kWGrad ? q_at : q_off;
      lds_load_group<kHalf>(on, q_base, off + (part - 2) * kHalf,
                            my_q + buf + (part - 2) * (kQBytes / 2));
      if constexpr (part == 3 && !kQTurned) q_base += kStep;
    }
  };
  auto load_part = [&](auto n, int step) __attribute__((always_inline)) {
    constexpr int part = decltype(n)::value;
    static_assert(part >= 0 && part < 4);
    uint32_t const buf = (step & 1) * kStage;
    if constexpr (k8 && !kFar) {  // all stages are whole
      load_near(n, before(step, steps), step);
    } else if (!kFar && step < whole) {
      load_near(n, -1, step);
    } else if (step < steps) {
      // A stage that the contraction ends in, or rows too far apart: full
      // addresses, zeros behind the end. The rows of a weight gradient often
      // have few stages, so its loads go out together.
      auto row_at = [&](char const* base, int64_t row, int64_t pitch) {
        return base + row * pitch;
      };
      char const* const pe = a.p + from.e * a.p_expert;
      char const* const qe = a.q + from.e * a.q_expert;
      int64_t const along = static_cast<int64_t>(step) * kStep;
#pragma unroll(kWGrad ? 4 : 1)
      for (int n = 0; n < (part < 2 ? kGroup : kHalf); ++n) {
        int const j = part < 2 ? part * kGroup + n : n;
        int const row = part < 2 ? p_row(j) : q_row(j);
        int const chunk = part < 2 ? p_chunk(j) : q_chunk(j);
        bool const turned_in = step * kDepth + row < depth;
        bool const direct_in = step * kStep + chunk * 16 < depth * kSize;
        char const* g;
        if constexpr (part < 2 && !kPTurned)
          g = row_at(pe, min(from.p0 + row, a.np - 1), a.p_row) + along +
              chunk * 16;
        else if constexpr (part < 2)
          g = row_at(pe,
                     kWGrad ? slots[step % kNoted][row] : step * kDepth + row,
                     a.p_row) +
              min(from.p0 + chunk * 8, a.np - 8) * 2;
        else if constexpr (!kQTurned)
          g = row_at(qe, slots[from_turn][q_of(part - 2, row)], a.q_row) +
              along + chunk * 16;
        else
          g = row_at(qe, slots[step % kNoted][row], a.q_row) +
              min(from.q0 + q_of(part - 2, chunk * 8), a.nq - 8) * 2;
        bool const in =
            (part < 2 ? kPTurned : kQTurned) ? turned_in : direct_in;
        uint32_t const to = part < 2 ? my_p : my_q + (part - 2) * (kQBytes / 2);
        lds_load16(in ? g : zeros, uniform(to + buf + j * 1024));
      }
    }
  };
  // A step's scales, 4 steps in a ring: the first BQ / 64 waves load those of
  // Q, the next one those of the tile's blocks of P.
  static_assert(!k8 || BQ / 64 < kWaves, "a wave for the scales of P");
  uint32_t const my_s =
      wave < BQ / 64 ? lds_addr(q_scale) + wave * 256 : lds_addr(p_scale);
  uint32_t const s_pitch = wave < BQ / 64 ? BQ * 4 : 256;
  auto load_scales = [&](int on, int step) __attribute__((always_inline)) {
    if constexpr (k8) {
      lds_load4(on & before(wave, BQ / 64 + 1), scale_at,
                uniform(my_s + (step & 3) * s_pitch));
      scale_at += 4;
    }
  };
  // Weight gradient: the first wave notes the slots of a stage's rows.
  int seg = 0, seg_begin = 0, seg_end = 0;
  auto note_slots = [&](Tile const& t, int step) {
    if constexpr (kWGrad) {
      if (threadIdx.x < kDepth) {
        int const i = step * kDepth + threadIdx.x;
        if (step == 0) {
          seg = 0;
          seg_begin = 0;
          seg_end = table.end[t.e * a.rows.sources];
        }
        if (i < t.valid) {
          while (i >= seg_end) {  // ends: the last end is t.valid
            ++seg;
            seg_begin = seg_end;
            seg_end = table.end[t.e * a.rows.sources + seg];
          }
          uint32_t const slot = seg * a.rows.length + i - seg_begin;
          slots[step % kNoted][threadIdx.x] = slot;
          p_rows[step % kNoted][threadIdx.x] =
              slot * static_cast<uint32_t>(a.p_row);
          q_rows[step % kNoted][threadIdx.x] =
              slot * static_cast<uint32_t>(a.q_row);
        }
      }
    }
  };
  auto note_rows = [&](Tile const& t, int turn) {
    if constexpr (!kWGrad)
      for (int j = threadIdx.x; j < BQ; j += kThreads)
        slots[turn][j] =
            slot_of(table, a.rows, t.e, min(t.q0 + j, t.valid - 1));
  };
  // The first two stages of a tile whose rows are noted.
  auto begin_tile = [&](Tile const& t, int turn) {
    if constexpr (kWGrad) {
      for (int step = 0; step < 3; ++step) note_slots(t, step);
    }
    // slots are noted, and nobody reads the stages any more
    stage_barrier<kLoads, kLoads + kStores>(0);
    set_tile(t, turn);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      int const on = before(step, steps);
      find_rows(step);
      unrolled<0, 3>([&](auto n) { load_part(n, step); });
      load_scales(on, step);
      load_part(std::integral_constant<int, 3>{}, step);
    }
  };

  // --- this lane's part of the LDS reads -----------------------------------
  // direct: chunks l / 16 and 4 + l / 16 of its row; turned: see turned()
  uint32_t p_lo, p_hi, q_lo, q_hi;
  {
    int const m = lane & 15, g = lane >> 4, r = (lane >> 2) & 3;
    if constexpr (!kPTurned) {
      int const row = wp * RP + (m >> 2) * 8 + (m & 3);
      int const f = ((row >> 1) & 1) | (((row >> 3) & 3) << 1);
      p_lo = lds0 + row * kStep + ((g ^ f) * 16);
      p_hi = lds0 + row * kStep + (((4 + g) ^ f) * 16);
    } else {
      int const c = wp * (RP / 8) + (lane & 3);
      p_lo = lds0 + (g * 8 + r) * kPPitch + ((c ^ (r << 2)) * 16);
      p_hi = lds0 + (g * 8 + r) * kPPitch + (((c + 4) ^ (r << 2)) * 16);
    }
    uint32_t const q = lds0 + kPBytes;
    if constexpr (!kQTurned) {
      int const row = wq * (RQ / 2) + m;
      int const f = (row >> 1) & 7;
      q_lo = q + row * kStep + ((g ^ f) * 16);
      q_hi = q + row * kStep + (((4 + g) ^ f) * 16);
    } else {
      constexpr int kMask = kQPitch / 16 - 1;
      int const c = wq * (RQ / 16) + (lane & 3);
      q_lo = q + (g * 8 + r) * kQPitch + ((c ^ ((r << 2) & kMask)) * 16);
      q_hi = q + (g * 8 + r) * kQPitch + (((c + 4) ^ ((r << 2) & kMask)) * 16);
    }
  }
  auto direct = [](uint32_t lo, uint32_t hi) {
    i32x4 const x = lds_read<i32x4>(lo), y = lds_read<i32x4>(hi);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // 16 columns of a turned operand: 64 elements of the contraction, 8 of each
  // half for a lane
  auto turned = [](uint32_t at, int pitch) {
    i16x4 const v0 = lds_read_turned(at);
    i16x4 const v1 = lds_read_turned(at + 4 * pitch);
    i16x4 const v2 = lds_read_turned(at + 32 * pitch);
    i16x4 const v3 = lds_read_turned(at + 36 * pitch);
    i32x4 const x = __builtin_bit_cast(
        i32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    i32x4 const y = __builtin_bit_cast(
        i32x4, __builtin_shufflevector(v2, v3, 0, 1, 2, 3, 4, 5, 6, 7));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  i32x8 pf[TP], qf[2];
  [[maybe_unused]] Wide pw[TP], qw;  // of this step, of this column
  float s[2];
  uint32_t const s_at = lds_addr(q_scale) + (wq * RQ + (lane & 15)) * 4;
  auto read_p = [&](int step, int i) __attribute__((always_inline)) {
    uint32_t const buf = (step & 1) * kStage;
    if constexpr (!kPTurned) {
      uint32_t const at = buf + ((i >> 1) * 32 + (i & 1) * 4) * kStep;
      pf[i] = direct(p_lo + at, p_hi + at);
    } else {
      pf[i] = turned((i >> 1 ? p_hi : p_lo) + buf + (i & 1) * 8, kPPitch);
    }
  };
  auto read_q = [&](int step, int j) __attribute__((always_inline)) {
    uint32_t const buf = (step & 1) * kStage + (j >= TQ / 2) * (kQBytes / 2);
    int const i = j % (TQ / 2);
    if constexpr (!kQTurned) {
      qf[j & 1] = direct(q_lo + buf + i * 16 * kStep,
                         q_hi + buf + i * 16 * kStep);
    } else {
      qf[j & 1] = turned((i >> 1 ? q_hi : q_lo) + buf + (i & 1) * 8, kQPitch);
    }
  };
  auto read_s = [&](int step, int j) __attribute__((always_inline)) {
    if constexpr (k8)
      s[j & 1] = lds_read<float>(s_at + (step & 3) * (BQ * 4) + j * 64);
  };

  Tile now = find_tile<kMode, BP, BQ>(a, table, tile, tiles_p);
  note_rows(now, 0);
  begin_tile(now, 0);
  // What may be in flight behind the loads that a barrier waits for: a stage's
  // loads, and for the first step and a half of a tile the stores of a whole
  // tile before it.
  int left = kLoads;
  for (int turn = 0;;) {
    f32x4 acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
      for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The next tile is looked up while the first stage is on its way.
    Tile const done = now;
    int const next_turn = turn < 2 ? turn + 1 : 0;
    first += gridDim.x;
    tile = tile_of(first);
    bool const more = tile < total;
    if (more) {
      now = find_tile<kMode, BP, BQ>(a, table, tile, tiles_p);
      note_rows(now, next_turn);
    }
    // Behind the first stage's loads: the second's, and the last tile's stores.
    stage_barrier<kLoads, kLoads + kStores>(before(1, steps) & left);
    read_q(0, 0);
    read_s(0, 0);
#pragma unroll
    for (int i = 0; i < TP; ++i) read_p(0, i);
    f32x4 d[4];
    d[2] = d[3] = f32x4{0.f, 0.f, 0.f, 0.f};
    s[1] = 0.f;

    for (int step = 0; step < steps; ++step) {
      float sw = 0.f;
      if constexpr (k8)
        sw = lds_read<float>(lds_addr(p_scale) + (step & 3) * 256 +
                             wp * RP / 128 * 4);
      int const on = before(step + 2, steps);
      note_slots(done, step + 3);
      find_rows(step + 2);
      // Twice in a step, when all waves have read what lies in P and the
      // first half of Q, and in the second, the loads of the stage after
      // next take their places; so loads have a step and a half to land.
      constexpr int kMid = (TQ / 2 - 1) * TP, kEnd = (TQ - 1) * TP;
      unrolled<0, kT>([&](auto at) __attribute__((always_inline)) {
        constexpr int t = decltype(at)::value, j = t / TP, i = t % TP;
        if constexpr (t == kMid || t == kEnd)
          stage_barrier<kLoads, kLoads + kStores>(on & left);
        if constexpr (t == kMid)
          if (step == 1) left = kLoads;
        if constexpr (k8) {
          // 8 bits: each product of a block of 128 is added, scaled, while
          // the next one is in the matrix unit
          constexpr int last = (t + kT - 2) % kT, jl = last / TP,
                        il = last % TP;
          if constexpr (kWide) {
            if constexpr (i == 0) qw = widened(qf[j & 1]);
            if constexpr (j == 0) pw[i] = widened(pf[i]);
            d[t & 3] = mfma_wide(pw[i], qw);
          } else {
            d[t & 3] = mfma8(pf[i], qf[j & 1]);
          }
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (i == 1) s[j & 1] *= sw;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[il][jl][r] = fmaf(d[last & 3][r], s[jl & 1], acc[il][jl][r]);
          // keeps the order of products and sums; a real instruction, as
          // the compiler counts it as one
          asm volatile("s_nop 0" ::"v"(acc[il][jl][0]), "v"(acc[il][jl][1]),
                       "v"(acc[il][jl][2]), "v"(acc[il][jl][3]));
        } else {
          // 16 bits: a stage is two products deep, the first for all tiles
          // of a column, then the second
          constexpr int h = i / 2;
          unrolled<0, 2>([&](auto o) __attribute__((always_inline)) {
            constexpr int ii = i % 2 * 2 + decltype(o)::value;
            acc[ii][j] = mfma16<kElem>(half<h>(pf[ii]), half<h>(qf[j & 1]),
                                       acc[ii][j]);
          });
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (i == 0) read_q(step + (j + 1) / TQ, (j + 1) % TQ);
        if constexpr (i == 1) read_s(step + (j + 1) / TQ, (j + 1) % TQ);
        if constexpr (k8) {
          if constexpr (j == TQ - 1) read_p(step + 1, i);
        } else {
          if constexpr (j == TQ - 1 && i >= 2) {
            read_p(step + 1, i * 2 - 4);
            read_p(step + 1, i * 2 - 3);
          }
        }
        // part 0 from kMid on, part 3 behind the barrier of kEnd
        constexpr int kGap = (kEnd - kMid) / 3;
        if constexpr (t == kMid || t == kMid + kGap || t == kMid + 2 * kGap)
          load_part(std::integral_constant<int, (t - kMid) / kGap>{}, step + 2);
        if constexpr (t == kEnd)
          load_part(std::integral_constant<int, 3>{}, step + 2);
        if constexpr (t == kEnd - 1) load_scales(on, step + 2);
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    if constexpr (k8) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[TP - 2][TQ - 1][r] =
            fmaf(d[2][r], s[1], acc[TP - 2][TQ - 1][r]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[TP - 1][TQ - 1][r] =
            fmaf(d[3][r], s[1], acc[TP - 1][TQ - 1][r]);
    }

    // The next tile's first loads go out before this one's results.
    if (more) begin_tile(now, next_turn);
    int const out_p = done.p0 + wp * RP + (lane >> 4) * 8;
    char* const out = a.out + done.e * a.out_expert +
                      static_cast<int64_t>(out_p) * kOutSize;
    auto row_of = [&](int j) {
      if constexpr (!kQTurned)
        return wq * RQ + j * 16 + (lane & 15);
      else
        return wq * RQ + (j >> 1) * 32 + ((lane & 15) >> 2) * 8 +
               (j & 1) * 4 + (lane & 3);
    };
    if (done.p0 + BP <= a.np) {
      // All columns are inside, and a row behind the last holds what a row
      // inside does, which it stores again: so every lane stores, and the
      // number of stores in flight is known.
      left = kLoads + kStores;
#pragma unroll
      for (int j = 0; j < TQ; ++j) {
        int64_t row;
        if constexpr (kWGrad) {
          int const q = done.q0 + row_of(j);
          row = q < a.nq ? q : a.nq - 8 + (q & 7);
        } else {
          row = slots[turn][row_of(j)];
        }
        char* const o = out + row * a.out_row;
#pragma unroll
        for (int i = 0; i < TP; i += 2)
          store8<kOut>(o + i * 16 * kOutSize, acc[i][j], acc[i + 1][j]);
      }
    } else {
      left = kLoads;
      int const end_q = kWGrad ? a.nq : done.valid;
#pragma unroll
      for (int j = 0; j < TQ; ++j) {
        if (done.q0 + row_of(j) >= end_q) continue;
        int64_t const row =
            kWGrad ? done.q0 + row_of(j) : slots[turn][row_of(j)];
        char* const o = out + row * a.out_row;
#pragma unroll
        for (int i = 0; i < TP; i += 2) {
          int const n = a.np - (out_p + i * 16);
          if (n >= 8)
            store8<kOut>(o + i * 16 * kOutSize, acc[i][j], acc[i + 1][j]);
          else
            store_few<kOut>(o + i * 16 * kOutSize, acc[i][j], acc[i + 1][j],
                            n);
        }
      }
    }
    if (!more) break;
    turn = next_turn;
  }
}

// Few rows, or few tiles in all: bound by the weights, which are read straight
// into the registers of the wave that multiplies them, and by the length of
// the contraction. A block has 16 TP columns and 64 rows of an expert at a
// time; its waves share the contraction, a quarter each, so that all of a small
// product's weights are on their way at once, and join their sums through LDS
// in a fixed order. The rows come from the caches. One row, 7168 x 2048, 8
// bits: 5.5 us, 2.7 TB/s, the launch included.
constexpr int kRowWaves = 4;

template <Elem kElem, int TP, int NQ>
struct RowPart {
  i32x8 p[TP], q[NQ];
  float s[NQ];
  float sw;
};

template <Elem kElem, Elem kOut, int TP, int NQ, Sums kSums>
__device__ __forceinline__ void multiply_rows(
    GemmArgs const& a, char const* const (&p_at)[TP],
    char const* const (&q_at)[4], char const* const (&qs_at)[4],
    float const* ps_at, int begin, int end, f32x4* joined, int wave, int lane) {
  constexpr bool k8 = kElem == Elem::kF8;
  constexpr bool kWide = k8 && kSums == Sums::k32;
  constexpr int kSize = k8 ? 1 : 2;
  // steps on their way: what 256 registers hold
  constexpr int kDeep = NQ == 1 ? 4 : NQ == 2 ? 3 : 2;
  int const bytes = a.depth * kSize;
  int const low = (lane >> 4) * 16, high = low + 64;  // of a step
  char const* const zeros = reinterpret_cast<char const*>(&zero_page);
  auto load16 = [&](char const* row, int at) {
    char const* const g = k8 || at < bytes ? row + at : zeros;
    return *reinterpret_cast<i32x4 const*>(g);
  };
  auto load = [&](RowPart<kElem, TP, NQ>& r, int step) {
    auto operand = [&](char const* row) {
      return __builtin_shufflevector(load16(row, step * kStep + low),
                                     load16(row, step * kStep + high), 0, 1, 2,
                                     3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int i = 0; i < TP; ++i) r.p[i] = operand(p_at[i]);
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      r.q[j] = operand(q_at[j]);
      if constexpr (k8)
        r.s[j] = *reinterpret_cast<float const*>(qs_at[j] + step * 4);
    }
    if constexpr (k8) r.sw = ps_at[step];
  };
  f32x4 acc[TP][NQ];
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](RowPart<kElem, TP, NQ> const& r) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      float const s = k8 ? r.s[j] * r.sw : 1.f;
      [[maybe_unused]] Wide q;
      if constexpr (kWide) q = widened(r.q[j]);
#pragma unroll
      for (int i = 0; i < TP; ++i) {
        if constexpr (k8) {
          f32x4 d;
          if constexpr (kWide)
            d = mfma_wide(widened(r.p[i]), q);
          else
            d = mfma8(r.p[i], r.q[j]);
#pragma unroll
          for (int v = 0; v < 4; ++v)
            acc[i][j][v] = fmaf(d[v], s, acc[i][j][v]);
        } else {
          acc[i][j] =
              mfma16<kElem>(half<0>(r.p[i]), half<0>(r.q[j]), acc[i][j]);
          acc[i][j] =
              mfma16<kElem>(half<1>(r.p[i]), half<1>(r.q[j]), acc[i][j]);
        }
      }
    }
  };
  RowPart<kElem, TP, NQ> part[kDeep];
#pragma unroll
  for (int n = 0; n < kDeep; ++n)
    if (begin + n < end) load(part[n], begin + n);
  for (int step = begin; step < end; step += kDeep) {
#pragma unroll
    for (int n = 0; n < kDeep; ++n) {
      if (step + n < end) add(part[n]);
      if (step + n + kDeep < end) load(part[n], step + n + kDeep);
    }
  }
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j)
      joined[((i * NQ + j) * kRowWaves + wave) * 64 + lane] = acc[i][j];
}

// Valid rows of expert e up to and with each source, to `ends`; and all.
__device__ __forceinline__ int count_rows(int* ends, SlotRows const& r,
                                          int e) {
  if (!r.counts) return r.length;
  if (threadIdx.x < 64) {
    int const lane = threadIdx.x;
    int carry = 0;
    for (int s0 = 0; s0 < r.sources; s0 += 64) {
      int v = s0 + lane < r.sources
                  ? min(max(r.counts[e * r.sources + s0 + lane], 0), r.length)
                  : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        int const o = __shfl_up(v, off);
        if (lane >= off) v += o;
      }
      if (s0 + lane < r.sources) ends[s0 + lane] = carry + v;
      carry += __shfl(v, 63);
    }
  }
  __syncthreads();
  return ends[r.sources - 1];
}
__device__ __forceinline__ int slot_at(int const* ends, SlotRows const& r,
                                       int i) {
  if (!r.counts) return i;
  int begin = 0;
  for (int s = 0; s < r.sources; ++s) {
    int const end = ends[s];
    if (i < end) return s * r.length + i - begin;
    begin = end;
  }
  return 0;
}

// 4 results of consecutive p, the first `n` of them.
template <Elem kOut>
__device__ __forceinline__ void store4(char* at, f32x4 v, int n) {
  using T = OutType<kOut>;
  if (n >= 4) {
    T four[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = static_cast<T>(v[k]);
    __builtin_memcpy(at, four, sizeof(four));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) reinterpret_cast<T*>(at)[k] = static_cast<T>(v[k]);
  }
}

template <Elem kElem, Elem kOut, int TP, Sums kSums>
__global__ __launch_bounds__(kRowWaves * 64, 2) void k_expert_rows(
    GemmArgs a) {
  constexpr bool k8 = kElem == Elem::kF8;
  constexpr int kSize = k8 ? 1 : 2;
  constexpr int kOutSize = kOut == Elem::kF32 ? 4 : 2;
  __shared__ f32x4 joined[TP * 4 * kRowWaves * 64];
  __shared__ int ends[kMaxSlotCells];
  int const wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int const e = blockIdx.y, p0 = blockIdx.x * (16 * TP);

  int const valid = count_rows(ends, a.rows, e);
  auto slot = [&](int i) { return slot_at(ends, a.rows, i); };

  char const* const pe = a.p + e * a.p_expert;
  char const* const qe = a.q + e * a.q_expert;
  char const* p_at[TP];
#pragma unroll
  for (int i = 0; i < TP; ++i)
    p_at[i] = pe + static_cast<int64_t>(
                       min(p0 + i * 16 + (lane & 15), a.np - 1)) *
                       a.p_row;
  float const* ps_at = nullptr;
  if constexpr (k8)
    ps_at = reinterpret_cast<float const*>(a.p_scales + e * a.ps_expert +
                                           p0 / 128 * a.ps_row);
  int const steps = (a.depth * kSize + kStep - 1) / kStep;
  int const begin = steps * wave / kRowWaves;
  int const end = steps * (wave + 1) / kRowWaves;

  for (int q0 = blockIdx.z * 64; q0 < valid; q0 += gridDim.z * 64) {
    int const tiles = min(4, (valid - q0 + 15) / 16);
    char const* q_at[4];
    char const* qs_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < tiles) {
        int64_t const row = slot(min(q0 + j * 16 + (lane & 15), valid - 1));
        q_at[j] = qe + row * a.q_row;
        if constexpr (k8)
          qs_at[j] = a.q_scales + e * a.qs_expert + row * a.qs_row;
      }
    auto go = [&](auto n) {
      multiply_rows<kElem, kOut, TP, decltype(n)::value, kSums>(
          a, p_at, q_at, qs_at, ps_at, begin, end, joined, wave, lane);
    };
    if (tiles == 1) go(std::integral_constant<int, 1>{});
    else if (tiles == 2) go(std::integral_constant<int, 2>{});
    else if (tiles == 3) go(std::integral_constant<int, 3>{});
    else go(std::integral_constant<int, 4>{});
    __syncthreads();
    for (int t = wave; t < TP * tiles; t += kRowWaves) {
      int const i = t / tiles, j = t - i * tiles;
      f32x4 sum = joined[t * kRowWaves * 64 + lane];
#pragma unroll
      for (int w = 1; w < kRowWaves; ++w)
        sum += joined[(t * kRowWaves + w) * 64 + lane];
      int const q = q0 + j * 16 + (lane & 15);
      int const p = p0 + i * 16 + (lane >> 4) * 4;
      if (q < valid && p < a.np) {
        char* const o = a.out + e * a.out_expert + slot(q) * a.out_row +
                        static_cast<int64_t>(p) * kOutSize;
        store4<kOut>(o, sum, a.np - p);
      }
    }
    __syncthreads();
  }
}

// The same where P is turned (weights as they lie for the rows' gradient) or
// both are (weight gradient), 16 bits: tiles of 64 x 64, whose 8 waves share
// the contraction in steps of 64. Each wave turns its part of an operand in
// its own piece of LDS, written from registers, so waves wait for nobody until
// they join their sums. Bound by the length of the contraction. 3246 rows of 2
// experts, weight gradient 56 x 72: 12 us.
constexpr int kLongWaves = 8;

template <Mode kMode, Elem kElem, Elem kOut>
__global__ __launch_bounds__(kLongWaves * 64, 2) void k_expert_long(
    GemmArgs a) {
  constexpr bool kWGrad = kMode == Mode::kWeightGrad;
  constexpr int kOutSize = kOut == Elem::kF32 ? 4 : 2;
  constexpr int kSide = 64, kRowBytes = kSide * 2, kPiece = kSide * kRowBytes;
  static_assert(kStep == 2 * kSide, "a step of a direct operand");
  // pieces of the waves, P before Q; then their sums, 16 tiles a wave
  __shared__ __attribute__((aligned(1024))) char lds[kLongWaves * 2 * kPiece];
  __shared__ int ends[kMaxSlotCells];
  f32x4* const joined = reinterpret_cast<f32x4*>(lds);
  int const wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int const e = blockIdx.y, p0 = blockIdx.x * kSide;
  int const valid = count_rows(ends, a.rows, e);
  char const* const pe = a.p + e * a.p_expert;
  char const* const qe = a.q + e * a.q_expert;
  int const depth = kWGrad ? valid : a.depth;
  int const steps = (depth + kSide - 1) / kSide;
  int const begin = static_cast<int64_t>(steps) * wave / kLongWaves;
  int const end = static_cast<int64_t>(steps) * (wave + 1) / kLongWaves;

  // this lane's part of a turned operand: 16 bytes of 8 rows
  int const row = lane >> 3, chunk = lane & 7;
  int64_t const p_col = static_cast<int64_t>(min(p0 + chunk * 8, a.np - 8)) * 2;
  char* const my_p = lds + wave * 2 * kPiece;
  char* const my_q = my_p + kPiece;
  int const put = row * kRowBytes + ((chunk ^ ((row & 3) << 2 & 7)) * 16);
  // and of the reads that turn it
  int const r = (lane >> 2) & 3, c = lane & 3;
  int const turn = ((lane >> 4) * 8 + r) * kRowBytes;
  uint32_t const get_lo = turn + ((c ^ (r << 2 & 7)) * 16);
  uint32_t const get_hi = turn + (((c + 4) ^ (r << 2 & 7)) * 16);
  auto turned = [&](char* piece, int i) {
    uint32_t const at =
        lds_addr(piece) + (i >> 1 ? get_hi : get_lo) + (i & 1) * 8;
    i16x4 const v0 = lds_read_turned(at);
    i16x4 const v1 = lds_read_turned(at + 4 * kRowBytes);
    i16x4 const v2 = lds_read_turned(at + 32 * kRowBytes);
    i16x4 const v3 = lds_read_turned(at + 36 * kRowBytes);
    i32x4 const x = __builtin_bit_cast(
        i32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    i32x4 const y = __builtin_bit_cast(
        i32x4, __builtin_shufflevector(v2, v3, 0, 1, 2, 3, 4, 5, 6, 7));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  int const q_end = kWGrad ? a.nq : valid;
  for (int q0 = blockIdx.z * kSide; q0 < q_end; q0 += gridDim.z * kSide) {
    int64_t const q_col =
        kWGrad ? static_cast<int64_t>(min(q0 + chunk * 8, a.nq - 8)) * 2 : 0;
    char const* q_at[4];
    if constexpr (!kWGrad) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q_at[j] = qe + static_cast<int64_t>(slot_at(
                           ends, a.rows,
                           min(q0 + j * 16 + (lane & 15), valid - 1))) *
                           a.q_row;
    }
    // the source that this lane's next row of the contraction lies in
    int seg = -1, seg_begin = 0, seg_end = 0;
    i32x4 const zero = {0, 0, 0, 0};
    struct Part {
      i32x4 p[8];
      i32x4 q[8];  // turned: 8 rows; direct: two halves of 4 tiles
    };
    auto load = [&](Part& t, int step) {
#pragma unroll
      for (int l = 0; l < 8; ++l) {
        int const i = step * kSide + l * 8 + row;
        t.p[l] = zero;
        if constexpr (kWGrad) t.q[l] = zero;
        if (i < depth) {
          int64_t at = i;
          if constexpr (kWGrad) {
            if (a.rows.counts) {
              while (i >= seg_end) {  // ends: the last end is `valid`
                ++seg;
                seg_begin = seg_end;
                seg_end = ends[seg];
              }
              at = static_cast<int64_t>(seg) * a.rows.length + i - seg_begin;
            }
            t.q[l] = *reinterpret_cast<i32x4 const*>(qe + at * a.q_row + q_col);
          }
          t.p[l] = *reinterpret_cast<i32x4 const*>(pe + at * a.p_row + p_col);
        }
      }
      if constexpr (!kWGrad) {
#pragma unroll
        for (int l = 0; l < 8; ++l) {
          int64_t const at = static_cast<int64_t>(step) * kStep +
                             (lane >> 4) * 16 + (l & 1) * 64;
          t.q[l] = at < static_cast<int64_t>(depth) * 2
                       ? *reinterpret_cast<i32x4 const*>(q_at[l >> 1] + at)
                       : zero;
        }
      }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Part part;
    if (begin < end) load(part, begin);
    for (int step = begin; step < end; ++step) {
      i32x8 pf[4], qf[4];
#pragma unroll
      for (int l = 0; l < 8; ++l) {
        *reinterpret_cast<i32x4*>(my_p + l * 8 * kRowBytes + put) = part.p[l];
        if constexpr (kWGrad)
          *reinterpret_cast<i32x4*>(my_q + l * 8 * kRowBytes + put) = part.q[l];
      }
      if constexpr (!kWGrad) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[j] = __builtin_shufflevector(part.q[2 * j], part.q[2 * j + 1], 0,
                                          1, 2, 3, 4, 5, 6, 7);
      }
      if (step + 1 < end) load(part, step + 1);
      // the lanes of this wave see each other's part
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pf[i] = turned(my_p, i);
        if constexpr (kWGrad) qf[i] = turned(my_q, i);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = mfma16<kElem>(half<0>(pf[i]), half<0>(qf[j]), acc[i][j]);
          acc[i][j] = mfma16<kElem>(half<1>(pf[i]), half<1>(qf[j]), acc[i][j]);
        }
    }
    __syncthreads();  // `joined` lies where the pieces do
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        joined[((i * 4 + j) * kLongWaves + wave) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < 16; t += kLongWaves) {
      int const i = t >> 2, j = t & 3, m = lane & 15;
      f32x4 sum = joined[t * kLongWaves * 64 + lane];
#pragma unroll
      for (int w = 1; w < kLongWaves; ++w)
        sum += joined[(t * kLongWaves + w) * 64 + lane];
      int const p = p0 + (i >> 1) * 32 + (lane >> 4) * 8 + (i & 1) * 4;
      int const q =
          q0 + (kWGrad ? (j >> 1) * 32 + (m >> 2) * 8 + (j & 1) * 4 + (m & 3)
                       : j * 16 + m);
      if (q < q_end && p < a.np) {
        int64_t const at = kWGrad ? q : slot_at(ends, a.rows, q);
        store4<kOut>(a.out + e * a.out_expert + at * a.out_row +
                         static_cast<int64_t>(p) * kOutSize,
                     sum, a.np - p);
      }
    }
    __syncthreads();
  }
}

int compute_units() {
  int dev = 0, n = 0;
  UCCL_CHECK_HIP(hipGetDevice(&dev));
  UCCL_CHECK_HIP(
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
  return n;
}

// Whether the offsets of a stage's loads from the tile's first address, with
// the loads' own share of them, fit 32 bits: `p_span` and `q_span` rows.
bool lies_near(GemmArgs const& a, int64_t p_span, int64_t q_span) {
  constexpr int64_t kEnd = (int64_t{1} << 32) - 16384;
  return p_span * a.p_row < kEnd && q_span * a.q_row < kEnd;
}

template <Mode kMode, Elem kElem, Elem kOut, int BP, int BQ, int WP, int WQ,
          bool kFar = false, Sums kSums = Sums::kUnit>
void launch_tiles(GemmArgs const& a, int blocks_per_cu, hipStream_t s) {
  int64_t const tiles_p = (a.np + BP - 1) / BP;
  int64_t const q = kMode == Mode::kWeightGrad
                        ? a.nq
                        : static_cast<int64_t>(a.rows.sources) * a.rows.length;
  int64_t const most = a.rows.experts * tiles_p * ((q + BQ - 1) / BQ);
  int64_t grid = std::min<int64_t>(most, compute_units() * blocks_per_cu);
  grid = (grid + 7) / 8 * 8;
  k_expert_gemm<kMode, kElem, kOut, BP, BQ, WP, WQ, kFar, kSums>
      <<<static_cast<int>(grid), WP * WQ * 64, 0, s>>>(a);
}

template <Elem kElem, Elem kOut, int TP, Sums kSums = Sums::kUnit>
void launch_rows(GemmArgs const& a, int expected_rows, hipStream_t s) {
  dim3 const grid((a.np + 16 * TP - 1) / (16 * TP), a.rows.experts,
                  std::min((expected_rows + 63) / 64, 1024));
  k_expert_rows<kElem, kOut, TP, kSums><<<grid, kRowWaves * 64, 0, s>>>(a);
}

template <Mode kMode, Elem kElem, Elem kOut>
void launch_long(GemmArgs const& a, int expected_rows, hipStream_t s) {
  dim3 const grid((a.np + 63) / 64, a.rows.experts,
                  std::min((expected_rows + 63) / 64, 1024));
  k_expert_long<kMode, kElem, kOut><<<grid, kLongWaves * 64, 0, s>>>(a);
}

// Which kernel, by the rows that an expert is expected to have and the tiles
// that this makes. Measured in us, as calls in a stream, experts of unlike
// popularity, rows of an expert on average:
//                      rows   1   2   4   8  16  24  32  48  64  96 128 192 256
//   8 bits, 32 experts, 4096 x 7168
//     k_expert_rows         106 134 165 171 213 252 290
//     tiles of 256 x 64     134 141 161 153 165 168 208 202 206 253 302 403
//     tiles of 256 x 128    140 150 165 159 167 170 173 178 223 233 238 300 405
//     tiles of 256 x 256    193 206 233 226 237 241 241 240 244 251 253 326 361
//   8 bits, 16 experts, 7168 x 2048
//     k_expert_rows          36  39  48  60  70  77  90
//     tiles of 256 x 64      39  39  40  41  42  42  43  61  62  76  94 128
//     tiles of 256 x 128     40  40  40  42  43  43  46  46  48  64  67  88 111
//     tiles of 256 x 256     56  57  57  60  63  63  63  65  63  67  68  98 106
//   8 bits, 8 experts, 4096 x 4096: 128 tiles of 256 x 64, half of the card
//     k_expert_rows          24  26  27  31  36  42  57
//     tiles of 256 x 64      34  35  35  35  35  36  36  37  37  38  68  69
//     tiles of 256 x 128     34  36  36  36  36  36  37  37  37  38  40  43  70
//     tiles of 256 x 256                                         52  53  56  58
//   16 bits, 32 experts, 4096 x 7168
//     k_expert_rows         192 251 313 309 375 441 513
//     tiles of 256 x 64     238 257 308 291 313 316 376 356 360 418 485 633
//     tiles of 256 x 128    250 270 309 294 313 316 319 325 401 398 404 512 682
//     tiles of 256 x 256    324 366 419 403 419 422 422 424 428 432 435 560 608
//   16 bits, 16 experts, 7168 x 2048
//     k_expert_rows          55  66  79 100 116 127 144
//     tiles of 256 x 64      65  80  96 111 111 112 111 124 123 132 158 197
//     tiles of 256 x 128     70  86  99 114 116 115 116 118 117 134 135 156 188
//     tiles of 256 x 256     95 103 116 126 127 128 128 130 132 135 137 171 182
//   16 bits, 8 experts, 4096 x 4096
//     k_expert_rows          35  46  47  47  55  62  84
//     tiles of 256 x 64      46  48  48  47  49  50  50  52  54  59  98 105
//     tiles of 256 x 128     55  56  58  57  58  58  59  59  60  65  68  75 124
//     tiles of 256 x 256                                         91  92 102 102
//   the same turned (row gradients), 16 experts, 7168 x 2048
//     tiles of 256 x 64      65  70  78  85  87  89  89 108 109 124 150 191
//     tiles of 256 x 128     72  77  84  91  92  93  93  96  95 123 125 152 186
//     tiles of 256 x 256     98 101 106 118 119 121 121 120 125 126 127 169 172
//   1 expert, 7168 x 2048, 8 bits        rows:   1    16    64
//     k_expert_rows                            5.5   7.6  16.4
//     tiles of 128 x 128                      20.0  20.1  20.4
//   32 experts, 4096 x 7168, 8 bits, rows too far apart for 32-bit offsets
//     k_expert_rows                    rows:   1   4   8  16  32
//                                            154 159 178 238 332
//     tiles of 128 x 128                     409 410 409 409 410
// Few tiles, experts of like popularity, one round of 128 x 128 or less:
//   128 rows of 4 / 8 experts   512 x 1024, 16 bits   1024 x 1024, 8 bits
//     k_expert_rows                    8.4 / 13.0           10.3 / 18.5
//     tiles of 128 x 128              14.3 / 14.5           12.5 / 12.9
//   tiles of 128 x 128:            128, 8 bits  128, 16 bits  256 to 280, 8 bits
//     8 experts x 200, 1024 x 1024  13.2 / 14.0  14.9 / 19.0
//     4 experts x 200, 2048 x 2048  20.4 / 21.2  23.9 / 31.4
//     16 experts x 200, 512 x 1024  13.1 / 14.1  15.1 / 19.0
//     2 experts x 200, 4096 x 1024  13.0 / 14.2  14.7 / 18.9
//     8 experts x 200, 2048 x 1024                            24.4 / 15.1
//   with 128 x 128 / 256 x 128; 8 bits fit once on a compute unit, so that the
//   odd tile more than there are units costs a round. (16 bits, 8 x 200 and
//   8 x 512 rows, 2048 x 1024: 19.9 / 20.2 and 29.6 / 35.9.)
//   row gradients, k_expert_long / tiles of 128 x 128, by tiles of 64 x 64
//                       tiles  64 or less     128            192         256
//     8 experts, 512 x 1024    7.6 / 14.2   9.5 / 14.5   9.7 / 14.9
//     8 experts, 1024 x 1024                7.9 / 14.4               9.8 / 14.7
//     4 experts, 1024 x 2048  10.7 / 23.6  13.9 / 23.9  15.1 / 24.4
//     3 experts, 1000 x 4096  20.2 / 42.2
//     16 experts, 512 x 512                 6.4 /  9.5               7.5 /  9.8
//     8 experts, 1024 x 256                 6.2 /  7.0               6.5 /  7.4
//   (up to 9.7 / 7.4 where an expert has more rows than expected), 384: 16.7 /
//   15.3, 12.8 / 10.3
//   weight gradients, k_expert_long / tiles of 256 x 128
//                         rows      139         512        2048        4096
//     256 tiles of 64 x 64
//       4 experts, 512 x 512     6.0 /  9.8  8.2 / 16.3 18.7 / 42.5 30.9 / 77.4
//       1 expert, 1024 x 1024    6.0 /  9.8  7.1 / 14.1 14.6 / 36.7 23.8 / 67.1
//       64 experts, 128 x 128    6.1 /  9.6  8.4 / 17.0 21.3 / 45.1 37.4 / 82.4
//     512 tiles
//       8 experts, 512 x 512    10.7 / 10.1 16.5 / 16.6 37.0 / 44.2 65.0 / 79.6
//       2 experts, 1024 x 1024  10.5 / 10.2 14.4 / 15.9 29.8 / 40.8 47.9 / 72.8
//     8 experts, 1000 x 1024    46.5 / 12.5 (256 x 256 15.8)
//     3 experts x 3345 rows, 88 x 3544 (336 tiles): 44.1 / 66.4
template <Mode kMode, Elem kElem, Elem kOut>
void launch_sized(GemmArgs const& a, int expected_rows, hipStream_t s) {
  auto tiles = [&](int p, int q) {
    return static_cast<int64_t>(a.rows.experts) * ((a.np + p - 1) / p) *
           ((expected_rows + q - 1) / q);
  };
  int const cus = compute_units();
  if constexpr (kMode == Mode::kProduct) {
    int const few = kElem != Elem::kF8      ? 8
                    : !a.near               ? 32
                    : tiles(256, 64) >= cus ? 2
                                            : 16;
    if (expected_rows <= few || tiles(16, 64) <= 2 * cus) {
      if (tiles(32, 64) >= 4 * cus)
        launch_rows<kElem, kOut, 2>(a, expected_rows, s);
      else
        launch_rows<kElem, kOut, 1>(a, expected_rows, s);
      return;
    }
  }
  if constexpr (kMode != Mode::kProduct) {
    bool const many_rows = kMode == Mode::kWeightGrad &&
                           a.rows.sources * a.rows.length > 2048;
    if (tiles(64, 64) <= (many_rows ? 2 : 1) * cus)
      return launch_long<kMode, kElem, kOut>(a, expected_rows, s);
  }
  if constexpr (kElem == Elem::kF8) {
    if (!a.near)
      return launch_tiles<kMode, kElem, kOut, 128, 128, 2, 2, true>(a, 2, s);
  }
  if constexpr (kMode != Mode::kWeightGrad) {
    if (tiles(128, 128) <= cus / 2)
      return launch_tiles<kMode, kElem, kOut, 128, 128, 2, 2>(a, 2, s);
    if (expected_rows <= 24)
      return launch_tiles<kMode, kElem, kOut, 256, 64, 4, 1>(a, 1, s);
    if (expected_rows <= 192)
      return launch_tiles<kMode, kElem, kOut, 256, 128, 4, 2>(a, 1, s);
  }
  if (tiles(256, 256) >= cus)
    launch_tiles<kMode, kElem, kOut, 256, 256, 4, 2>(a, 1, s);
  else
    launch_tiles<kMode, kElem, kOut, 256, 128, 4, 2>(a, 1, s);
}

// 8-bit operands, sums of 32 bits: a like choice among fewer kernels. The
// widened operands take the registers that a tile of 256 x 256 would need (it
// spills, and gains 3% at 32768 rows of 8 experts). Measured in us, experts of
// unlike popularity, rows on average:
//   32 experts, 4096 x 7168           rows:   1    2    4    8   32   48   96  128
//     k_expert_rows                         135  175  221  231  431
//     tiles of 256 x 64                     162  167  187  183  246  260  336  403
//     tiles of 256 x 128                    203  219  246  241  250  250  321  352
//   16 experts, 7168 x 2048
//     k_expert_rows                          50   57   68   87  139
//     tiles of 256 x 64                      52   53   53   55   56   80  105  131
//     tiles of 256 x 128                     63   64   64   64   66   67   98   99
//   8 experts, 4096 x 4096 (128 tiles of 256 x 64: half of the card)
//     k_expert_rows                          25   32   36   43   79
//     tiles of 256 x 64                      49   49   49   49   50   50   53   97
//     tiles of 256 x 128                     60   61   60   61   61   62   61   63
//   32 experts, 4096 x 7168, rows too far apart for 32-bit offsets
//     k_expert_rows                         192       211  238  516
//     tiles of 128 x 128                    512       512  513  513
template <Elem kOut>
void launch_wide(GemmArgs const& a, int expected_rows, hipStream_t s) {
  constexpr Mode kMode = Mode::kProduct;
  constexpr Elem kElem = Elem::kF8;
  auto tiles = [&](int p, int q) {
    return static_cast<int64_t>(a.rows.experts) * ((a.np + p - 1) / p) *
           ((expected_rows + q - 1) / q);
  };
  int const cus = compute_units();
  int const few = !a.near ? 32 : tiles(256, 64) < cus ? 8 : 2;
  if (expected_rows <= few || tiles(16, 64) <= 2 * cus)
    launch_rows<kElem, kOut, 1, Sums::k32>(a, expected_rows, s);
  else if (!a.near)
    launch_tiles<kMode, kElem, kOut, 128, 128, 2, 2, true, Sums::k32>(a, 2, s);
  else if (expected_rows <= 32)
    launch_tiles<kMode, kElem, kOut, 256, 64, 4, 1, false, Sums::k32>(a, 1, s);
  else
    launch_tiles<kMode, kElem, kOut, 256, 128, 4, 2, false, Sums::k32>(a, 1,
                                                                       s);
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
  int64_t const slots = static_cast<int64_t>(m.rows.sources) * m.rows.length;
  a.near = lies_near(a, 256, slots);
  a.depth = m.k;
  if (m.elem == Elem::kF8) {
    a.p_scales = static_cast<char const*>(m.w_scales.p);
    a.ps_expert = m.w_scales.expert_stride * 4;
    a.ps_row = m.w_scales.row_stride * 4;
    a.q_scales = static_cast<char const*>(m.x_scales.p);
    a.qs_expert = m.x_scales.expert_stride * 4;
    a.qs_row = m.x_scales.row_stride * 4;
    if (!m.precise)
      by_out<Mode::kProduct, Elem::kF8>(a, m.out_elem, m.expected_rows, s);
    else if (m.out_elem == Elem::kBF16)
      launch_wide<Elem::kBF16>(a, m.expected_rows, s);
    else if (m.out_elem == Elem::kF16)
      launch_wide<Elem::kF16>(a, m.expected_rows, s);
    else
      launch_wide<Elem::kF32>(a, m.expected_rows, s);
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
  int64_t const slots = static_cast<int64_t>(w.rows.sources) * w.rows.length;
  a.near = lies_near(a, slots, slots);
  a.nq = w.n;
  if (w.elem == Elem::kBF16)
    by_out<Mode::kWeightGrad, Elem::kBF16>(a, w.out_elem, w.n, s);
  else
    by_out<Mode::kWeightGrad, Elem::kF16>(a, w.out_elem, w.n, s);
}

}  // namespace ep
}  // namespace uccl
