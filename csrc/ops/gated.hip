// Gated linear layer h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients (gfx950, MFMA, fp32 accumulation).
//
//   weight [2F][D] = Wg over Wu, bias [2F] = bg, bu;  act: silu g s(g), gelu g Phi(g), sigmoid s(g)
//   forward     both products of a tile in one kernel; bias, activation, product and rounding in its epilogue
//   backward    g and u from the fp32 accumulators again -- kept by the forward pass, or computed once more where that
//               is cheaper (saves()) -- dg = dh u act'(g), du = dh act(g), rounded once to the operand type;
//               dx = dg Wg + du Wu,  dW = [dg | du]^T x,  db = column sums (fp32, of the unrounded values)
// The rounding of dg and du to bf16 operands is the one besides the results' own: a norm error of 0.0023 in dx and dW against
// 64 bits, 0.0017 without it (25600 x 256 x 1024).  More bits would need a second product of the remainders, twice the time
// of dx and dW; fp32 operands keep them.
//
// bf16 operands run on v_mfma_f32_32x32x16_bf16, fp32 on v_mfma_f32_32x32x2_f32.
#include <hip/hip_bf16.h>
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <pybind11/pybind11.h>

#include "../common.h"

namespace py = pybind11;

namespace gsc {
namespace gated {

typedef __hip_bfloat16 bf16;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef short s16x8_any __attribute__((ext_vector_type(8), aligned(2)));   // at any element's alignment

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(short v) { return __bfloat162float(__builtin_bit_cast(bf16, v)); }
__device__ __forceinline__ short to_s(float v) { return __builtin_bit_cast(short, __float2bfloat16(v)); }

// ---- activations

enum Act { SILU = 0, GELU = 1, SIGMOID = 2 };

// FULL (fp32 operands): exponential and reciprocal to an ulp.  bf16 results are rounded to 2^-8 behind them: the hardware's
// are enough there (relative error of the exponential 2^-24 (|argument| + 2)).
template <bool FULL>
__device__ __forceinline__ float exp_of(float x) { return FULL ? expf(x) : __expf(x); }
template <bool FULL>
__device__ __forceinline__ float inverse(float x) { return FULL ? 1.f / x : __builtin_amdgcn_rcpf(x); }

template <bool FULL>
__device__ __forceinline__ float sigmoid(float g) { return inverse<FULL>(1.f + exp_of<FULL>(-g)); }

// Phi(g) = erfc(-g / sqrt 2) / 2 and e = exp(-g^2 / 2), the exponential that the derivative needs as well.  With z = |g| /
// sqrt 2 and t = 1 / (1 + 0.4 z), exp(z^2) erfc(z) / 2 = t Q(t): Q is the polynomial of degree 8 of least maximal relative
// error over |g| <= 14 (6e-8, fitted in 64 bits), so the small values of the negative side are right to their last digits,
// but for the rounding of g^2 / 2 in the exponent.
template <bool FULL>
__device__ __forceinline__ float normal_cdf(float g, float& e) {
  e = exp_of<FULL>(-0.5f * g * g);
  const float t = inverse<FULL>(1.f + 0.4f * 0.70710678f * fabsf(g));
  const float q =
      0.112817116f + t * (0.113221556f + t * (0.100943796f + t * (0.0966966152f + t * (0.0398782045f + t *
      (0.0439822488f + t * (0.0419935584f + t * (-0.0701595694f + t * 0.0206265077f)))))));
  const float tail = t * q * e;
  return g < 0.f ? tail : 1.f - tail;
}

template <int ACT, bool FULL>
__device__ __forceinline__ float act_fwd(float g) {
  float e;
  if (ACT == GELU) return g * normal_cdf<FULL>(g, e);
  const float s = sigmoid<FULL>(g);
  return ACT == SILU ? g * s : s;
}

// a = act(g), d = act'(g)
template <int ACT, bool FULL>
__device__ __forceinline__ void act_both(float g, float& a, float& d) {
  if (ACT == GELU) {
    float e;
    const float phi = normal_cdf<FULL>(g, e);
    a = g * phi;
    d = phi + g * e * 0.39894228f;
    return;
  }
  const float s = sigmoid<FULL>(g);
  a = ACT == SILU ? g * s : s;
  d = ACT == SILU ? s * (1.f + g * (1.f - s)) : s * (1.f - s);
}

struct Bias {
  const void* p;
  int bf;
  __device__ __forceinline__ float at(long i) const {
    if (!p) return 0.f;
    return bf ? __bfloat162float(reinterpret_cast<const bf16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
  }
};

// Row of accumulator register r of lane: v_mfma 32x32 C layout (the column is lane & 31).
__device__ __forceinline__ constexpr int acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// ---------------------------------------------------------------------------------------------------------------
// Tiles.  out = sum_k A(r, k) B(c, k) on BM x BN tiles, K in steps of 128 bytes (64 bf16, 32 fp32).  A step's operands
// are loaded into registers two steps before they are stored to LDS and three before the products take them: the
// products alone (2048 cycles a step on a 256 x 256 tile) hide less than the latency of loads that miss the L2.
//
//   row operand (k contiguous)    LDS [R][128 B], 16-byte chunk c of row r in slot c ^ ((r >> 1) & 7): the 16 rows of a
//                                 fragment read cover all 64 banks once
//   column operand (r contiguous) LDS [k][R]; bf16: chunk c of row k in slot c ^ 4 (k & 3), so the four rows of a
//                                 transposing read (ds_read_b64_tr_b16) fall on four different quarters of the banks;
//                                 fp32: slot c ^ 8 ((k >> 2) & 1), so the two halves of a wave read different banks
// Lane l of a wave copy holds the 16 bytes of slot l of its 1 KB of LDS: the slots are permuted on the address side.  Rows
// and chunks outside the matrices get an offset past the buffer descriptor's end: the load returns zeros.  Operands are
// 16-byte aligned with rows of a multiple of 8 elements (the caller pads others), so a chunk is inside or outside as a
// whole.

constexpr unsigned kOut = 0x80000000u;   // past every descriptor (2^31 - 1 bytes)

template <class T>
struct Elem;
template <>
struct Elem<bf16> {
  static constexpr int STEP = 64, CHUNK = 8;   // k per step, elements per 16 bytes
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<float> {
  static constexpr int STEP = 32, CHUNK = 4;
  typedef f32x4 frag;   // a lane's k = 8 s + 4 half ..: product t takes element t, k = 8 s + t and 8 s + 4 + t
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
};

template <class T, int R, int WAVES, bool COL>
struct Copy {
  static constexpr int PER = R / 8 / WAVES;   // 1 KB wave copies per wave and step
  static constexpr int CH = Elem<T>::CHUNK;
  static_assert(R % (8 * WAVES) == 0 && (!COL || R >= (CH == 8 ? 128 : 64)), "tile");
  static constexpr int CPR = COL ? R / CH : 8;   // chunks per stored row
  unsigned off[PER];
  long step;        // elements per step
  static __device__ __forceinline__ int row_of(int i, int wave, int lane) { return (i * WAVES + wave) * 64 / CPR + lane / CPR; }
  static __device__ __forceinline__ int chunk_of(int r, int lane) {
    return (lane % CPR) ^ (!COL ? (r >> 1) & 7 : CH == 8 ? (r & 3) << 2 : ((r >> 2) & 1) << 3);
  }
  // r0: first row (column) of the tile, rows: their count in the matrix, ld: elements between stored rows
  __device__ __forceinline__ void init(long r0, long rows, long ld, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = row_of(i, wave, lane), c = chunk_of(r, lane);
      off[i] = (COL ? r0 + CH * c : r0 + r) < rows ? (unsigned)(r * ld * sizeof(T) + 16 * c) : kOut;
    }
    step = COL ? Elem<T>::STEP * ld : Elem<T>::STEP;
  }
  // Piece i.  base: the tile's first element at this step, left: k that remain (>= a step: all)
  __device__ __forceinline__ u32x4 load(int i, const T* base, int left, int wave, int lane) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, 0x7fffffff, 0x00027000);
    unsigned o = off[i];
    if (left < Elem<T>::STEP) {
      const int r = row_of(i, wave, lane);
      o = (COL ? r : CH * chunk_of(r, lane)) < left ? o : kOut;
    }
    return __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0);
  }
  static __device__ __forceinline__ void store(int i, const u32x4& reg, T* img, int wave, int lane) {
    *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(img) + 1024 * (i * WAVES + wave) + 16 * lane) = reg;
  }
};

// Addresses of a wave's 32-row fragments in an image of R rows (columns).  Fragment i covers rows r0 + 32 i.  Everything
// but one register per k step (row image) or per fragment (column image) is an immediate offset of the read.
template <class T, int R, bool COL, int N>
struct Frags {
  static constexpr int STEP = Elem<T>::STEP, CH = Elem<T>::CHUNK;
  typedef typename Elem<T>::frag frag;
  const T* at[COL ? N : 4];
  __device__ __forceinline__ void init(const T* img, int r0, int lane) {
    if constexpr (!COL) {
      const int r = r0 + (lane & 31), c = (lane >> 5) ^ ((r >> 1) & 7);
#pragma unroll
      for (int s = 0; s < 4; ++s) at[s] = img + r * STEP + CH * (c ^ (2 * s));
    } else if constexpr (CH == 8) {
      const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
#pragma unroll
      for (int i = 0; i < N; ++i)
        at[i] = img + (8 * (g >> 1) + q) * R + 8 * ((((r0 >> 3) + 4 * i) ^ (q << 2)) + 2 * (g & 1) + (p >> 1)) + 4 * (p & 1);
    } else {
      const int h = lane >> 5;
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = img + 4 * h * R + ((r0 + 32 * i + (lane & 31)) ^ (h << 5));
    }
  }
  // fragment i of quarter s of the step; shift: elements to the image in use
  __device__ __forceinline__ frag read(int i, int s, int shift) const {
    if constexpr (!COL) {
      return *reinterpret_cast<const frag*>(at[s] + shift + 32 * STEP * i);
    } else if constexpr (CH == 8) {
      const T* a = at[i] + shift + 16 * s * R;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * R));
      return __builtin_bit_cast(frag, (s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}));
    } else {
      const T* a = at[i] + shift + 8 * s * R;
      return frag{a[0], a[R], a[2 * R], a[3 * R]};
    }
  }
};

struct TileArgs {
  const void* a[2];   // operands of the two K segments (dx: gate and up halves), one segment otherwise
  const void* b[2];   // pair kernels: gate and up rows instead
  long lda, ldb;
  int segs;
  long M, N, K;       // rows, columns (pair: F) and K of a segment
  int tm, tn;         // tiles
  int chunk;          // steps of a split (blockIdx.y)
  Bias bias;
  const void* dh;
  long lddh;
  void* out;
  long ldo;
  long half;          // dgu: column of du
  long slab;          // elements between the fp32 partial results (FWD, PART: accumulators) of two splits
  int tmh;            // dW: tile rows of the gate half (the up half follows), 0 otherwise
  float* part;
  float* saved;       // accumulators of the pair products, [tile][register quarter][thread][4]
  float* splits;      // the same of each split (FWD, PART)
  int nsplits;
  int act;
};

// Workgroups are dealt to the 8 XCDs in turn: each XCD takes a contiguous run of tiles, walked in strips of 8 tile rows
// (fewer where its run is short: about square), so the operand panels its CUs share stay in its own L2.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& pm, int& pn) {
  const int total = tm * tn, per = total / 8, rem = total % 8, x = id & 7;
  const int t = x * per + (x < rem ? x : rem) + (id >> 3);
  const int h = per >= 32 ? 8 : per >= 8 ? 4 : 2;
  const int width = h * tn, g = t / width, first = g * h, rows = tm - first < h ? tm - first : h;
  pm = first + (t % width) % rows;
  pn = (t % width) / rows;
}

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Sum over the 32 lanes of each half wave, in its lane 31 (DPP adds in a fixed order).
__device__ __forceinline__ float half_wave_sum(float v) {
#define GSC_ADD_DPP(ctrl, mask)                                                                                      \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, mask, 0xf, true))
  GSC_ADD_DPP(0x111, 0xf);   // row_shr 1, 2, 4, 8: lane 15 of each 16 holds their sum
  GSC_ADD_DPP(0x112, 0xf);
  GSC_ADD_DPP(0x114, 0xf);
  GSC_ADD_DPP(0x118, 0xf);
  GSC_ADD_DPP(0x142, 0xa);   // row_bcast 15 into rows 1 and 3
#undef GSC_ADD_DPP
  return v;
}

// finish(activation) with the activation as a constant: a branch per element would keep the elements' exponentials and
// reciprocals from overlapping.
template <bool PAIR, class F>
__host__ __device__ __forceinline__ void by_act(int act, F&& finish) {
  if (PAIR && act == GELU) finish(std::integral_constant<int, GELU>{});
  else if (PAIR && act == SIGMOID) finish(std::integral_constant<int, SIGMOID>{});
  else finish(std::integral_constant<int, SILU>{});
}

// What leaves a tile: FWD h, BWD dgu (and the bias gradient's partial sums), OUT the product in T, SUM in fp32 (split
// partial results, gradients of fp32 masters), PART a pair's accumulators over a split of K, which a FWD tile adds.
enum Epi { FWD = 0, BWD = 1, OUT = 2, SUM = 3, PART = 4 };

template <class T, int RM, int RN, int WM, int WN, int EPI, bool KEPT>
struct Shape {
  static constexpr int WAVES = WM * WN, NT = 64 * WAVES, BM = 32 * RM * WM, BN = 32 * RN * WN, STEP = Elem<T>::STEP;
  static constexpr bool PAIR = EPI == FWD || EPI == BWD || EPI == PART, SWAP = Elem<T>::CHUNK == 8 && EPI != SUM;
  static constexpr int BH = PAIR ? BN / 2 : BN;            // columns of one product
  static constexpr int SH = PAIR ? RN / 2 : RN;            // 32-column fragments of one product per wave
  static constexpr int ASZ = BM * STEP, BSZ = BN * STEP, OPS = KEPT ? 0 : 2 * (ASZ + BSZ) * (int)sizeof(T);
  static constexpr int OC = EPI == FWD ? BH : BN, OLD = OC + 8;   // output columns of the tile, staged row stride
  static constexpr int STG = SWAP && EPI != PART ? BM * OLD * 2 : 0;
  static constexpr int USE = OPS > STG ? OPS : STG, LDS = USE + (PAIR ? 2 * BH * 4 : 0);   // bytes
  static_assert(!PAIR || 2 * BH <= NT, "a bias element per thread");
};

// bf16 tiles swap the operands of the matrix instruction, so that a lane holds four neighbouring columns of one row and
// stages them in LDS with one 8-byte write; fp32 results leave from the accumulators as 128-byte row pieces.
// KEPT: the products come from memory (BWD: those the forward pass kept, FWD: the splits').
//
// Bound by the matrix cores and how well they are fed where K is long.  8192 x 2048 x 8192 bf16: forward 464 us (gelu,
// 1.18 PFLOP/s; silu 447; 545 - 554 us when it keeps its products: 537 MB written), dx 438 us (1.25), dW 449 us (1.2); a
// library product of that size reaches 1.45.  The matrix cores are busy 52 - 66 % of the cycles: each SIMD has two waves,
// and what one waits for at a step's barrier the other hides only in part.  A third set of operands on the way, LDS
// filled without registers, a workgroup that walks over several tiles and loads that touch the next step's lines ahead
// were slower or equal.
// Bound by the epilogue and the latency of a tile where K is short.  25600 x 256 x 1024 bf16 (K = 4 steps, 800 tiles on
// 256 CUs, the last of them in 64-row tiles): forward 47 us (gelu 51), backward pair 73 us (gelu 78; of them the products
// 24, silu and its derivative 10, stores 10, dh 6), dx and dW 38 us each.
// The pair from kept products is bound by memory: 8192 x 2048 x 8192, 0.94 GB in 265 - 272 us.
// fp32 2500 x 257 x 515: forward 29 us, pair 12, dx and dW 24 - 26 each: 180 - 360 tiles for 256 CUs.
template <class T, int RM, int RN, int WM, int WN, bool ACOL, bool BCOL, int EPI, bool KEPT>
__device__ __forceinline__ void tile(const TileArgs& g, int block, char* smem) {
  typedef Elem<T> E;
  typedef Shape<T, RM, RN, WM, WN, EPI, KEPT> S;
  constexpr int WAVES = S::WAVES, NT = S::NT, BM = S::BM, BN = S::BN, BH = S::BH, SH = S::SH, ASZ = S::ASZ, BSZ = S::BSZ,
                OC = S::OC, OLD = S::OLD, USE = S::USE;
  constexpr bool PAIR = S::PAIR, SWAP = S::SWAP;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // steps of a segment; first and number of this split's, over all segments
  const int steps = (int)((g.K + E::STEP - 1) / E::STEP), t0 = blockIdx.y * g.chunk;
  const int total = min(g.chunk, steps * g.segs - t0);

  // two images of each operand: A0 A1 | B0 B1
  T *const ia = reinterpret_cast<T*>(smem), *const ib = ia + 2 * ASZ;
  float* const sbias = reinterpret_cast<float*>(smem + USE);   // bg, bu of the tile's columns
  // Two sets of registers: a step's operands wait in set t & 1.
  constexpr int PA = Copy<T, BM, WAVES, ACOL>::PER, PB = Copy<T, BH, WAVES, BCOL>::PER, NB = PAIR ? 2 : 1;
  u32x4 ra[2][PA], rb[2][NB][PB];
  Copy<T, BM, WAVES, ACOL> ca;
  Copy<T, BH, WAVES, BCOL> cb;
  int pm, pn;
  tile_of(block, g.tm, g.tn, pm, pn);
  const int up = !PAIR && g.tmh && pm >= g.tmh, part_row = pm * WM + wm;   // up: rows of dW's up half
  if (up) pm -= g.tmh;
  const long m0 = (long)pm * BM, n0 = (long)pn * BH;
  const long a0 = (ACOL ? m0 : m0 * g.lda) + up * g.half, b0 = BCOL ? n0 : n0 * g.ldb;
  ca.init(m0, g.M, g.lda, wave, lane);
  cb.init(n0, g.N, g.ldb, wave, lane);
  // Where the next loads of A and of B are: steps of both segments in order, then zeros.
  struct Cursor {
    const T* p;
    int left, count;   // k that remain in the segment, steps of the split
  };
  auto start = [&](const void* const* base, long at, long step, bool two) {
    const int seg = two && t0 >= steps ? 1 : 0, st = t0 - seg * steps;
    return Cursor{reinterpret_cast<const T*>(base[seg]) + at + st * step, (int)g.K - E::STEP * st, total};
  };
  auto advance = [&](Cursor& c, const void* const* base, long at, long step, bool two) {
    c.p += step;
    c.left -= E::STEP;
    if (two && c.left <= 0) {
      c.p = reinterpret_cast<const T*>(base[1]) + at;
      c.left = (int)g.K;
    }
    if (--c.count <= 0) c.left = 0;
  };
  const bool two = !PAIR && g.segs > 1;
  const long wu = PAIR ? reinterpret_cast<const T*>(g.b[1]) - reinterpret_cast<const T*>(g.b[0]) : 0;   // up rows
  Cursor at_a = start(g.a, a0, ca.step, two), at_b = start(g.b, b0, cb.step, two);
  auto load_a = [&](int set, int i) {
    ra[set][i] = ca.load(i, at_a.p, at_a.left, wave, lane);
    if (i == PA - 1) advance(at_a, g.a, a0, ca.step, two);
  };
  auto load_b = [&](int set, int i) {
    rb[set][i / PB][i % PB] = cb.load(i % PB, at_b.p + i / PB * wu, at_b.left, wave, lane);
    if (i == NB * PB - 1) advance(at_b, g.b, b0, cb.step, two);
  };
  auto load = [&](int set) {
#pragma unroll
    for (int q = 0; q < PA; ++q) load_a(set, q);
#pragma unroll
    for (int q = 0; q < NB * PB; ++q) load_b(set, q);
  };
  if constexpr (!KEPT) {
    load(0);
    load(1);
  }
  if (PAIR && tid < 2 * BH) {
    const long n = n0 + tid % BH;
    sbias[tid] = n < g.N ? g.bias.at(tid < BH ? n : g.N + n) : 0.f;
  }
  auto store_a = [&](int set, int buf, int i) { ca.store(i, ra[set][i], ia + buf * ASZ, wave, lane); };
  auto store_b = [&](int set, int buf, int i) {
    cb.store(i % PB, rb[set][i / PB][i % PB], ib + buf * BSZ + i / PB * BH * E::STEP, wave, lane);
  };
  Frags<T, BM, ACOL, RM> fa_at;
  Frags<T, BH, BCOL, SH> fb_at;
  fa_at.init(ia, 32 * wm * RM, lane);
  fb_at.init(ib, 32 * wn * SH, lane);

  f32x16 acc[RM][RN];
  // A quarter of a step: the products of fragments that are there, each fragment of A replaced by the next quarter's
  // right behind its last product, B's read into a second set; the stores and loads of a later step's operands in
  // between.  So nothing waits for LDS but the barrier of each step, which stands before its last quarter, when the
  // next step's operands are stored.  (The order is pinned: the scheduler would gather the reads and wait for them.)
  typename E::frag fa[RM], fb[2][RN];
  auto read_a = [&](int i, int s, int buf) { fa[i] = fa_at.read(i, s, buf * ASZ); };
  auto read_b = [&](int s, int buf) {
#pragma unroll
    for (int j = 0; j < RN; ++j) fb[s & 1][j] = fb_at.read(j % SH, s, buf * BSZ + (j / SH) * BH * E::STEP);
  };
  auto quarter = [&](int buf, int s) {
    if (s == 3) lds_barrier();
    const int ns = (s + 1) & 3, nbuf = s == 3 ? buf ^ 1 : buf;
    read_b(ns, nbuf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
      for (int j = 0; j < RN; ++j)
        acc[i][j] = SWAP ? E::mma(fb[s & 1][j], fa[i], acc[i][j]) : E::mma(fa[i], fb[s & 1][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
      read_a(i, ns, nbuf);
      if (s == 1) {
#pragma unroll
        for (int q = i * PA / RM; q < (i + 1) * PA / RM; ++q) {
          store_a(buf ^ 1, buf ^ 1, q);
          load_a(buf ^ 1, q);
        }
      }
      if (s == 2) {
#pragma unroll
        for (int q = i * NB * PB / RM; q < (i + 1) * NB * PB / RM; ++q) {
          store_b(buf ^ 1, buf ^ 1, q);
          load_b(buf ^ 1, q);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (!KEPT) {
#pragma unroll
  for (int q = 0; q < PA; ++q) store_a(0, 0, q);
#pragma unroll
  for (int q = 0; q < NB * PB; ++q) store_b(0, 0, q);
  load(0);
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  lds_barrier();
#pragma unroll
  for (int i = 0; i < RM; ++i) read_a(i, 0, 0);
  read_b(0, 0);
  // Steps go in pairs without a branch between them (an odd count ends with a step of zeros): across a branch the
  // compiler waits for every load that either side may have sent.
  for (int t = 0; t < total; t += 2) {
#pragma unroll
    for (int s = 0; s < 4; ++s) quarter(0, s);
#pragma unroll
    for (int s = 0; s < 4; ++s) quarter(1, s);
  }
  }

  // ---- epilogue
  if constexpr (PAIR) {
    constexpr int Q = RM * RN * 4;   // four accumulators each
    const long at = ((long)pm * g.tn + pn) * Q * NT + tid;
    auto quad = [&](int k) {
      const f32x16& c = acc[k / 4 / RN][k / 4 % RN];
      const int e = k % 4 * 4;
      return f32x4{c[e], c[e + 1], c[e + 2], c[e + 3]};
    };
    if constexpr (KEPT) {
      const f32x4* from = reinterpret_cast<const f32x4*>(EPI == FWD ? g.splits : g.saved) + at;
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const f32x4 v = from[k * NT];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[k / 4 / RN][k / 4 % RN][k % 4 * 4 + e] = v[e];
      }
      if constexpr (EPI == FWD) {
        for (int z = 1; z < g.nsplits; ++z) {
          from += g.slab / 4;
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const f32x4 v = from[k * NT];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[k / 4 / RN][k / 4 % RN][k % 4 * 4 + e] += v[e];
          }
        }
      }
    }
    float* to = EPI == PART ? g.splits + blockIdx.y * g.slab : EPI == FWD ? g.saved : nullptr;
    if (to) {
#pragma unroll
      for (int k = 0; k < Q; ++k) reinterpret_cast<f32x4*>(to)[at + k * NT] = quad(k);
    }
    if constexpr (KEPT) __syncthreads();   // the biases are stored
  }
  if constexpr (EPI != PART) {
  // bf16 backward: the tile of dh passes through registers, in 16-byte pieces at any alignment (rows may end inside one)
  constexpr int DPT = EPI == BWD && SWAP ? BM * BH / 8 / NT : 1;
  s16x8 dh[DPT];
  if constexpr (EPI == BWD && SWAP) {
#pragma unroll
    for (int q = 0; q < DPT; ++q) {
      const int idx = q * NT + tid, row = idx / (BH / 8), c = idx % (BH / 8) * 8;
      dh[q] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (m0 + row < g.M && n0 + c < g.N) {
        const short* p = reinterpret_cast<const short*>(g.dh) + (m0 + row) * g.lddh + n0 + c;
        const int left = (int)min(g.N - n0 - c, 8L);
        if (left == 8) {
          dh[q] = *reinterpret_cast<const s16x8_any*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < 7; ++e) dh[q][e] = e < left ? p[min(e, left - 1)] : (short)0;
        }
      }
    }
  }
  if constexpr (!SWAP) {
    auto finish = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    const int row0 = 32 * wm * RM + 4 * (lane >> 5);
    const long left = g.M - m0 - row0;
#pragma unroll
    for (int j = 0; j < SH; ++j) {
      const int col = 32 * (wn * SH + j) + (lane & 31);
      const long n = n0 + col;
      const bool in = n < g.N;
      float* o = reinterpret_cast<float*>(g.out) + blockIdx.y * g.slab + (m0 + row0 + up * g.M) * g.ldo + n;
      const float* dv = EPI == BWD ? reinterpret_cast<const float*>(g.dh) + (m0 + row0) * g.lddh + n : nullptr;
      const float bg = PAIR ? sbias[col] : 0.f, bu = PAIR ? sbias[BH + col] : 0.f;
      float sg = 0.f, su = 0.f;
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 32 * i + acc_row(r, 0), next = r == 15 ? 32 * (i + 1) : 32 * i + acc_row(r + 1, 0);
          if (in && row < left) {
            if constexpr (EPI == BWD) {
              float a, d;
              act_both<ACT, true>(acc[i][j][r] + bg, a, d);
              const float u = acc[i][j + SH][r] + bu;
              const float dg = *dv * u * d, du = *dv * a;
              o[0] = dg;
              o[g.half] = du;
              sg += dg;
              su += du;
            } else if constexpr (EPI == FWD) {
              *o = act_fwd<ACT, true>(acc[i][j][r] + bg) * (acc[i][j + SH][r] + bu);
            } else {
              *o = acc[i][j][r];
            }
          } else if (EPI == BWD && n >= g.N && n < g.half && row < left) {
            o[0] = o[g.half] = 0.f;   // the padding is an operand of dx
          }
          o += (next - row) * g.ldo;
          if (EPI == BWD) dv += (next - row) * g.lddh;
        }
      if (EPI == BWD && g.part) {
        sg += __shfl_xor(sg, 32);
        su += __shfl_xor(su, 32);
        if (lane < 32 && in) {
          g.part[(long)part_row * 2 * g.half + n] = sg;
          g.part[(long)part_row * 2 * g.half + g.half + n] = su;
        }
      }
    }
    };
    by_act<PAIR>(g.act, finish);
  } else {
    short* stage = reinterpret_cast<short*>(smem);
    lds_barrier();   // the operand images are free
    if constexpr (EPI == BWD) {
#pragma unroll
      for (int q = 0; q < DPT; ++q) {
        const int idx = q * NT + tid, row = idx / (BH / 8), c = idx % (BH / 8) * 8;
        *reinterpret_cast<s16x8*>(stage + row * OLD + c) = dh[q];
      }
      lds_barrier();
    }
    auto finish = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    const long left = g.M - m0 - 32 * wm * RM;   // rows of the matrix from this wave's first on
#pragma unroll
    for (int j = 0; j < SH; ++j) {
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int col = 32 * (wn * SH + j) + 8 * rg + 4 * (lane >> 5);   // this lane's four columns
        f32x4 bg, bu;
        float sg[4] = {0.f, 0.f, 0.f, 0.f}, su[4] = {0.f, 0.f, 0.f, 0.f};
        if (PAIR) {
          bg = *reinterpret_cast<const f32x4*>(sbias + col);
          bu = *reinterpret_cast<const f32x4*>(sbias + BH + col);
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          short* p = stage + (32 * (wm * RM + i) + (lane & 31)) * OLD + col;
          s16x4 v, w;
          if constexpr (EPI == BWD) w = *reinterpret_cast<const s16x4*>(p);
          const bool in = 32 * i + (lane & 31) < left;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float c = acc[i][j][4 * rg + e];
            if constexpr (EPI == OUT) {
              v[e] = to_s(c);
            } else if constexpr (EPI == FWD) {
              v[e] = to_s(act_fwd<ACT, false>(c + bg[e]) * (acc[i][j + SH][4 * rg + e] + bu[e]));
            } else {
              // columns outside have dh = 0
              float a, d;
              act_both<ACT, false>(c + bg[e], a, d);
              const float x = to_f((short)w[e]);
              const float dg = x * (acc[i][j + SH][4 * rg + e] + bu[e]) * d, du = x * a;
              v[e] = to_s(dg);
              w[e] = to_s(du);
              sg[e] += in ? dg : 0.f;   // not by dh = 0: a row outside has g, u = 0 w, NaN where w is infinite
              su[e] += in ? du : 0.f;
            }
          }
          *reinterpret_cast<s16x4*>(p) = v;
          if constexpr (EPI == BWD) *reinterpret_cast<s16x4*>(p + BH) = w;
        }
        if (EPI == BWD && g.part) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sg[e] = half_wave_sum(sg[e]);
            su[e] = half_wave_sum(su[e]);
          }
          if ((lane & 31) == 31 && n0 + col < g.half) {
            float* row = g.part + (long)part_row * 2 * g.half + n0 + col;
            *reinterpret_cast<f32x4*>(row) = f32x4{sg[0], sg[1], sg[2], sg[3]};
            *reinterpret_cast<f32x4*>(row + g.half) = f32x4{su[0], su[1], su[2], su[3]};
          }
        }
      }
    }
    };
    by_act<PAIR>(g.act, finish);
    lds_barrier();
    // rows of the staged tile leave in 16-byte pieces; dgu rows are padded to whole pieces (with zeros), others may end
    // inside one or start off 16 bytes
    const long cols = EPI == BWD ? g.half : g.N;
    bf16* out = reinterpret_cast<bf16*>(g.out);
    const bool vec = ((uintptr_t)out % 16 == 0) && g.ldo % 8 == 0;
    for (int idx = tid; idx < BM * (OC / 8); idx += NT) {
      const int row = idx / (OC / 8), c = idx % (OC / 8) * 8;
      const long m = m0 + row, n = n0 + (EPI == BWD ? c % BH : c);
      if (m >= g.M || n >= cols) continue;
      const short* src = stage + row * OLD + c;
      bf16* dst = out + (m + up * g.M) * g.ldo + n + (EPI == BWD && c >= BH ? g.half : 0);
      if (vec && n + 8 <= cols) {
        *reinterpret_cast<s16x8*>(dst) = *reinterpret_cast<const s16x8*>(src);
      } else {
        for (int e = 0; e < 8 && n + e < cols; ++e) dst[e] = __builtin_bit_cast(bf16, src[e]);
      }
    }
  }
  }
}

template <class T, int RM, int RN, int WM, int WN, bool ACOL, bool BCOL, int EPI, bool KEPT>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(TileArgs g) {
  __shared__ __attribute__((aligned(1024))) char smem[Shape<T, RM, RN, WM, WN, EPI, KEPT>::LDS];
  tile<T, RM, RN, WM, WN, ACOL, BCOL, EPI, KEPT>(g, blockIdx.x, smem);
}

// A pair's rows in two parts: `first` tiles of 256 rows, and tiles of 64 rows behind them in the same launch.
template <class T, int EPI, bool KEPT>
__global__ __launch_bounds__(512, 2) void two_part_kernel(TileArgs g, TileArgs tail, int first) {
  __shared__ __attribute__((aligned(1024))) char smem[Shape<T, 4, 2, 2, 4, EPI, KEPT>::LDS];
  static_assert(Shape<T, 1, 2, 2, 4, EPI, KEPT>::LDS <= sizeof(smem), "tile");
  if ((int)blockIdx.x < first) tile<T, 4, 2, 2, 4, false, false, EPI, KEPT>(g, blockIdx.x, smem);
  else tile<T, 1, 2, 2, 4, false, false, EPI, KEPT>(tail, blockIdx.x - first, smem);
}

// ---------------------------------------------------------------------------------------------------------------

// Few rows (M <= 16 MF): bound by reading the weights once.  A workgroup takes 16 columns of F and all rows; its 8 waves
// take the k steps of 32 in turn (512 contiguous bytes of every weight row at a time), weights and rows straight from
// memory into v_mfma_f32_16x16x32_bf16 fragments, and add their sums in LDS in order.  Rows and columns past the ends
// repeat the last one: their results are not stored.  8 x 2048 x 8192: 14 us (67 MB of weights, 4.8 TB/s); 1 x 256 x 1024:
// 4.2 us (latency).
template <int MF, int ACT>
__global__ __launch_bounds__(512) void rows_kernel(const bf16* x, long ldx, const bf16* w, long ldw, Bias bias, bf16* h, int M,
                                                   int K, long F) {
  __shared__ f32x4 red[8][2][MF][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const long f0 = (long)blockIdx.x * 16, fr = f0 + r < F ? f0 + r : F - 1;
  const bf16 *wg = w + fr * ldw, *wu = wg + F * ldw;
  const bf16* xr[MF];
  f32x4 g[MF], u[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    xr[i] = x + (long)min(16 * i + r, M - 1) * ldx;
    g[i] = u[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const bf16x8 zero = {};
#pragma unroll 4
  for (int k0 = 32 * wave; k0 < K; k0 += 256) {
    const int k = k0 + 8 * q, kc = k < K ? k : 0;
    const bf16x8 a = *reinterpret_cast<const bf16x8*>(wg + kc), b = *reinterpret_cast<const bf16x8*>(wu + kc);
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const bf16x8 c = *reinterpret_cast<const bf16x8*>(xr[i] + kc);
      g[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k < K ? a : zero, k < K ? c : zero, g[i], 0, 0, 0);
      u[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k < K ? b : zero, k < K ? c : zero, u[i], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    red[wave][0][i][lane] = g[i];
    red[wave][1][i][lane] = u[i];
  }
  __syncthreads();
  if (wave >= MF) return;
  const int m = 16 * wave + r;   // this lane: row m, columns f0 + 4 q ..
  const long f = f0 + 4 * q;
  f32x4 sg = red[0][0][wave][lane], su = red[0][1][wave][lane];
#pragma unroll
  for (int z = 1; z < 8; ++z) {
    sg += red[z][0][wave][lane];
    su += red[z][1][wave][lane];
  }
  if (m >= M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (f + e < F) h[m * F + f + e] = __float2bfloat16(act_fwd<ACT, false>(sg[e] + bias.at(f + e)) * (su[e] + bias.at(F + f + e)));
}

// dst [rows + rows2][ldd]: the rows of src and of src2, zeros behind each.
template <class T>
__global__ __launch_bounds__(256) void pad_kernel(const T* src, long lds_, long rows, const T* src2, long lds2, long rows2,
                                                  T* dst, long ldd, long cols) {
  const long n = (rows + rows2) * ldd;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / ldd, c = i - r * ldd;
    dst[i] = c >= cols ? T(0.f) : r < rows ? src[r * lds_ + c] : src2[(r - rows) * lds2 + c];
  }
}

// out[i] = sum over the splits' partial results, in a fixed order (16 of 2048 x 256: 6.7 us, 5.2 TB/s).
__global__ __launch_bounds__(256) void splits_kernel(const float* slabs, long slab, int splits, long n, void* out, int out_bf) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < splits; ++z) s += slabs[z * slab + i];
    if (out_bf) reinterpret_cast<bf16*>(out)[i] = __float2bfloat16(s);
    else reinterpret_cast<float*>(out)[i] = s;
  }
}

// out[c] = sum over the partial rows [gate F, padding | up F, padding]: 16 columns x 16 row phases a workgroup, phases added
// in order.
__global__ __launch_bounds__(256) void colsum_kernel(const float* part, long rows, long F, long half, void* out, int out_bf) {
  __shared__ float red[16][17];
  const int cl = threadIdx.x & 15, ph = threadIdx.x >> 4;
  const long c = (long)blockIdx.x * 16 + cl, at = c < F ? c : c - F + half;
  float s = 0.f;
  if (c < 2 * F) {
#pragma unroll 4
    for (long z = ph; z < rows; z += 16) s += part[z * 2 * half + at];
  }
  red[ph][cl] = s;
  __syncthreads();
  if (ph || c >= 2 * F) return;
#pragma unroll
  for (int q = 1; q < 16; ++q) s += red[q][cl];
  if (out_bf) reinterpret_cast<bf16*>(out)[c] = __float2bfloat16(s);
  else reinterpret_cast<float*>(out)[c] = s;
}

static long up8(long n) { return (n + 7) / 8 * 8; }
static long tiles(long n, long t) { return (n + t - 1) / t; }
static unsigned flat_grid(long n) { return (unsigned)std::max<long>(1, std::min<long>((n + 255) / 256, 4096)); }

static void check_sizes(long M, long D, long F, int act) {
  GSC_CHECK(M >= 1 && D >= 1 && F >= 1 && M <= 0x7fffffffL && D <= 1000000L && F <= 1000000L,
            "gated_linear: rows must be in 1 .. 2^31 - 1, D and F in 1 .. 1,000,000");
  GSC_CHECK(act >= 0 && act <= 2, "gated_linear: unknown activation");
}

// Operands of the tiles: 16-byte aligned rows; 256 of them within the 2^31 bytes of a descriptor.
static void check_operand(uintptr_t p, long ld) {
  GSC_CHECK(p % 16 == 0 && ld % 8 == 0 && ld <= 2000000L, "gated_linear: an operand needs 16-byte aligned rows of at most 2,000,000 elements");
}

static int cu_count() {
  static const int n = [] {
    int dev = 0, v = 256;
    if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev);
    return v > 0 ? v : 256;
  }();
  return n;
}

template <class T, int RM, int RN, int WM, int WN, bool ACOL, bool BCOL, int EPI, bool KEPT = false>
static void launch(TileArgs g, int splits, hipStream_t s) {
  constexpr int BM = 32 * RM * WM, BH = EPI == SUM || EPI == OUT ? 32 * RN * WN : 16 * RN * WN;
  const long tm = tiles(g.M, BM), tn = tiles(g.N, BH);
  GSC_CHECK((g.tmh ? 2 : 1) * tm * tn * (64 * WM * WN) <= 0xffffffffL, "gated_linear: too many tiles");   // threads of a grid
  if (g.tmh) g.tmh = (int)tm;
  g.tm = (int)(g.tmh ? 2 * tm : tm);
  g.tn = (int)tn;
  const int all = (int)(tiles(g.K, Elem<T>::STEP) * g.segs);
  g.chunk = (int)tiles(all, splits);
  hipLaunchKernelGGL((tile_kernel<T, RM, RN, WM, WN, ACOL, BCOL, EPI, KEPT>), dim3((unsigned)(g.tm * g.tn), (unsigned)tiles(all, g.chunk)),
                     dim3(64 * WM * WN), 0, s, g);
  check_launch();
}

// Rows of a product's tiles (M x N results, bn columns to 256 rows): 256 where those fill the CUs (forward of 8192 x 2048 x
// 8192 bf16: 486 us, 613 us on 128 rows), 128 otherwise (dW of 25600 x 256 x 1024 in splits: 39 + 7 us, on 256 rows 44 +
// 12 us in 31 splits, 49 + 7 us in 16), and for
// fp32 64 where 128 x 128 tiles leave CUs idle (a step of one keeps a CU's matrix cores 4096 cycles; dx and dW of
// 2500 x 120 x 520: 30 us on 128 rows, 19 us on 64; large products need the larger tiles' reuse: 64 x 64 alone would read
// 9 TB/s).
static int tile_rows(int bf, long M, long N, long bn) {
  if (tiles(M, 256) * tiles(N, bn) >= cu_count()) return 256;
  return bf || tiles(M, 128) * tiles(N, bn / 2) >= cu_count() ? 128 : 64;
}
static int pair_rows(int bf, long M, long F) { return tile_rows(bf, M, F, 128); }

// Rows of a bf16 pair in tiles of 256 rows: all, or as many tile rows as fill whole rounds of the CUs, where 64-row tiles of
// the others fill no more than one: 25600 x 256 x 1024 is 3.1 rounds; forward 51 us in 256-row tiles alone, 48 us in two
// parts, backward pair 82 and 73 us (128-row tiles behind: 49 and 76 us).
constexpr long kTail = 64;
static long full_rows(int bf, long M, long F) {
  if (!bf || pair_rows(bf, M, F) != 256) return M;
  const long tm = tiles(M, 256), tn = tiles(F, 128), cus = cu_count(), full = tm * tn / cus * cus / tn;
  return full < tm && tiles(M - 256 * full, kTail) * tn <= cus ? 256 * full : M;
}
// Partial rows of the bias gradient: two wave rows a tile.
static long part_rows(int bf, long M, long F) {
  const long full = full_rows(bf, M, F);
  return 2 * (tiles(full, pair_rows(bf, M, F)) + tiles(M - full, kTail));
}

// Most rows of the few-rows kernel (2048 x 8192 bf16, it and the tiles: 8 rows 13 and 21 us, 32 rows 18 and 20, 64 rows 26
// and 21).
constexpr long kRows = 32;

// Whether the forward pass keeps its products: 8 bytes a result written and read again at 4.7 TB/s against 4 D operations
// at 1.15 PFLOP/s (bf16) or 0.13 (fp32): from D = 1,000 or 110.  (8192 x 2048 x 8192: backward pair 557 us recomputing,
// 270 us from the kept products, forward 464 -> 545 us; 25600 x 256 x 1024: 82 us recomputing, 210 MB kept.)
static bool saves(int bf, long M, long D) { return D >= (bf ? 1024 : 128) && !(bf && M <= kRows); }

// fp32 elements of the kept products, 0 where nothing is kept.
long saved_elements(int bf, long M, long D, long F) {
  if (!saves(bf, M, D)) return 0;
  const long r = pair_rows(bf, M, F), full = full_rows(bf, M, F);
  return (tiles(full, r) * r + tiles(M - full, kTail) * kTail) * tiles(F, r == 256 ? 128 : 64) * (r == 256 ? 256 : 128);
}

// fp32 elements of a split's accumulators.
static long pair_slab(int bf, long M, long F) {
  const int r = pair_rows(bf, M, F);
  return tiles(M, r) * r * tiles(F, 64) * 128;
}

// Splits of a pair's K where its tiles are few: n of them divide the steps of a tile (0.53 us each in bf16, 2.2 or, on 64
// rows, 1.1 in fp32) by n and cost n times the accumulators of a tile read by one workgroup (0.12 TB/s), n times all of them
// written and read (4.7 TB/s) and about 6 us for the second launch: the n where both are equal, at least two steps each, and
// workgroups for two per CU in bf16, for one in fp32 (whose steps are bound by the matrix cores); not on more than a quarter
// of the CUs in bf16, where the weights already come at the rate of the memory.  In one piece and as called:
//   100 x 4096 x 256    bf16 34 us, 20 (7 pieces)   fp32 146, 23      512 x 4096 x 1024   bf16 36 us, 25 (4)   fp32 155, 90
//   64 x 2048 x 512     bf16 19 us, 14              fp32 74, 18       300 x 2048 x 1024   bf16 20 us, not split (23 in 6)
//   128 x 8192 x 512    bf16 64 us, 30              fp32 288, 43      200 x 4096 x 8192   bf16 41 us, not split (44 in 2)
static int pair_splits(int bf, long M, long D, long F) {
  const int r = pair_rows(bf, M, F);
  const long steps = tiles(up8(D), bf ? 64 : 32), t = tiles(M, r) * tiles(F, 64), cus = cu_count();
  if (r == 256 || (bf && (M <= kRows || 4 * t > cus))) return 1;
  const double all = steps * (bf ? 0.53 : r / 64 * 1.1);
  const double each = r * 128 * 4 / 0.12e6 + pair_slab(bf, M, F) * 8 / 4.7e6;
  const long n = std::min<long>({(long)(std::sqrt(all / each) + 0.5), (bf ? 2 : 1) * cus / t, steps / 2});
  return n > 1 && all - all / n > 6 + n * each ? (int)tiles(steps, tiles(steps, n)) : 1;
}
// fp32 elements of the forward pass's workspace (0: none).
long forward_space(int bf, long M, long D, long F) {
  check_sizes(M, D, F, 0);
  const int n = pair_splits(bf, M, D, F);
  return n > 1 ? n * pair_slab(bf, M, F) : 0;
}

// Both parts of a pair in one launch: `full` rows in tiles of 256, the others in tiles of kTail.
template <int EPI, bool KEPT>
static void two_parts(TileArgs g, long full, hipStream_t s) {
  TileArgs tail = g;
  g.tn = tail.tn = (int)tiles(g.N, 128);
  g.tm = (int)(full / 256);
  tail.tm = (int)tiles(g.M - full, kTail);
  g.M = full;
  tail.M -= full;
  g.chunk = tail.chunk = (int)tiles(g.K, Elem<bf16>::STEP);
  tail.a[0] = reinterpret_cast<const bf16*>(g.a[0]) + full * g.lda;
  tail.dh = g.dh ? reinterpret_cast<const bf16*>(g.dh) + full * g.lddh : nullptr;
  tail.out = reinterpret_cast<bf16*>(g.out) + full * g.ldo;
  tail.part = g.part ? g.part + 2 * (long)g.tm * 2 * g.half : nullptr;
  tail.saved = g.saved ? g.saved + full * g.tn * 256 : nullptr;
  const long first = (long)g.tm * g.tn, blocks = first + (long)tail.tm * tail.tn;
  GSC_CHECK(blocks * 512 <= 0xffffffffL, "gated_linear: too many tiles");
  hipLaunchKernelGGL((two_part_kernel<bf16, EPI, KEPT>), dim3((unsigned)blocks), dim3(512), 0, s, g, tail, (int)first);
  check_launch();
}

template <class T, int EPI, bool KEPT = false>
static void pair(const TileArgs& g, hipStream_t s) {
  constexpr bool SPLIT = EPI == PART || (EPI == FWD && KEPT);   // never in 256-row tiles
  if constexpr (sizeof(T) == 2 && !SPLIT) {
    const long full = full_rows(1, g.M, g.N);
    if (full < g.M) return two_parts<EPI, KEPT>(g, full, s);
  }
  const int splits = EPI == PART ? g.nsplits : 1;
  switch (pair_rows(sizeof(T) == 2, g.M, g.N)) {
    case 256:
      if constexpr (!SPLIT) launch<T, 4, 2, 2, 4, false, false, EPI, KEPT>(g, 1, s);
      break;
    case 128: launch<T, 2, 2, 2, 2, false, false, EPI, KEPT>(g, splits, s); break;
    default:
      if constexpr (sizeof(T) == 4) launch<T, 1, 2, 2, 2, false, false, EPI, KEPT>(g, splits, s);
  }
}
// The plain products on the same tiles.
template <class T, bool ACOL, bool BCOL, int EPI>
static void product(const TileArgs& g, int rows, int splits, hipStream_t s) {
  switch (rows) {
    case 256: launch<T, 4, 2, 2, 4, ACOL, BCOL, EPI>(g, splits, s); break;
    case 128: launch<T, 2, 2, 2, 2, ACOL, BCOL, EPI>(g, splits, s); break;
    default:
      if constexpr (sizeof(T) == 4) launch<T, 1, 1, 2, 2, ACOL, BCOL, EPI>(g, splits, s);
  }
}

static TileArgs pair_args(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, long M, long D,
                          long F, int act) {
  check_sizes(M, D, F, act);
  check_operand(x, ldx);
  check_operand(w, ldw);
  TileArgs g{};
  g.a[0] = ptr<const void>(x);
  g.b[0] = ptr<const void>(w);
  g.b[1] = ptr<const void>(w + F * ldw * (bf ? 2 : 4));
  g.lda = ldx;
  g.ldb = ldw;
  g.segs = 1;
  g.M = M;
  g.N = F;
  g.K = up8(D);   // rows are padded with zeros
  g.bias = Bias{ptr<const void>(bias), bias_bf};
  g.act = act;
  return g;
}

// work: n splits' accumulators (n > 1).
static void run_forward(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t h,
                        uintptr_t saved, long saved_size, uintptr_t work, int n, long M, long D, long F, int act,
                        uintptr_t stream) {
  TileArgs g = pair_args(x, ldx, w, ldw, bf, bias, bias_bf, M, D, F, act);
  g.out = ptr<void>(h);
  g.ldo = F;
  g.saved = ptr<float>(saved);
  GSC_CHECK(!saved || saves(bf, M, D), "gated_linear: these products are not kept");
  GSC_CHECK(!saved || saved_size >= saved_elements(bf, M, D, F), "gated_linear: too little space for the kept products");
  const hipStream_t s = stream_of(stream);
  if (bf && M <= kRows) {
    by_act<true>(act, [&](auto a) {
      constexpr int ACT = decltype(a)::value;
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)tiles(F, 16)), dim3(512), 0, s, ptr<const bf16>(x), ldx,
                           ptr<const bf16>(w), ldw, g.bias, ptr<bf16>(h), (int)M, (int)g.K, F);
      };
      if (M <= 16) go(rows_kernel<1, ACT>);
      else go(rows_kernel<2, ACT>);
    });
    check_launch();
  } else if (n > 1) {
    g.splits = ptr<float>(work);
    g.nsplits = n;
    g.slab = pair_slab(bf, M, F);
    if (bf) pair<bf16, PART>(g, s), pair<bf16, FWD, true>(g, s);
    else pair<float, PART>(g, s), pair<float, FWD, true>(g, s);
  } else {
    if (bf) pair<bf16, FWD>(g, s);
    else pair<float, FWD>(g, s);
  }
}
// Without gradients, K in one piece.
void forward(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t h, uintptr_t saved,
             long M, long D, long F, int act, uintptr_t stream) {
  GSC_CHECK(!saved, "gated_linear: this forward pass keeps no products");
  run_forward(x, ldx, w, ldw, bf, bias, bias_bf, h, 0, 0, 0, 1, M, D, F, act, stream);
}
// Keeps its products in saved (saved_size elements; 0: does not) and splits K through work (work_size elements, at least
// forward_space()).
void forward_split(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t h,
                   uintptr_t saved, long saved_size, uintptr_t work, long work_size, long M, long D, long F, int act,
                   uintptr_t stream) {
  const long need = forward_space(bf, M, D, F);
  GSC_CHECK(!need || (work && work_size >= need), "gated_linear: too little workspace for the forward pass");
  run_forward(x, ldx, w, ldw, bf, bias, bias_bf, h, saved, saved_size, work, need ? pair_splits(bf, M, D, F) : 1, M, D, F, act,
              stream);
}

void pad(uintptr_t src, long lds_, long rows, uintptr_t src2, long lds2, long rows2, uintptr_t dst, long ldd, int bf, long cols,
         uintptr_t stream) {
  GSC_CHECK(rows >= 1 && rows2 >= 0 && cols >= 1 && cols <= ldd, "gated_linear: pad");
  const hipStream_t s = stream_of(stream);
  auto go = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(pad_kernel<T>, dim3(flat_grid((rows + rows2) * ldd)), dim3(256), 0, s, ptr<const T>(src), lds_, rows,
                       ptr<const T>(src2), lds2, rows2, ptr<T>(dst), ldd, cols);
  };
  if (bf) go((bf16*)nullptr);
  else go((float*)nullptr);
  check_launch();
}

// dgu rows [dg, zeros to a multiple of 8 | du, zeros] from x, the weights and dh; part (absent: no bias gradient) takes
// the column sums' partial rows.
static void backward_pair(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t dh, long lddh,
                   uintptr_t dgu, uintptr_t part, uintptr_t db, int db_bf, uintptr_t saved, long M, long D, long F, int act,
                   uintptr_t stream) {
  TileArgs g = pair_args(x, ldx, w, ldw, bf, bias, bias_bf, M, D, F, act);
  const hipStream_t s = stream_of(stream);
  g.dh = ptr<const void>(dh);
  g.lddh = lddh;
  g.out = ptr<void>(dgu);
  g.half = up8(F);
  g.ldo = 2 * g.half;
  g.part = db ? ptr<float>(part) : nullptr;
  g.saved = ptr<float>(saved);
  GSC_CHECK((saved != 0) == (saved_elements(bf, M, D, F) != 0), "gated_linear: the kept products of the forward pass");
  if (saved) {
    if (bf) pair<bf16, BWD, true>(g, s);
    else pair<float, BWD, true>(g, s);
  } else {
    if (bf) pair<bf16, BWD>(g, s);
    else pair<float, BWD>(g, s);
  }
  if (db) {
    hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)tiles(2 * F, 16)), dim3(256), 0, s, ptr<const float>(part),
                       part_rows(bf, M, F), F, g.half, ptr<void>(db), db_bf);
    check_launch();
  }
}

// Splits of a product's K (t tiles, `outputs` results): n splits divide the time of a tile's steps (0.7 us
// each, of 64) by n and cost n fp32 results written and read again (4 TB/s): the n where the two are equal, two workgroups
// per CU and at least 4 steps each.  dX of 256 / 2560 rows of 256 x 1024: 22.5 / 22.8 us unsplit, 10.8 / 17 us split;
// of 25,600 rows 40 us unsplit, 58 us in two.
static int k_splits(long t, long K, long outputs) {
  const double n = std::sqrt((double)K / 64 * 0.7e-6 / ((double)outputs * 8 / 4e12));
  return (int)std::max<long>(1, std::min<long>({(long)(n + 0.5), (2L * cu_count() + t - 1) / t, K / 256, 64}));
}

static int x_splits(int bf, long M, long D, long F) {
  const int r = tile_rows(bf, M, D, 256);
  return r == 256 ? 1 : k_splits(tiles(M, r) * tiles(D, r), 2 * F, M * D);
}
static void add_splits(uintptr_t slabs, const TileArgs& g, int bf, int splits, long n, uintptr_t out, int out_bf, hipStream_t s) {
  const long all = tiles(g.K, bf ? 64 : 32) * g.segs;
  hipLaunchKernelGGL(splits_kernel, dim3(flat_grid(n)), dim3(256), 0, s, ptr<const float>(slabs), n,
                     (int)tiles(all, tiles(all, splits)), n, ptr<void>(out), out_bf);
  check_launch();
}

static void backward_x(uintptr_t dgu, uintptr_t w, long ldw, int bf, uintptr_t dx, int dx_bf, uintptr_t slabs, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  check_operand(dgu, 2 * up8(F));
  check_operand(w, ldw);
  const int es = bf ? 2 : 4, splits = x_splits(bf, M, D, F);
  GSC_CHECK(bf || !dx_bf, "gated_linear: fp32 operands give fp32 gradients");
  TileArgs g{};
  g.a[0] = ptr<const void>(dgu);
  g.a[1] = ptr<const void>(dgu + up8(F) * es);
  g.b[0] = ptr<const void>(w);
  g.b[1] = ptr<const void>(w + F * ldw * es);
  g.lda = 2 * up8(F);
  g.ldb = ldw;
  g.segs = 2;
  g.M = M;
  g.N = D;
  g.K = F;
  g.out = ptr<void>(splits > 1 ? slabs : dx);
  g.ldo = D;
  g.slab = M * D;
  const int rows = tile_rows(bf, M, D, 256);
  if (!bf) product<float, false, true, SUM>(g, rows, splits, s);
  else if (splits > 1 || !dx_bf) product<bf16, false, true, SUM>(g, rows, splits, s);
  else product<bf16, false, true, OUT>(g, rows, splits, s);
  if (splits > 1) add_splits(slabs, g, bf, splits, M * D, dx, dx_bf, s);
}

static int w_splits(int bf, long M, long D, long F) {
  const int r = tile_rows(bf, 2 * F, D, 256);
  return r == 256 ? 1 : k_splits(2 * tiles(F, r) * tiles(D, r), M, 2 * F * D);
}

static void backward_w(uintptr_t dgu, uintptr_t x, long ldx, int bf, uintptr_t dw, int dw_bf, uintptr_t slabs, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  check_operand(dgu, 2 * up8(F));
  check_operand(x, ldx);
  const int splits = w_splits(bf, M, D, F);
  GSC_CHECK(bf || !dw_bf, "gated_linear: fp32 operands give fp32 gradients");
  TileArgs g{};
  g.a[0] = ptr<const void>(dgu);
  g.b[0] = ptr<const void>(x);
  g.lda = 2 * up8(F);
  g.ldb = ldx;
  g.segs = 1;
  g.M = F;
  g.N = D;
  g.K = M;
  g.half = up8(F);
  g.tmh = 1;
  g.ldo = D;
  g.slab = 2 * F * D;
  g.out = ptr<void>(splits > 1 ? slabs : dw);
  const int rows = tile_rows(bf, 2 * F, D, 256);
  if (!bf) product<float, true, true, SUM>(g, rows, splits, s);
  else if (splits > 1 || !dw_bf) product<bf16, true, true, SUM>(g, rows, splits, s);
  else product<bf16, true, true, OUT>(g, rows, splits, s);
  if (splits > 1) add_splits(slabs, g, bf, splits, 2 * F * D, dw, dw_bf, s);
}

// The backward pass's workspace: dgu, the bias gradient's partial sums, and the partial results of dx and dW, which one
// stretch serves in turn.  Offsets in bytes.
struct Space {
  long part, slabs, size;
};
static Space space_of(int bf, long M, long D, long F, bool need_x, bool need_w, bool need_b) {
  auto up = [](long n) { return (n + 255) / 256 * 256; };
  const int xs = need_x ? x_splits(bf, M, D, F) : 1, ws = need_w ? w_splits(bf, M, D, F) : 1;
  Space sp;
  sp.part = up(M * 2 * up8(F) * (bf ? 2 : 4));
  sp.slabs = sp.part + (need_b ? up(part_rows(bf, M, F) * 2 * up8(F) * 4) : 0);
  sp.size = sp.slabs + 4 * std::max(xs > 1 ? xs * M * D : 0, ws > 1 ? ws * 2 * F * D : 0);
  return sp;
}
long workspace(int bf, long M, long D, long F, bool need_x, bool need_w, bool need_b) {
  check_sizes(M, D, F, 0);
  return space_of(bf, M, D, F, need_x, need_w, need_b).size;
}

// dx, dw, db (0: not asked for) from x, the weights, dh and the kept products (saved_size elements; 0: computed again), in
// work_size bytes of workspace.
void backward(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t dh, long lddh,
              uintptr_t saved, long saved_size, uintptr_t dx, int dx_bf, uintptr_t dw, int dw_bf, uintptr_t db, int db_bf,
              uintptr_t work, long work_size, long M, long D, long F, int act, uintptr_t stream) {
  check_sizes(M, D, F, act);
  const Space sp = space_of(bf, M, D, F, dx != 0, dw != 0, db != 0);
  GSC_CHECK(work && work_size >= sp.size, "gated_linear: too little workspace for the backward pass");
  GSC_CHECK(!saved || saved_size >= saved_elements(bf, M, D, F), "gated_linear: too few kept products");
  const uintptr_t dgu = work, slabs = work + sp.slabs;
  backward_pair(x, ldx, w, ldw, bf, bias, bias_bf, dh, lddh, dgu, work + sp.part, db, db_bf, saved, M, D, F, act, stream);
  if (dx) backward_x(dgu, w, ldw, bf, dx, dx_bf, slabs, M, D, F, stream);
  if (dw) backward_w(dgu, x, ldx, bf, dw, dw_bf, slabs, M, D, F, stream);
}

}  // namespace gated

void register_gated(py::module_& m) {
  m.def("gated_forward", &gated::forward, "h = act(x Wg^T + bg) * (x Wu^T + bu)");
  m.def("gated_forward_split", &gated::forward_split, "the same, products kept for the backward pass, K split through a workspace");
  m.def("gated_forward_space", &gated::forward_space, "fp32 elements of the forward pass's workspace (0: none)");
  m.def("gated_pad", &gated::pad, "the rows of two matrices copied to a padded row length, zeros behind them");
  m.def("gated_workspace", &gated::workspace, "bytes of the backward pass's workspace");
  m.def("gated_backward", &gated::backward, "dx, dW and the bias gradient");
  m.def("gated_saved_elements", &gated::saved_elements, "fp32 elements of the products the forward pass keeps (0: none)");
}

}  // namespace gsc
