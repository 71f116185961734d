// Gated linear layer h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients (gfx950, MFMA, fp32 accumulation).
//
//   weight [2F][D] = Wg over Wu, bias [2F] = bg, bu;  act: silu g s(g), gelu g Phi(g), sigmoid s(g)
//   forward     g, u per 64 x 64 tile in one kernel; act, product and rounding in its epilogue
//   backward    g, u again (nothing but x is kept), dg = dh u act'(g), du = dh act(g) from the fp32 accumulators,
//               rounded once to the operand type;  dx = dg Wg + du Wu,  dW = [dg | du]^T x,  db = column sums (fp32)
//
// T = bf16 runs on v_mfma_f32_32x32x16_bf16, T = float on v_mfma_f32_32x32x2_f32.
#include <hip/hip_bf16.h>
#include <algorithm>
#include <pybind11/pybind11.h>

#include "../common.h"

namespace py = pybind11;

namespace gsc {
namespace gated {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __hip_bfloat16 bf16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

enum Act { SILU = 0, GELU = 1, SIGMOID = 2 };

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + __expf(-g)); }

__device__ __forceinline__ float act_fwd(int act, float g) {
  if (act == GELU) return g * (0.5f + 0.5f * erff(g * 0.70710678f));
  const float s = sigmoid(g);
  return act == SILU ? g * s : s;
}

// a = act(g), d = act'(g)
__device__ __forceinline__ void act_both(int act, float g, float& a, float& d) {
  if (act == GELU) {
    const float phi = 0.5f + 0.5f * erff(g * 0.70710678f);
    a = g * phi;
    d = phi + g * __expf(-0.5f * g * g) * 0.39894228f;
    return;
  }
  const float s = sigmoid(g);
  a = act == SILU ? g * s : s;
  d = act == SILU ? s * (1.f + g * (1.f - s)) : s * (1.f - s);
}

// One operand, element (r, k) at p[r sr + k sk].
template <class T>
struct Mat {
  const T* p;
  long sr, sk;
};

template <class T>
struct Tile;  // LDS image of 64 rows x BK, and the products of one BK step
template <>
struct Tile<bf16> {
  static constexpr int BK = 32, LD = 40;  // 80-byte rows
  static __device__ __forceinline__ void mul(const bf16* a, const bf16* b, int lane, f32x16& c) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int s = 0; s < BK / 16; ++s)
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(a + r * LD + 16 * s + 8 * h),
                                                  *reinterpret_cast<const bf16x8*>(b + r * LD + 16 * s + 8 * h), c, 0, 0, 0);
  }
};
template <>
struct Tile<float> {
  static constexpr int BK = 16, LD = 20;
  static __device__ __forceinline__ void mul(const float* a, const float* b, int lane, f32x16& c) {
    const int r = lane & 31, h = lane >> 5;
    // a lane's four floats are k = 8 s + 4 h ..: product t takes k = 8 s + t and 8 s + 4 + t of both operands
#pragma unroll
    for (int s = 0; s < BK / 8; ++s) {
      const f32x4 fa = *reinterpret_cast<const f32x4*>(a + r * LD + 8 * s + 4 * h);
      const f32x4 fb = *reinterpret_cast<const f32x4*>(b + r * LD + 8 * s + 4 * h);
#pragma unroll
      for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[t], fb[t], c, 0, 0, 0);
    }
  }
};

template <class T>
__device__ __forceinline__ void stage(const Mat<T>& m, long r0, long rows, long k0, long K, T* img) {
  constexpr int BK = Tile<T>::BK, LD = Tile<T>::LD;
  for (int i = threadIdx.x; i < 64 * BK; i += 256) {
    // neighbouring threads take neighbouring elements of the operand's contiguous dimension
    const int r = m.sk == 1 ? i / BK : i % 64, k = m.sk == 1 ? i % BK : i / 64;
    const bool in = r0 + r < rows && k0 + k < K;
    img[r * LD + k] = in ? m.p[(r0 + r) * m.sr + (k0 + k) * m.sk] : from_f<T>(0.f);
  }
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
__device__ __forceinline__ int acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// BWD 0: h[m][f].  BWD 1: dgu[m][f] = dg, dgu[m][F + f] = du, and part[2 * tile + wave row][0 .. 2F) = their column sums.
template <class T, int BWD>
__global__ __launch_bounds__(256) void pair_kernel(Mat<T> x, Mat<T> w, Bias bias, const T* dh, long lddh, T* out, float* part,
                                                   long M, long D, long F, int act) {
  constexpr int IMG = 64 * Tile<T>::LD;
  __shared__ __attribute__((aligned(16))) T img[3 * IMG];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const long m0 = (long)blockIdx.x * 64, f0 = (long)blockIdx.y * 64;
  const Mat<T> wu{w.p + F * w.sr, w.sr, w.sk};
  f32x16 g, u;
#pragma unroll
  for (int r = 0; r < 16; ++r) g[r] = u[r] = 0.f;
  for (long k0 = 0; k0 < D; k0 += Tile<T>::BK) {
    stage(x, m0, M, k0, D, img);
    stage(w, f0, F, k0, D, img + IMG);
    stage(wu, f0, F, k0, D, img + 2 * IMG);
    __syncthreads();
    const T* a = img + wm * 32 * Tile<T>::LD;
    Tile<T>::mul(a, img + IMG + wn * 32 * Tile<T>::LD, lane, g);
    Tile<T>::mul(a, img + 2 * IMG + wn * 32 * Tile<T>::LD, lane, u);
    __syncthreads();
  }
  const long f = f0 + wn * 32 + (lane & 31);
  const float bg = f < F ? bias.at(f) : 0.f, bu = f < F ? bias.at(F + f) : 0.f;
  float sg = 0.f, su = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const long m = m0 + wm * 32 + acc_row(r, lane);
    if (m >= M || f >= F) continue;
    const float gv = g[r] + bg, uv = u[r] + bu;
    if (!BWD) {
      out[m * F + f] = from_f<T>(act_fwd(act, gv) * uv);
    } else {
      float a, d;
      act_both(act, gv, a, d);
      const float dv = to_f(dh[m * lddh + f]);
      const float dg = dv * uv * d, du = dv * a;
      out[m * 2 * F + f] = from_f<T>(dg);
      out[m * 2 * F + F + f] = from_f<T>(du);
      sg += dg;
      su += du;
    }
  }
  if (BWD && part) {
    sg += __shfl_xor(sg, 32);
    su += __shfl_xor(su, 32);
    if (lane < 32 && f < F) {
      float* row = part + (2 * (long)blockIdx.x + wm) * 2 * F;
      row[f] = sg;
      row[F + f] = su;
    }
  }
}

// out[r][c] = sum_k A(r, k) B(c, k), rounded once to the output type.
template <class T>
__global__ __launch_bounds__(256) void prod_kernel(Mat<T> a, Mat<T> b, void* out, int out_bf, long ldo, long R, long C, long K) {
  constexpr int IMG = 64 * Tile<T>::LD;
  __shared__ __attribute__((aligned(16))) T img[2 * IMG];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const long r0 = (long)blockIdx.x * 64, c0 = (long)blockIdx.y * 64;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  for (long k0 = 0; k0 < K; k0 += Tile<T>::BK) {
    stage(a, r0, R, k0, K, img);
    stage(b, c0, C, k0, K, img + IMG);
    __syncthreads();
    Tile<T>::mul(img + wm * 32 * Tile<T>::LD, img + IMG + wn * 32 * Tile<T>::LD, lane, acc);
    __syncthreads();
  }
  const long c = c0 + wn * 32 + (lane & 31);
  if (c >= C) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const long row = r0 + wm * 32 + acc_row(r, lane);
    if (row >= R) continue;
    if (out_bf) reinterpret_cast<bf16*>(out)[row * ldo + c] = __float2bfloat16(acc[r]);
    else reinterpret_cast<float*>(out)[row * ldo + c] = acc[r];
  }
}

// out[c] = sum over the partial rows, in a fixed order.
__global__ __launch_bounds__(256) void colsum_kernel(const float* part, long rows, long C, void* out, int out_bf) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float s = 0.f;
  for (long z = 0; z < rows; ++z) s += part[z * C + c];
  if (out_bf) reinterpret_cast<bf16*>(out)[c] = __float2bfloat16(s);
  else reinterpret_cast<float*>(out)[c] = s;
}


// ---------------------------------------------------------------------------------------------------------------
// bf16 tiles.  out = sum_k A(r, k) B(c, k) on BM x BN tiles, K in steps of 64, both operands copied straight from
// memory into LDS (buffer loads to LDS, 16 bytes a lane) one step ahead of the products.
//
//   row operand (k contiguous)   LDS [R][64], 16-byte chunk c of row r in slot c ^ ((r >> 1) & 7): the 16 rows of a
//                                fragment read cover all 64 banks once
//   column operand (r contiguous) LDS [64][R], chunk c of row k in slot c ^ 4 (k & 3): the four rows of a transposing
//                                read (ds_read_b64_tr_b16) fall on four different 64-byte quarters of the banks
// The copy to LDS writes lane l's 16 bytes at 16 l, so the slots are permuted on the address side.  Rows and chunks
// outside the matrices get an offset past the buffer descriptor's end: the load returns zeros.  Operands are 16-byte
// aligned with rows of a multiple of 8 elements (the caller pads others), so a chunk is inside or outside as a whole.

constexpr unsigned kOut = 0x80000000u;   // past every descriptor (2^31 - 1 bytes)
typedef __attribute__((address_space(3))) short lds_short;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int R, int WAVES, bool COL>
struct Copy {
  static constexpr int PER = R / 8 / WAVES;   // 1 KB wave copies per wave and step
  static_assert(R % (8 * WAVES) == 0 && (!COL || R == 128 || R == 256), "tile");
  unsigned off[PER];
  int kk[PER];      // k (row operand: of the chunk's first element; column operand: of the row) inside a step
  unsigned step;    // bytes per step
  // r0: first row (column) of the tile, rows: their count in the matrix, ld: elements between stored rows
  __device__ __forceinline__ void init(long r0, long rows, long ld, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = i * WAVES + wave;
      if (!COL) {
        const int r = 8 * q + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        off[i] = r0 + r < rows ? (unsigned)(r * ld * 2 + 16 * c) : kOut;
        kk[i] = 8 * c;
      } else {
        constexpr int CPR = R / 8;   // chunks per stored row
        const int k = q * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ ((k & 3) << 2);
        off[i] = r0 + 8 * c < rows ? (unsigned)(k * ld * 2 + 16 * c) : kOut;
        kk[i] = k;
      }
    }
    step = COL ? (unsigned)(64 * ld * 2) : 128u;
  }
  // base: the tile's first element at this step, left: k that remain (>= 64: all)
  __device__ __forceinline__ void load(const bf16* base, long left, short* img, int wave) const {
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, 0x7fffffff, 0x00027000);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned o = left >= 64 || kk[i] < left ? off[i] : kOut;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_short*)(img + 512 * (i * WAVES + wave)), 16, o, 0, 0, 0);
    }
  }
};

// Addresses of a wave's 32 x 16 fragments in an image of R rows (columns).  Fragment i covers rows r0 + 32 i; r0 is a
// multiple of 32 N for column images.  Everything but one register per k step (row image) or per fragment (column image)
// is an immediate offset of the read.
template <int R, bool COL, int N>
struct Frags {
  const short* at[COL ? N : 4];
  __device__ __forceinline__ void init(const short* img, int r0, int lane) {
    if constexpr (!COL) {
      const int r = r0 + (lane & 31), c = (lane >> 5) ^ ((r >> 1) & 7);
#pragma unroll
      for (int s = 0; s < 4; ++s) at[s] = img + r * 64 + 8 * (c ^ (2 * s));
    } else {
      const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
#pragma unroll
      for (int i = 0; i < N; ++i)
        at[i] = img + (8 * (g >> 1) + q) * R + 8 * ((((r0 >> 3) + 4 * i) ^ (q << 2)) + 2 * (g & 1) + (p >> 1)) + 4 * (p & 1);
    }
  }
  // fragment i of k step s; shift: elements to the image in use
  __device__ __forceinline__ bf16x8 read(int i, int s, int shift) const {
    if constexpr (!COL) {
      return *reinterpret_cast<const bf16x8*>(at[s] + shift + 32 * 64 * i);
    } else {
      const short* a = at[i] + shift + 16 * s * R;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * R));
      return __builtin_bit_cast(bf16x8, (s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}));
    }
  }
};

struct TileArgs {
  const bf16* a[2];   // operands of the two K segments (dx: gate and up halves), one segment otherwise
  const bf16* b[2];   // pair kernels: gate and up rows instead
  long lda, ldb;
  int segs;
  long M, N, K;       // rows, columns (pair: F) and K of a segment
  int tm, tn;         // tiles
  long kchunk;        // K of a split (whole steps; one segment only), K otherwise
  Bias bias;
  const bf16* dh;
  long lddh;
  void* out;
  int out_bf;
  long ldo;
  long half;          // dgu: column of du
  long slab;          // elements between the fp32 partial results of two splits
  int tmh;            // dW: tile rows of the gate half (the up half follows), 0 otherwise
  float* part;
  int act;
};

// Workgroups are dealt to the 8 XCDs in turn: each XCD takes a contiguous run of tiles, walked in strips of 8 tile
// rows, so the operand panels its 32 CUs share stay in its own L2.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& pm, int& pn) {
  const int total = tm * tn, per = total / 8, rem = total % 8, x = id & 7;
  const int t = x * per + (x < rem ? x : rem) + (id >> 3);
  const int width = 8 * tn, g = t / width, first = g * 8, rows = tm - first < 8 ? tm - first : 8;
  pm = first + (t % width) % rows;
  pn = (t % width) / rows;
}

enum Epi { FWD = 0, BWD = 1, OUT = 2 };

template <int RM, int RN, int WM, int WN, bool ACOL, bool BCOL, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(TileArgs g) {
  constexpr int WAVES = WM * WN, BM = 32 * RM * WM, BN = 32 * RN * WN;
  constexpr bool PAIR = EPI != OUT;
  constexpr int BH = PAIR ? BN / 2 : BN;            // columns of one product
  constexpr int SH = PAIR ? RN / 2 : RN;            // 32-column fragments of one product per wave
  constexpr int ASZ = BM * 64, BSZ = BN * 64;
  constexpr int OC = EPI == FWD ? BH : BN, OLD = OC + 8;   // output columns of the tile, staged row stride
  constexpr int OPS = 2 * (ASZ + BSZ), STG = BM * OLD;
  __shared__ __attribute__((aligned(1024))) short smem[OPS > STG ? OPS : STG];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int pm, pn;
  tile_of(blockIdx.x, g.tm, g.tn, pm, pn);
  const int up = EPI == OUT && g.tmh && pm >= g.tmh;   // dW: rows of the up half
  if (up) pm -= g.tmh;
  const long m0 = (long)pm * BM, n0 = (long)pn * BH;
  const long k0 = (long)blockIdx.y * g.kchunk, kend = k0 + g.kchunk < g.K ? k0 + g.kchunk : g.K;
  const int steps = (int)((kend - k0 + 63) / 64), total = steps * g.segs;

  // two images of each operand: A0 A1 | B0 B1
  short *const ia = smem, *const ib = smem + 2 * ASZ;
  Copy<BM, WAVES, ACOL> ca;
  Copy<BH, WAVES, BCOL> cb;
  ca.init(m0, g.M, g.lda, wave, lane);
  cb.init(n0, g.N, g.ldb, wave, lane);
  const long a0 = (ACOL ? m0 + k0 * g.lda : m0 * g.lda + k0) + up * g.half, b0 = BCOL ? n0 + k0 * g.ldb : n0 * g.ldb + k0;
  auto load = [&](int t, int buf) {
    const int seg = t >= steps ? 1 : 0, st = t - seg * steps;
    const long left = kend - k0 - 64L * st;
    ca.load(g.a[PAIR ? 0 : seg] + a0 + (long)st * (ca.step / 2), left, ia + buf * ASZ, wave);
    const long bo = b0 + (long)st * (cb.step / 2);
    if (PAIR) {
      cb.load(g.b[0] + bo, left, ib + buf * BSZ, wave);
      cb.load(g.b[1] + bo, left, ib + buf * BSZ + BH * 64, wave);
    } else {
      cb.load(g.b[seg] + bo, left, ib + buf * BSZ, wave);
    }
  };
  Frags<BM, ACOL, RM> fa_at;
  Frags<BH, BCOL, SH> fb_at;
  fa_at.init(ia, 32 * wm * RM, lane);
  fb_at.init(ib, 32 * wn * SH, lane);

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  auto step = [&](int t, int buf) {
    // this step's copies have landed and every wave has read the other images
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + 1 < total) load(t + 1, buf ^ 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 fa[RM], fb[RN];
#pragma unroll
      for (int i = 0; i < RM; ++i) fa[i] = fa_at.read(i, s, buf * ASZ);
#pragma unroll
      for (int j = 0; j < RN; ++j) fb[j] = fb_at.read(j % SH, s, buf * BSZ + (j / SH) * BH * 64);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  };
  load(0, 0);
  for (int t = 0; t < total; t += 2) {
    step(t, 0);
    if (t + 1 < total) step(t + 1, 1);
  }

  // ---- epilogue
  const int cl = lane & 31;
  if constexpr (EPI == OUT) {
    if (!g.out_bf) {   // fp32: 128-byte row pieces straight from the accumulators
      const int row0 = 32 * wm * RM + 4 * (lane >> 5);
#pragma unroll 1
      for (int j = 0; j < SH; ++j) {
        const long n = n0 + 32 * (wn * SH + j) + cl;
        float* o = reinterpret_cast<float*>(g.out) + blockIdx.y * g.slab + (m0 + row0 + up * g.M) * g.ldo + n;
        const long left = n < g.N ? g.M - m0 - row0 : 0;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 32 * i + acc_row(r, 0);
            float v = acc[i][0][r];
#pragma unroll
            for (int q = 1; q < SH; ++q) v = j == q ? acc[i][q][r] : v;
            if (row < left) *o = v;
            o += (r == 15 ? 32 * (i + 1) - row : acc_row(r + 1, 0) - acc_row(r, 0)) * g.ldo;
          }
      }
      return;
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();   // the operand images are free
#pragma unroll
  for (int j = 0; j < SH; ++j) {
    const int col = 32 * (wn * SH + j) + cl;
    const long n = n0 + col;
    float bg = 0.f, bu = 0.f, sg = 0.f, su = 0.f;
    if (PAIR && n < g.N) {
      bg = g.bias.at(n);
      bu = g.bias.at(g.N + n);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = 32 * (wm * RM + i) + acc_row(r, lane);
        const long m = m0 + row;
        if constexpr (EPI == OUT) {
          smem[row * OLD + col] = __builtin_bit_cast(short, __float2bfloat16(acc[i][j][r]));
        } else {
          const float gv = acc[i][j][r] + bg, uv = acc[i][j + SH][r] + bu;
          if constexpr (EPI == FWD) {
            smem[row * OLD + col] = __builtin_bit_cast(short, __float2bfloat16(act_fwd(g.act, gv) * uv));
          } else {
            float dg = 0.f, du = 0.f;
            if (m < g.M && n < g.N) {
              float a, d;
              act_both(g.act, gv, a, d);
              const float dv = to_f(g.dh[m * g.lddh + n]);
              dg = dv * uv * d;
              du = dv * a;
            }
            smem[row * OLD + col] = __builtin_bit_cast(short, __float2bfloat16(dg));
            smem[row * OLD + BH + col] = __builtin_bit_cast(short, __float2bfloat16(du));
            sg += dg;
            su += du;
          }
        }
      }
    }
    if (EPI == BWD && g.part) {
      sg += __shfl_xor(sg, 32);
      su += __shfl_xor(su, 32);
      if (lane < 32 && n < g.N) {
        float* row = g.part + ((long)pm * WM + wm) * 2 * g.N;
        row[n] = sg;
        row[g.N + n] = su;
      }
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // rows of the staged tile leave in 16-byte pieces; dgu rows are padded to whole pieces (with zeros), others may end
  // inside one or start off 16 bytes
  const long cols = EPI == BWD ? g.half : g.N;
  bf16* out = reinterpret_cast<bf16*>(g.out);
  const bool vec = ((uintptr_t)out % 16 == 0) && g.ldo % 8 == 0;
  for (int idx = tid; idx < BM * (OC / 8); idx += 64 * WAVES) {
    const int row = idx / (OC / 8), c = idx % (OC / 8) * 8;
    const long m = m0 + row, n = n0 + (EPI == BWD ? c % BH : c);
    if (m >= g.M || n >= cols) continue;
    const short* src = smem + row * OLD + c;
    bf16* dst = out + (m + up * g.M) * g.ldo + n + (EPI == BWD && c >= BH ? g.half : 0);
    if (vec && n + 8 <= cols) {
      *reinterpret_cast<s16x8*>(dst) = *reinterpret_cast<const s16x8*>(src);
    } else {
      for (int e = 0; e < 8 && n + e < cols; ++e) dst[e] = __builtin_bit_cast(bf16, src[e]);
    }
  }
}

// dst [rows][ldd]: the rows of src, zeros behind them.
template <class T>
__global__ __launch_bounds__(256) void pad_kernel(const T* src, long lds_, T* dst, long ldd, long rows, long cols) {
  const long n = rows * ldd;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / ldd, c = i - r * ldd;
    dst[i] = c < cols ? src[r * lds_ + c] : from_f<T>(0.f);
  }
}

// out[i] = sum over the splits' partial results, in a fixed order.
__global__ __launch_bounds__(256) void splits_kernel(const float* slabs, long slab, int splits, long n, void* out, int out_bf) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < splits; ++z) s += slabs[z * slab + i];
    if (out_bf) reinterpret_cast<bf16*>(out)[i] = __float2bfloat16(s);
    else reinterpret_cast<float*>(out)[i] = s;
  }
}

static long up8(long n) { return (n + 7) / 8 * 8; }
static unsigned tiles(long n, long t = 64) { return (unsigned)((n + t - 1) / t); }
static unsigned flat_grid(long n) { return (unsigned)std::max<long>(1, std::min<long>((n + 255) / 256, 4096)); }

static void check_sizes(long M, long D, long F, int act) {
  GSC_CHECK(M >= 1 && D >= 1 && F >= 1 && M <= 0x7fffffffL && D <= 4000000L && F <= 4000000L,
            "gated_linear: rows must be in 1 .. 2^31 - 1, D and F in 1 .. 4,000,000");
  GSC_CHECK(act >= 0 && act <= 2, "gated_linear: unknown activation");
}

// Operands of the bf16 tiles: 16-byte aligned rows.
static void check_operand(uintptr_t p, long ld) {
  GSC_CHECK(p % 16 == 0 && ld % 8 == 0 && ld <= 4000000L, "gated_linear: a bf16 operand needs 16-byte aligned rows");
}

static int cu_count() {
  static const int n = [] {
    int dev = 0, v = 256;
    if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev);
    return v > 0 ? v : 256;
  }();
  return n;
}

template <int RM, int RN, int WM, int WN, bool ACOL, bool BCOL, int EPI>
static void launch(TileArgs g, int splits, hipStream_t s) {
  constexpr int BM = 32 * RM * WM, BH = EPI == OUT ? 32 * RN * WN : 16 * RN * WN;
  g.tm = (int)tiles(g.M, BM);
  g.tn = (int)tiles(g.N, BH);
  if (g.tmh) {
    g.tmh = g.tm;
    g.tm *= 2;
  }
  GSC_CHECK((long)g.tm * g.tn <= 0x7fffffffL, "gated_linear: too many tiles");
  hipLaunchKernelGGL((tile_kernel<RM, RN, WM, WN, ACOL, BCOL, EPI>), dim3((unsigned)(g.tm * g.tn), splits), dim3(64 * WM * WN),
                     0, s, g);
  check_launch();
}

// 256-row tiles where they fill the CUs, 128-row tiles otherwise.
static bool large(long M, long N, long bn) { return (long)tiles(M, 256) * tiles(N, bn) >= cu_count(); }

static int pair_rows(long M, long F) { return large(M, F, 128) ? 256 : 128; }

template <int EPI>
static void pair_bf16(TileArgs g, hipStream_t s) {
  if (pair_rows(g.M, g.N) == 256) launch<4, 2, 2, 4, false, false, EPI>(g, 1, s);
  else launch<2, 2, 2, 2, false, false, EPI>(g, 1, s);
}

template <class T, int BWD>
static void pair(uintptr_t x, long ldx, uintptr_t w, long ldw, Bias b, uintptr_t dh, long lddh, uintptr_t out, uintptr_t part,
                 long M, long D, long F, int act, hipStream_t s) {
  hipLaunchKernelGGL((pair_kernel<T, BWD>), dim3(tiles(M), tiles(F)), dim3(256), 0, s, Mat<T>{ptr<const T>(x), ldx, 1},
                     Mat<T>{ptr<const T>(w), ldw, 1}, b, ptr<const T>(dh), lddh, ptr<T>(out), ptr<float>(part), M, D, F, act);
  check_launch();
}

static TileArgs pair_args(uintptr_t x, long ldx, uintptr_t w, long ldw, Bias b, long M, long D, long F, int act) {
  check_operand(x, ldx);
  check_operand(w, ldw);
  TileArgs g{};
  g.a[0] = ptr<const bf16>(x);
  g.b[0] = ptr<const bf16>(w);
  g.b[1] = g.b[0] + F * ldw;
  g.lda = ldx;
  g.ldb = ldw;
  g.segs = 1;
  g.M = M;
  g.N = F;
  g.K = g.kchunk = up8(D);   // rows are padded with zeros
  g.bias = b;
  g.act = act;
  return g;
}

void forward(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t h, long M, long D,
             long F, int act, uintptr_t stream) {
  check_sizes(M, D, F, act);
  const Bias b{ptr<const void>(bias), bias_bf};
  const hipStream_t s = stream_of(stream);
  if (!bf) {
    pair<float, 0>(x, ldx, w, ldw, b, 0, 0, h, 0, M, D, F, act, s);
    return;
  }
  TileArgs g = pair_args(x, ldx, w, ldw, b, M, D, F, act);
  g.out = ptr<void>(h);
  g.ldo = F;
  pair_bf16<FWD>(g, s);
}

void pad(uintptr_t src, long lds_, uintptr_t dst, long ldd, int bf, long rows, long cols, uintptr_t stream) {
  GSC_CHECK(rows >= 1 && cols >= 1 && cols <= ldd, "gated_linear: pad");
  const hipStream_t s = stream_of(stream);
  const dim3 grid(flat_grid(rows * ldd));
  if (bf) hipLaunchKernelGGL((pad_kernel<bf16>), grid, dim3(256), 0, s, ptr<const bf16>(src), lds_, ptr<bf16>(dst), ldd, rows, cols);
  else hipLaunchKernelGGL((pad_kernel<float>), grid, dim3(256), 0, s, ptr<const float>(src), lds_, ptr<float>(dst), ldd, rows, cols);
  check_launch();
}

// Elements of dgu rows: [dg, zeros to a multiple of 8 | du, zeros] for bf16, [dg | du] for fp32.
static long half_of(int bf, long F) { return bf ? up8(F) : F; }

static long part_rows(int bf, long M, long F) {
  if (!bf) return 2L * tiles(M);
  return 2L * tiles(M, pair_rows(M, F));
}

// fp32 elements of the bias gradient's partial sums.
long bias_workspace(int bf, long M, long F) { return part_rows(bf, M, F) * 2 * F; }

// dgu from x, the weights and dh; part (absent: no bias gradient) takes the column sums' partial rows.
void backward_pair(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t dh, long lddh,
                   uintptr_t dgu, uintptr_t part, uintptr_t db, int db_bf, long M, long D, long F, int act,
                   uintptr_t stream) {
  check_sizes(M, D, F, act);
  GSC_CHECK(!db || part, "gated_linear: the bias gradient needs a workspace");
  const Bias b{ptr<const void>(bias), bias_bf};
  const hipStream_t s = stream_of(stream);
  if (bf) {
    TileArgs g = pair_args(x, ldx, w, ldw, b, M, D, F, act);
    g.dh = ptr<const bf16>(dh);
    g.lddh = lddh;
    g.out = ptr<void>(dgu);
    g.half = half_of(bf, F);
    g.ldo = 2 * g.half;
    g.part = db ? ptr<float>(part) : nullptr;
    pair_bf16<BWD>(g, s);
  } else {
    pair<float, 1>(x, ldx, w, ldw, b, dh, lddh, dgu, db ? part : 0, M, D, F, act, s);
  }
  if (db) {
    hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)((2 * F + 255) / 256)), dim3(256), 0, s, ptr<const float>(part),
                       part_rows(bf, M, F), 2 * F, ptr<void>(db), db_bf);
    check_launch();
  }
}

template <class T>
static void prod(Mat<T> a, Mat<T> b, uintptr_t out, int out_bf, long R, long C, long K, hipStream_t s) {
  hipLaunchKernelGGL((prod_kernel<T>), dim3(tiles(R), tiles(C)), dim3(256), 0, s, a, b, ptr<void>(out), out_bf, C, R, C, K);
  check_launch();
}

void backward_x(uintptr_t dgu, uintptr_t w, long ldw, int bf, uintptr_t dx, int dx_bf, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  if (!bf) {
    prod<float>({ptr<const float>(dgu), 2 * F, 1}, {ptr<const float>(w), 1, ldw}, dx, dx_bf, M, D, 2 * F, s);
    return;
  }
  check_operand(dgu, 2 * up8(F));
  check_operand(w, ldw);
  TileArgs g{};
  g.a[0] = ptr<const bf16>(dgu);
  g.a[1] = g.a[0] + up8(F);
  g.b[0] = ptr<const bf16>(w);
  g.b[1] = g.b[0] + F * ldw;
  g.lda = 2 * up8(F);
  g.ldb = ldw;
  g.segs = 2;
  g.M = M;
  g.N = D;
  g.K = g.kchunk = F;
  g.out = ptr<void>(dx);
  g.out_bf = dx_bf;
  g.ldo = D;
  if (large(M, D, 256)) launch<4, 2, 2, 4, false, true, OUT>(g, 1, s);
  else launch<2, 2, 2, 2, false, true, OUT>(g, 1, s);
}

// Splits of dW's reduction over the rows: enough workgroups for two per CU, at least 512 rows each.
static int w_splits(long M, long D, long F) {
  if (large(2 * F, D, 256)) return 1;
  const long t = 2L * tiles(F, 128) * tiles(D, 128);
  return (int)std::max<long>(1, std::min<long>({(2L * cu_count() + t - 1) / t, M / 512, 64}));
}

long w_workspace(int bf, long M, long D, long F) {
  const int n = bf ? w_splits(M, D, F) : 1;
  return n > 1 ? n * 2 * F * D : 0;
}

void backward_w(uintptr_t dgu, uintptr_t x, long ldx, int bf, uintptr_t dw, int dw_bf, uintptr_t slabs, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  if (!bf) {
    prod<float>({ptr<const float>(dgu), 1, 2 * F}, {ptr<const float>(x), 1, ldx}, dw, dw_bf, 2 * F, D, M, s);
    return;
  }
  check_operand(dgu, 2 * up8(F));
  check_operand(x, ldx);
  const int splits = w_splits(M, D, F);
  GSC_CHECK(splits == 1 || slabs, "gated_linear: the weight gradient needs a workspace");
  TileArgs g{};
  g.a[0] = ptr<const bf16>(dgu);
  g.b[0] = ptr<const bf16>(x);
  g.lda = 2 * up8(F);
  g.ldb = ldx;
  g.segs = 1;
  g.M = F;
  g.N = D;
  g.K = M;
  g.kchunk = (M + splits - 1) / splits;
  g.kchunk = (g.kchunk + 63) / 64 * 64;
  g.half = up8(F);
  g.tmh = 1;
  g.ldo = D;
  const int used = (int)((M + g.kchunk - 1) / g.kchunk);
  if (splits > 1) {
    g.out = ptr<void>(slabs);
    g.slab = 2 * F * D;
  } else {
    g.out = ptr<void>(dw);
    g.out_bf = dw_bf;
  }
  if (large(2 * F, D, 256)) launch<4, 2, 2, 4, true, true, OUT>(g, used, s);
  else launch<2, 2, 2, 2, true, true, OUT>(g, used, s);
  if (splits > 1) {
    hipLaunchKernelGGL(splits_kernel, dim3(flat_grid(2 * F * D)), dim3(256), 0, s, ptr<const float>(slabs), g.slab, used,
                       2 * F * D, ptr<void>(dw), dw_bf);
    check_launch();
  }
}

}  // namespace gated

void register_gated(py::module_& m) {
  m.def("gated_forward", &gated::forward, "h = act(x Wg^T + bg) * (x Wu^T + bu)");
  m.def("gated_pad", &gated::pad, "rows copied to a padded row length, zeros behind them");
  m.def("gated_bias_workspace", &gated::bias_workspace, "fp32 elements of the bias gradient's partial sums");
  m.def("gated_weight_workspace", &gated::w_workspace, "fp32 elements of the weight gradient's partial results");
  m.def("gated_backward_pair", &gated::backward_pair, "dgu = [dh u act'(g) | dh act(g)] and the bias gradient");
  m.def("gated_backward_x", &gated::backward_x, "dx = dgu W");
  m.def("gated_backward_w", &gated::backward_w, "dW = dgu^T x");
}

}  // namespace gsc
