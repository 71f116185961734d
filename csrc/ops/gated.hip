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

static unsigned tiles(long n) { return (unsigned)((n + 63) / 64); }

static void check_sizes(long M, long D, long F, int act) {
  GSC_CHECK(M >= 1 && D >= 1 && F >= 1 && M <= 0x7fffffffL && D <= 0x7fffffffL && F <= 64L * 65535,
            "gated_linear: rows and D must be in 1 .. 2^31 - 1, F in 1 .. 4,194,240");
  GSC_CHECK(act >= 0 && act <= 2, "gated_linear: unknown activation");
}

template <class T, int BWD>
static void pair(uintptr_t x, long ldx, uintptr_t w, long ldw, Bias b, uintptr_t dh, long lddh, uintptr_t out, uintptr_t part,
                 long M, long D, long F, int act, hipStream_t s) {
  hipLaunchKernelGGL((pair_kernel<T, BWD>), dim3(tiles(M), tiles(F)), dim3(256), 0, s, Mat<T>{ptr<const T>(x), ldx, 1},
                     Mat<T>{ptr<const T>(w), ldw, 1}, b, ptr<const T>(dh), lddh, ptr<T>(out), ptr<float>(part), M, D, F, act);
  check_launch();
}

void forward(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t h, long M, long D,
             long F, int act, uintptr_t stream) {
  check_sizes(M, D, F, act);
  const Bias b{ptr<const void>(bias), bias_bf};
  if (bf) pair<bf16, 0>(x, ldx, w, ldw, b, 0, 0, h, 0, M, D, F, act, stream_of(stream));
  else pair<float, 0>(x, ldx, w, ldw, b, 0, 0, h, 0, M, D, F, act, stream_of(stream));
}

long bias_workspace(long M, long F) { return 2L * tiles(M) * 2 * F; }

// dgu [M][2F] from x, the weights and dh; part (absent: no bias gradient) takes the column sums' partial rows.
void backward_pair(uintptr_t x, long ldx, uintptr_t w, long ldw, int bf, uintptr_t bias, int bias_bf, uintptr_t dh, long lddh,
                   uintptr_t dgu, uintptr_t part, uintptr_t db, int db_bf, long M, long D, long F, int act,
                   uintptr_t stream) {
  check_sizes(M, D, F, act);
  GSC_CHECK(!db || part, "gated_linear: the bias gradient needs a workspace");
  const Bias b{ptr<const void>(bias), bias_bf};
  const hipStream_t s = stream_of(stream);
  if (bf) pair<bf16, 1>(x, ldx, w, ldw, b, dh, lddh, dgu, db ? part : 0, M, D, F, act, s);
  else pair<float, 1>(x, ldx, w, ldw, b, dh, lddh, dgu, db ? part : 0, M, D, F, act, s);
  if (db) {
    hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)((2 * F + 255) / 256)), dim3(256), 0, s, ptr<const float>(part),
                       2L * tiles(M), 2 * F, ptr<void>(db), db_bf);
    check_launch();
  }
}

template <class T>
static void prod(Mat<T> a, Mat<T> b, uintptr_t out, int out_bf, long R, long C, long K, hipStream_t s) {
  GSC_CHECK(tiles(C) <= 65535, "gated_linear: D too large");
  hipLaunchKernelGGL((prod_kernel<T>), dim3(tiles(R), tiles(C)), dim3(256), 0, s, a, b, ptr<void>(out), out_bf, C, R, C, K);
  check_launch();
}

void backward_x(uintptr_t dgu, uintptr_t w, long ldw, int bf, uintptr_t dx, int dx_bf, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  if (bf) prod<bf16>({ptr<const bf16>(dgu), 2 * F, 1}, {ptr<const bf16>(w), 1, ldw}, dx, dx_bf, M, D, 2 * F, s);
  else prod<float>({ptr<const float>(dgu), 2 * F, 1}, {ptr<const float>(w), 1, ldw}, dx, dx_bf, M, D, 2 * F, s);
}

void backward_w(uintptr_t dgu, uintptr_t x, long ldx, int bf, uintptr_t dw, int dw_bf, long M, long D, long F,
                uintptr_t stream) {
  check_sizes(M, D, F, 0);
  const hipStream_t s = stream_of(stream);
  if (bf) prod<bf16>({ptr<const bf16>(dgu), 1, 2 * F}, {ptr<const bf16>(x), 1, ldx}, dw, dw_bf, 2 * F, D, M, s);
  else prod<float>({ptr<const float>(dgu), 1, 2 * F}, {ptr<const float>(x), 1, ldx}, dw, dw_bf, 2 * F, D, M, s);
}

}  // namespace gated

void register_gated(py::module_& m) {
  m.def("gated_forward", &gated::forward, "h = act(x Wg^T + bg) * (x Wu^T + bu)");
  m.def("gated_bias_workspace", &gated::bias_workspace, "fp32 elements of the bias gradient's partial sums");
  m.def("gated_backward_pair", &gated::backward_pair, "dgu = [dh u act'(g) | dh act(g)] and the bias gradient");
  m.def("gated_backward_x", &gated::backward_x, "dx = dgu W");
  m.def("gated_backward_w", &gated::backward_w, "dW = dgu^T x");
}

}  // namespace gsc
