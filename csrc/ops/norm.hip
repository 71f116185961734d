// Layer norm over the last dimension, forward and backward (gfx950).
//
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_c g - xh mean_c(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// x, y, dy, dx are bf16 or fp32; w and b fp32 or bf16 each (absent: 1 and 0).  Every sum and statistic is fp32; an
// output is rounded once.
#include <hip/hip_bf16.h>
#include <algorithm>
#include <pybind11/pybind11.h>

#include "../common.h"

namespace py = pybind11;

namespace gsc {
namespace norm {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

// A per-column parameter: fp32 or bf16, or absent.
struct Param {
  const void* p;
  int bf16;
  __device__ __forceinline__ float at(int c, float none) const {
    if (!p) return none;
    return bf16 ? __bfloat162float(reinterpret_cast<const __hip_bfloat16*>(p)[c]) : reinterpret_cast<const float*>(p)[c];
  }
};

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T>
__global__ __launch_bounds__(256) void fwd_kernel(const T* x, long ldx, Param w, Param b, T* y, float* mean, float* rstd,
                                                  int C, float eps) {
  __shared__ float red[4];
  const long row = blockIdx.x;
  const T* xr = x + row * ldx;
  float s = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) s += to_f(xr[c]);
  const float mu = block_sum(s, red) / (float)C;
  float q = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float d = to_f(xr[c]) - mu;
    q += d * d;
  }
  const float r = 1.f / sqrtf(block_sum(q, red) / (float)C + eps);
  for (int c = threadIdx.x; c < C; c += 256)
    y[row * C + c] = from_f<T>((to_f(xr[c]) - mu) * r * w.at(c, 1.f) + b.at(c, 0.f));
  if (threadIdx.x == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

template <class T>
__global__ __launch_bounds__(256) void bwd_x_kernel(const T* x, long ldx, const T* dy, long lddy, Param w,
                                                    const float* mean, const float* rstd, T* dx, int C) {
  __shared__ float red[4];
  const long row = blockIdx.x;
  const T* xr = x + row * ldx;
  const T* gr = dy + row * lddy;
  const float mu = mean[row], r = rstd[row];
  float s = 0.f, q = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float g = to_f(gr[c]) * w.at(c, 1.f);
    s += g;
    q += g * ((to_f(xr[c]) - mu) * r);
  }
  const float ms = block_sum(s, red) / (float)C, mq = block_sum(q, red) / (float)C;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float g = to_f(gr[c]) * w.at(c, 1.f);
    dx[row * C + c] = from_f<T>(r * (g - ms - (to_f(xr[c]) - mu) * r * mq));
  }
}

// Partial column sums over the rows z, z + S, ...: part[z][0][c] = sum dy xh, part[z][1][c] = sum dy.
template <class T>
__global__ __launch_bounds__(256) void bwd_w_kernel(const T* x, long ldx, const T* dy, long lddy, const float* mean,
                                                    const float* rstd, float* part, long M, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float dw = 0.f, db = 0.f;
  for (long m = blockIdx.y; m < M; m += gridDim.y) {
    const float g = to_f(dy[m * lddy + c]);
    dw += g * ((to_f(x[m * ldx + c]) - mean[m]) * rstd[m]);
    db += g;
  }
  part[((long)blockIdx.y * 2) * C + c] = dw;
  part[((long)blockIdx.y * 2 + 1) * C + c] = db;
}

// Sum of the S partials in a fixed order.
__global__ __launch_bounds__(256) void bwd_w_reduce_kernel(const float* part, int S, int C, void* dw, int dw_bf16,
                                                           void* db, int db_bf16) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float s[2] = {0.f, 0.f};
  for (int z = 0; z < S; ++z)
    for (int k = 0; k < 2; ++k) s[k] += part[((long)z * 2 + k) * C + c];
  void* out[2] = {dw, db};
  const int bf[2] = {dw_bf16, db_bf16};
  for (int k = 0; k < 2; ++k) {
    if (!out[k]) continue;
    if (bf[k]) reinterpret_cast<__hip_bfloat16*>(out[k])[c] = __float2bfloat16(s[k]);
    else reinterpret_cast<float*>(out[k])[c] = s[k];
  }
}

static int splits_of(long M) { return (int)std::max<long>(1, std::min<long>(256, M / 16)); }

template <class T>
static void run_fwd(uintptr_t x, long ldx, Param w, Param b, uintptr_t y, uintptr_t mean, uintptr_t rstd, long M, int C,
                    float eps, hipStream_t s) {
  hipLaunchKernelGGL((fwd_kernel<T>), dim3((unsigned)M), dim3(256), 0, s, ptr<const T>(x), ldx, w, b, ptr<T>(y),
                     ptr<float>(mean), ptr<float>(rstd), C, eps);
  check_launch();
}

template <class T>
static void run_bwd(uintptr_t x, long ldx, uintptr_t dy, long lddy, Param w, uintptr_t mean, uintptr_t rstd, uintptr_t dx,
                    uintptr_t part, long M, int C, hipStream_t s) {
  if (dx)
    hipLaunchKernelGGL((bwd_x_kernel<T>), dim3((unsigned)M), dim3(256), 0, s, ptr<const T>(x), ldx, ptr<const T>(dy), lddy,
                       w, ptr<const float>(mean), ptr<const float>(rstd), ptr<T>(dx), C);
  if (part)
    hipLaunchKernelGGL((bwd_w_kernel<T>), dim3((C + 255) / 256, splits_of(M)), dim3(256), 0, s, ptr<const T>(x), ldx,
                       ptr<const T>(dy), lddy, ptr<const float>(mean), ptr<const float>(rstd), ptr<float>(part), M, C);
  check_launch();
}

static void check_sizes(long M, long C) {
  GSC_CHECK(M >= 1 && M <= 0x7fffffffL && C >= 1 && C <= 0x7fffffffL, "layer_norm: rows and columns must be in 1 .. 2^31 - 1");
}

void forward(uintptr_t x, long ldx, int bf16, uintptr_t w, int w_bf16, uintptr_t b, int b_bf16, uintptr_t y,
             uintptr_t mean, uintptr_t rstd, long M, long C, float eps, uintptr_t stream) {
  check_sizes(M, C);
  const Param pw{ptr<const void>(w), w_bf16}, pb{ptr<const void>(b), b_bf16};
  if (bf16) run_fwd<__hip_bfloat16>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, stream_of(stream));
  else run_fwd<float>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, stream_of(stream));
}

// fp32 elements of the backward's partial column sums.
long workspace(long M, long C) { return 2 * C * splits_of(M); }

void backward(uintptr_t x, long ldx, uintptr_t dy, long lddy, int bf16, uintptr_t w, int w_bf16, uintptr_t mean,
              uintptr_t rstd, uintptr_t dx, uintptr_t dw, int dw_bf16, uintptr_t db, int db_bf16, uintptr_t part, long M,
              long C, uintptr_t stream) {
  check_sizes(M, C);
  const hipStream_t s = stream_of(stream);
  const Param pw{ptr<const void>(w), w_bf16};
  const bool params = dw || db;
  GSC_CHECK(!params || part, "layer_norm: parameter gradients need a workspace");
  if (bf16) run_bwd<__hip_bfloat16>(x, ldx, dy, lddy, pw, mean, rstd, dx, params ? part : 0, M, (int)C, s);
  else run_bwd<float>(x, ldx, dy, lddy, pw, mean, rstd, dx, params ? part : 0, M, (int)C, s);
  if (params) {
    hipLaunchKernelGGL(bwd_w_reduce_kernel, dim3((unsigned)((C + 255) / 256)), dim3(256), 0, s, ptr<const float>(part),
                       splits_of(M), (int)C, ptr<void>(dw), dw_bf16, ptr<void>(db), db_bf16);
    check_launch();
  }
}

}  // namespace norm

void register_norm(py::module_& m) {
  m.def("layer_norm_forward", &norm::forward, "layer norm of rows: y, and mean / 1/std per row when asked for");
  m.def("layer_norm_workspace", &norm::workspace, "fp32 elements the backward's parameter gradients need");
  m.def("layer_norm_backward", &norm::backward, "layer norm gradients (dx, and dw / db through the workspace)");
}

}  // namespace gsc
