// Layer norm over the last dimension, forward and backward (gfx950).
//
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_c g - xh mean_c(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// x, y, dy, dx are bf16 or fp32; w and b fp32 or bf16 each (absent: 1 and 0).  Every sum and statistic is fp32, the variance
// from the centred values; an output is rounded once.
//
// Bound by memory: a row is read once into registers (G lanes x N pieces of VEC elements), both passes over it run there.
// The backward pass keeps the gradient sums of its columns in registers over all rows that a group of lanes takes, adds the
// groups of a workgroup in LDS and leaves one partial row per workgroup; a second kernel adds those in a fixed order.
#include <hip/hip_bf16.h>
#include <algorithm>
#include <pybind11/pybind11.h>

#include "../common.h"

namespace py = pybind11;

namespace gsc {
namespace norm {

typedef __hip_bfloat16 bf16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

// VEC elements at p as floats: 16 bytes (VEC 8 of bf16, 4 of fp32) or one element.
template <int VEC>
__device__ __forceinline__ void load(const bf16* p, float* v) {
  if constexpr (VEC == 8) {
    const s16x8 q = *reinterpret_cast<const s16x8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __bfloat162float(__builtin_bit_cast(bf16, (short)q[e]));
  } else {
    v[0] = __bfloat162float(*p);
  }
}
template <int VEC>
__device__ __forceinline__ void load(const float* p, float* v) {
  if constexpr (VEC == 4) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q[e];
  } else {
    v[0] = *p;
  }
}
template <int VEC>
__device__ __forceinline__ void store(bf16* p, const float* v) {
  if constexpr (VEC == 8) {
    s16x8 q;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __builtin_bit_cast(short, __float2bfloat16(v[e]));
    *reinterpret_cast<s16x8*>(p) = q;
  } else {
    *p = __float2bfloat16(v[0]);
  }
}
template <int VEC>
__device__ __forceinline__ void store(float* p, const float* v) {
  if constexpr (VEC == 4) *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  else *p = v[0];
}

// A per-column parameter: fp32 or bf16, or absent; 16-byte aligned where VEC > 1.
struct Param {
  const void* p;
  int bf;
  __device__ __forceinline__ float at(long c, float none) const {
    if (!p) return none;
    return bf ? __bfloat162float(reinterpret_cast<const bf16*>(p)[c]) : reinterpret_cast<const float*>(p)[c];
  }
  // columns c .. c + VEC - 1
  template <int VEC>
  __device__ __forceinline__ void get(int c, float none, float* v) const {
    if constexpr (VEC == 1) {
      v[0] = at(c, none);
    } else if (!p) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = none;
    } else if (!bf) {
#pragma unroll
      for (int e = 0; e < VEC; e += 4) load<4>(reinterpret_cast<const float*>(p) + c + e, v + e);
    } else if constexpr (VEC == 8) {
      load<8>(reinterpret_cast<const bf16*>(p) + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) load<1>(reinterpret_cast<const bf16*>(p) + c + e, v + e);
    }
  }
};

// Sum over G lanes (all of them get it): rotations inside 16 lanes, exchanges beyond, LDS beyond a wave.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* red) {
#define GSC_ROR(n)                                                                                            \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, true))
  if constexpr (G >= 16) GSC_ROR(8);
  if constexpr (G == 8) v += __shfl_xor(v, 4);
  if constexpr (G >= 16) GSC_ROR(4);
  if constexpr (G >= 16) {
    GSC_ROR(2);
    GSC_ROR(1);
  } else {
    v += __shfl_xor(v, 2);
    v += __shfl_xor(v, 1);
  }
#undef GSC_ROR
  if constexpr (G >= 32) v += __shfl_xor(v, 16);
  if constexpr (G >= 64) v += __shfl_xor(v, 32);
  if constexpr (G > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) v += red[i];
  }
  return v;
}

// Grids of one workgroup per row (or few) have two dimensions: one holds at most 2^32 - 1 threads.
__device__ __forceinline__ long block_of() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }
static dim3 grid_of(long blocks) {
  const long x = std::min<long>(blocks, 1L << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

template <class T, int VEC, int G, int N>
__global__ __launch_bounds__(G > 256 ? G : 256) void fwd_kernel(const T* x, long ldx, Param w, Param b, T* y, float* mean,
                                                                float* rstd, long M, int C, float eps) {
  constexpr int NT = G > 256 ? G : 256, E = VEC * N;
  __shared__ float red[16];
  const int lane = threadIdx.x % G;
  const long row0 = block_of() * (NT / G) + threadIdx.x / G, row = row0 < M ? row0 : M - 1;
  const T* xr = x + row * ldx;
  float v[E];
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[n * VEC + e] = 0.f;
    if (c < C) load<VEC>(xr + c, v + n * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[n * VEC + e];
  }
  const float inv = 1.f / (float)C, mu = group_sum<G>(s, red) * inv;
  float q = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
    if ((n * G + lane) * VEC < C) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[n * VEC + e] -= mu;
        q += v[n * VEC + e] * v[n * VEC + e];
      }
    }
  const float r = 1.f / sqrtf(group_sum<G>(q, red) * inv + eps);
  if (row0 >= M) return;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
    if (c >= C) break;
    float wv[VEC], bv[VEC];
    w.get<VEC>(c, 1.f, wv);
    b.get<VEC>(c, 0.f, bv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[n * VEC + e] = v[n * VEC + e] * r * wv[e] + bv[e];
    store<VEC>(y + row * C + c, v + n * VEC);
  }
  if (lane == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

// dx (if not null) of rows i, i + groups, ..; part (if not null): part[block][0][c] = sum dy xh, part[block][1][c] = sum dy
// over the block's rows.
template <class T, int VEC, int G, int N>
__global__ __launch_bounds__(G > 256 ? G : 256) void bwd_kernel(const T* x, long ldx, const T* dy, long lddy, Param w,
                                                                const float* mean, const float* rstd, T* dx, float* part,
                                                                long M, int C) {
  constexpr int NT = G > 256 ? G : 256, E = VEC * N, WG = NT / G;   // groups of the workgroup
  __shared__ float red[16];
  const int lane = threadIdx.x % G, grp = threadIdx.x / G;
  float wv[E], dw[E], db[E], xv[E], gv[E];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) wv[n * VEC + e] = dw[n * VEC + e] = db[n * VEC + e] = 0.f;
    if (c < C) w.get<VEC>(c, 1.f, wv + n * VEC);
  }
  const float inv = 1.f / (float)C;
  const long stride = (long)gridDim.x * WG;
  // every group of a workgroup makes the same number of turns (the sums of wide rows meet at barriers)
  for (long base = (long)blockIdx.x * WG; base < M; base += stride) {
    const long row0 = base + grp;
    const bool in = row0 < M;
    const long row = in ? row0 : M - 1;
    const float mu = mean[row], r = rstd[row];
    const T *xr = x + row * ldx, *gr = dy + row * lddy;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * G + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        xv[n * VEC + e] = mu;
        gv[n * VEC + e] = 0.f;
      }
      if (in && c < C) {
        load<VEC>(xr + c, xv + n * VEC);
        load<VEC>(gr + c, gv + n * VEC);
      }
    }
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      xv[i] = (xv[i] - mu) * r;
      dw[i] += gv[i] * xv[i];
      db[i] += gv[i];
      gv[i] *= wv[i];
      s += gv[i];
      q += gv[i] * xv[i];
    }
    if (dx) {
      const float ms = group_sum<G>(s, red) * inv, mq = group_sum<G>(q, red) * inv;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * G + lane) * VEC;
        if (!in || c >= C) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) gv[n * VEC + e] = r * (gv[n * VEC + e] - ms - xv[n * VEC + e] * mq);
        store<VEC>(dx + row * C + c, gv + n * VEC);
      }
    }
  }
  if (!part) return;
  float* out = part + (long)blockIdx.x * 2 * C;
  if constexpr (G < 64) {   // the groups of a wave
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int o = G; o < 64; o *= 2) {
        dw[i] += __shfl_xor(dw[i], o);
        db[i] += __shfl_xor(db[i], o);
      }
  }
  if constexpr (G <= 64 && NT > 64) {   // the waves of the workgroup, in order
    constexpr int W = NT / 64, K = G * E;
    __shared__ float sum[2][K];
#pragma unroll
    for (int z = 0; z < W; ++z) {
      if ((int)(threadIdx.x >> 6) == z && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int k = i * G + lane;
          sum[0][k] = z ? sum[0][k] + dw[i] : dw[i];
          sum[1][k] = z ? sum[1][k] + db[i] : db[i];
        }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x; k < 2 * K; k += NT) {
      const int i = (k % K) / G, l = k % G, c = ((i / VEC) * G + l) * VEC + i % VEC;
      if (c < C) out[(long)(k / K) * C + c] = sum[k / K][k % K];
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = ((i / VEC) * G + lane) * VEC + i % VEC;
      if (c < C) {
        out[c] = dw[i];
        out[C + c] = db[i];
      }
    }
  }
}

// ---- rows too long for registers: three passes over a row by a workgroup, column sums by a kernel of their own

template <class T>
__global__ __launch_bounds__(1024) void fwd_long_kernel(const T* x, long ldx, Param w, Param b, T* y, float* mean,
                                                        float* rstd, long M, int C, float eps) {
  __shared__ float red[16];
  const long row = block_of();
  if (row >= M) return;
  const T* xr = x + row * ldx;
  float s = 0.f;
  for (int c = threadIdx.x; c < C; c += 1024) s += to_f(xr[c]);
  const float mu = group_sum<1024>(s, red) / (float)C;
  float q = 0.f;
  for (int c = threadIdx.x; c < C; c += 1024) {
    const float d = to_f(xr[c]) - mu;
    q += d * d;
  }
  const float r = 1.f / sqrtf(group_sum<1024>(q, red) / (float)C + eps);
  for (int c = threadIdx.x; c < C; c += 1024)
    y[row * C + c] = from_f<T>((to_f(xr[c]) - mu) * r * w.at(c, 1.f) + b.at(c, 0.f));
  if (threadIdx.x == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

template <class T>
__global__ __launch_bounds__(1024) void bwd_long_kernel(const T* x, long ldx, const T* dy, long lddy, Param w,
                                                        const float* mean, const float* rstd, T* dx, long M,
                                                        int C) {
  __shared__ float red[16];
  const long row = block_of();
  if (row >= M) return;
  const T *xr = x + row * ldx, *gr = dy + row * lddy;
  const float mu = mean[row], r = rstd[row];
  float s = 0.f, q = 0.f;
  for (int c = threadIdx.x; c < C; c += 1024) {
    const float g = to_f(gr[c]) * w.at(c, 1.f);
    s += g;
    q += g * ((to_f(xr[c]) - mu) * r);
  }
  const float ms = group_sum<1024>(s, red) / (float)C, mq = group_sum<1024>(q, red) / (float)C;
  for (int c = threadIdx.x; c < C; c += 1024) {
    const float g = to_f(gr[c]) * w.at(c, 1.f);
    dx[row * C + c] = from_f<T>(r * (g - ms - (to_f(xr[c]) - mu) * r * mq));
  }
}

template <class T>
__global__ __launch_bounds__(256) void bwd_long_sums_kernel(const T* x, long ldx, const T* dy, long lddy, const float* mean,
                                                            const float* rstd, float* part, long M, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float dw = 0.f, db = 0.f;
  for (long m = blockIdx.y; m < M; m += gridDim.y) {
    const float g = to_f(dy[m * lddy + c]);
    dw += g * ((to_f(x[m * ldx + c]) - mean[m]) * rstd[m]);
    db += g;
  }
  part[(long)blockIdx.y * 2 * C + c] = dw;
  part[((long)blockIdx.y * 2 + 1) * C + c] = db;
}

// Sum of the partial rows: 16 columns x 64 row phases a workgroup, phases added in order.
__global__ __launch_bounds__(1024) void sums_kernel(const float* part, int rows, int C, void* dw, int dw_bf, void* db,
                                                    int db_bf) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, ph = threadIdx.x >> 4;
  const long k = (long)blockIdx.x * 16 + cl;   // column of [dw | db]
  float s = 0.f;
  if (k < 2L * C) {
#pragma unroll 8
    for (int z = ph; z < rows; z += 64) s += part[(long)z * 2 * C + k];
  }
  red[ph][cl] = s;
  __syncthreads();
  if (ph || k >= 2L * C) return;
  for (int q = 1; q < 64; ++q) s += red[q][cl];
  const bool second = k >= C;
  void* out = second ? db : dw;
  if (!out) return;
  const long c = second ? k - C : k;
  if (second ? db_bf : dw_bf) reinterpret_cast<bf16*>(out)[c] = __float2bfloat16(s);
  else reinterpret_cast<float*>(out)[c] = s;
}

// ---- launches

// Lanes per row and pieces per lane of a row of C elements in pieces of VEC: the fewest lanes that hold it in 16 elements
// each (8 where an element is a piece) -- the backward pass keeps five values an element in registers, and with 32 of them
// too few waves fit to cover the loads (16384 x 8192 bf16: 237 us with 256 lanes, 175 us with 512).
// g = 0: too long for registers.
struct Shape {
  int g, n;
};
static Shape shape_of(long C, int vec) {
  const long p = (C + vec - 1) / vec;   // pieces
  for (int g : {8, 16, 32, 64})
    if (p <= g) return {g, 1};
  const int most = vec == 8 ? 2 : vec == 4 ? 4 : 8;
  for (int g : {64, 256, 512, 1024})
    for (int n : {1, 2, 4, 8})
      if (n <= most && (g == 256 || 2 * n >= most) && p <= (long)g * n) return {g, n};
  return {0, 0};
}

static int vec_of(uintptr_t x, long ldx, uintptr_t y, long ldy, uintptr_t w, uintptr_t b, long C, int bf) {
  const int v = bf ? 8 : 4;
  return (x | y | w | b) % 16 == 0 && ldx % v == 0 && ldy % v == 0 && C % v == 0 ? v : 1;
}

// Partial rows of the backward: workgroups, each over rows / workgroups rows (at most 1,024, and 8 MB of partial sums or 512).
static int parts_of(long M, long C, int vec) {
  const Shape sh = shape_of(C, vec);
  if (!sh.g) return (int)std::max<long>(1, std::min<long>({256, M / 16, (1L << 27) / C}));   // at most 1 GB
  const long wg = sh.g > 256 ? 1 : 256 / sh.g;
  return (int)std::max<long>(1, std::min<long>({(M + wg - 1) / wg, 1024, std::max<long>(512, (1L << 21) / (2 * C))}));
}

// f(lanes, pieces) with both as constants.
template <int VEC, class F>
static void by_shape(Shape sh, F&& f) {
#define GSC_SHAPE(G, N)                                                      \
  if (sh.g == G && sh.n == N) {                                              \
    f(std::integral_constant<int, G>{}, std::integral_constant<int, N>{});   \
    return;                                                                  \
  }
  GSC_SHAPE(8, 1) GSC_SHAPE(16, 1) GSC_SHAPE(32, 1) GSC_SHAPE(64, 1)
  if constexpr (VEC == 8) {
    GSC_SHAPE(64, 2) GSC_SHAPE(256, 1) GSC_SHAPE(256, 2) GSC_SHAPE(512, 2) GSC_SHAPE(1024, 2)
  } else if constexpr (VEC == 4) {
    GSC_SHAPE(64, 2) GSC_SHAPE(64, 4) GSC_SHAPE(256, 2) GSC_SHAPE(256, 4) GSC_SHAPE(512, 4) GSC_SHAPE(1024, 4)
  } else {
    GSC_SHAPE(64, 4) GSC_SHAPE(64, 8) GSC_SHAPE(256, 4) GSC_SHAPE(256, 8) GSC_SHAPE(512, 8) GSC_SHAPE(1024, 8)
  }
#undef GSC_SHAPE
  GSC_CHECK(false, "layer_norm: no kernel for this shape");
}

template <class T, int VEC>
static void run_fwd(uintptr_t x, long ldx, Param w, Param b, uintptr_t y, uintptr_t mean, uintptr_t rstd, long M, int C,
                    float eps, hipStream_t s) {
  const Shape sh = shape_of(C, VEC);
  if (!sh.g) {
    hipLaunchKernelGGL((fwd_long_kernel<T>), grid_of(M), dim3(1024), 0, s, ptr<const T>(x), ldx, w, b, ptr<T>(y),
                       ptr<float>(mean), ptr<float>(rstd), M, C, eps);
  } else {
    by_shape<VEC>(sh, [&](auto g, auto n) {
      constexpr int G = decltype(g)::value, N = decltype(n)::value, NT = G > 256 ? G : 256;
      hipLaunchKernelGGL((fwd_kernel<T, VEC, G, N>), grid_of((M + NT / G - 1) / (NT / G)), dim3(NT), 0, s,
                         ptr<const T>(x), ldx, w, b, ptr<T>(y), ptr<float>(mean), ptr<float>(rstd), M, C, eps);
    });
  }
  check_launch();
}

template <class T, int VEC>
static void run_bwd(uintptr_t x, long ldx, uintptr_t dy, long lddy, Param w, uintptr_t mean, uintptr_t rstd, uintptr_t dx,
                    uintptr_t part, long M, int C, hipStream_t s) {
  const Shape sh = shape_of(C, VEC);
  const int parts = parts_of(M, C, VEC);
  if (!sh.g) {
    if (dx)
      hipLaunchKernelGGL((bwd_long_kernel<T>), grid_of(M), dim3(1024), 0, s, ptr<const T>(x), ldx, ptr<const T>(dy),
                         lddy, w, ptr<const float>(mean), ptr<const float>(rstd), ptr<T>(dx), M, C);
    if (part)
      hipLaunchKernelGGL((bwd_long_sums_kernel<T>), dim3((C + 255) / 256, parts), dim3(256), 0, s, ptr<const T>(x), ldx,
                         ptr<const T>(dy), lddy, ptr<const float>(mean), ptr<const float>(rstd), ptr<float>(part), M, C);
  } else {
    by_shape<VEC>(sh, [&](auto g, auto n) {
      constexpr int G = decltype(g)::value, N = decltype(n)::value, NT = G > 256 ? G : 256;
      hipLaunchKernelGGL((bwd_kernel<T, VEC, G, N>), dim3((unsigned)parts), dim3(NT), 0, s, ptr<const T>(x), ldx,
                         ptr<const T>(dy), lddy, w, ptr<const float>(mean), ptr<const float>(rstd), ptr<T>(dx),
                         ptr<float>(part), M, C);
    });
  }
  check_launch();
}

static void check_sizes(long M, long C) {
  GSC_CHECK(M >= 1 && M <= 0x7fffffffL && C >= 1 && C <= 1L << 24,
            "layer_norm: rows must be in 1 .. 2^31 - 1, columns in 1 .. 2^24");
}

void forward(uintptr_t x, long ldx, int bf, uintptr_t w, int w_bf, uintptr_t b, int b_bf, uintptr_t y, uintptr_t mean,
             uintptr_t rstd, long M, long C, float eps, uintptr_t stream) {
  check_sizes(M, C);
  const Param pw{ptr<const void>(w), w_bf}, pb{ptr<const void>(b), b_bf};
  const hipStream_t s = stream_of(stream);
  const bool vec = vec_of(x, ldx, y, C, w, b, C, bf) > 1;
  if (bf && vec) run_fwd<bf16, 8>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else if (bf) run_fwd<bf16, 1>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else if (vec) run_fwd<float, 4>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else run_fwd<float, 1>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
}

// fp32 elements of the backward's partial column sums, whatever its operands' alignment.
static long workspace(long M, long C, int bf) {
  check_sizes(M, C);
  return 2 * C * std::max(parts_of(M, C, bf ? 8 : 4), parts_of(M, C, 1));
}

static void backward(uintptr_t x, long ldx, uintptr_t dy, long lddy, int bf, uintptr_t w, int w_bf, uintptr_t mean, uintptr_t rstd,
              uintptr_t dx, uintptr_t dw, int dw_bf, uintptr_t db, int db_bf, uintptr_t part, long M, long C,
              uintptr_t stream) {
  check_sizes(M, C);
  const hipStream_t s = stream_of(stream);
  const Param pw{ptr<const void>(w), w_bf};
  const bool params = dw || db;
  GSC_CHECK(!params || part, "layer_norm: parameter gradients need a workspace");
  const uintptr_t p = params ? part : 0;
  const int vec = vec_of(x, ldx, dy, lddy, w, 0, C, bf);
  if (vec == 8) run_bwd<bf16, 8>(x, ldx, dy, lddy, pw, mean, rstd, dx, p, M, (int)C, s);
  else if (bf) run_bwd<bf16, 1>(x, ldx, dy, lddy, pw, mean, rstd, dx, p, M, (int)C, s);
  else if (vec == 4) run_bwd<float, 4>(x, ldx, dy, lddy, pw, mean, rstd, dx, p, M, (int)C, s);
  else run_bwd<float, 1>(x, ldx, dy, lddy, pw, mean, rstd, dx, p, M, (int)C, s);
  if (params) {
    hipLaunchKernelGGL(sums_kernel, dim3((unsigned)((2 * C + 15) / 16)), dim3(1024), 0, s, ptr<const float>(part),
                       parts_of(M, C, vec), (int)C, ptr<void>(dw), dw_bf, ptr<void>(db), db_bf);
    check_launch();
  }
}

// A backward pass prepared by its forward pass: what is known then, and the call with the rest (0: not asked for).
struct Backward {
  int bf, w_bf;
  uintptr_t stats;   // mean [M], 1/std [M]
  long M, C;
  int dw_bf, db_bf;
  long space;        // fp32 elements of its workspace
  Backward(int bf, int w_bf, uintptr_t stats, long M, long C, int dw_bf, int db_bf)
      : bf(bf), w_bf(w_bf), stats(stats), M(M), C(C), dw_bf(dw_bf), db_bf(db_bf), space(workspace(M, C, bf)) {}
  void run(uintptr_t x, long ldx, uintptr_t dy, long lddy, uintptr_t w, uintptr_t dx, uintptr_t dw, uintptr_t db,
           uintptr_t part, uintptr_t stream) const {
    backward(x, ldx, dy, lddy, bf, w, w_bf, stats, stats + 4 * M, dx, dw, dw_bf, db, db_bf, part, M, C, stream);
  }
};

}  // namespace norm

void register_norm(py::module_& m) {
  m.def("layer_norm_forward", &norm::forward, "layer norm of rows: y, and mean / 1/std per row when asked for");
  py::class_<norm::Backward>(m, "LayerNormBackward", "layer norm gradients (dx, and dw / db through the workspace)")
      .def(py::init<int, int, uintptr_t, long, long, int, int>())
      .def_readonly("space", &norm::Backward::space)
      .def("__call__", &norm::Backward::run);
}

}  // namespace gsc
