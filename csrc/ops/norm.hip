// Layer norm over the last dimension, forward and backward (gfx950).
//
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_c g - xh mean_c(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// x, y, dy, dx are bf16 or fp32; w and b fp32 or bf16 each (absent: 1 and 0).  Every sum and statistic is fp32, the mean
// corrected by that of the centred values, the variance from those; an output is rounded once.
//
// Bound by memory: a row is read once into registers (G lanes x N pieces of VEC elements), both passes over it run there.
// The backward pass keeps the gradient sums of its columns in registers over all rows that a group of lanes takes, adds the
// groups of a workgroup in LDS and leaves one partial row per workgroup; a second kernel adds those in a fixed order.
// Repeated calls, bytes read and written a second (a large copy: 4.7 TB/s; what fits the 256 MB cache stays there), and of the
// backward's time that of the partial rows' sums:
//   bf16 16384 x 8192    forward 121 us, 4.4 TB/s   backward 176 - 185 us, 4.5 TB/s (sums 12)
//   bf16 65536 x 1024    40 us, 6.7                 85 us, 4.7 (5)          bf16 25600 x 256   6.5 us, 4.0   15 us, 2.6 (4)
//   fp32 32768 x 1023    42 us, 6.4                 85 us, 4.7 (6)
// The correction of the mean costs 3 - 5 % of a wide row's forward pass (16384 x 8192: 118 us without), nothing elsewhere.
#include <hip/hip_bf16.h>
#include <algorithm>
#include <pybind11/pybind11.h>

#include "../common.h"

namespace py = pybind11;

namespace gsc {
namespace norm {

typedef __hip_bfloat16 bf16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ unsigned bits(bf16 v) { return __builtin_bit_cast(unsigned short, v); }

// VEC elements of a row of C >= VEC from column c < C on, in accesses of 16 bytes (8 of bf16 parameters of fp32 rows) at
// any element's alignment: rows of odd lengths start anywhere.  The last piece of a row is read VEC elements before the
// row's end and shifted, so nothing outside the row is touched; elements past the end are 0.  Loading and unpacking are two
// steps, so that a caller sends all its loads first.  (16384 x 8192 bf16 off 16-byte alignment, element by element: forward
// 297 us, backward 480 us; in pieces 143 and 170 us, on aligned rows 121 and 180 us.)  VEC 1: rows shorter than a piece.
template <class T, int VEC>
struct Piece {
  static constexpr int D = VEC == 1 ? 1 : VEC * (int)sizeof(T) / 4;
  typedef unsigned raw __attribute__((ext_vector_type(D), aligned(sizeof(T))));
  unsigned d[D];
  __device__ __forceinline__ void load(const T* row, int c, int C) {
    if constexpr (VEC == 1) {
      if constexpr (sizeof(T) == 2) d[0] = bits(row[c]);
      else d[0] = __builtin_bit_cast(unsigned, row[c]);
    } else {
      const raw q = *reinterpret_cast<const raw*>(row + min(c, C - VEC));
#pragma unroll
      for (int i = 0; i < D; ++i) d[i] = q[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < D; ++i) d[i] = 0;
  }
  __device__ __forceinline__ void shift(int c, int C) {
    if constexpr (VEC > 1) {
      if (c > C - VEC) {   // one lane of a row, and only where VEC does not divide C
        const int s = (c - C + VEC) * (int)sizeof(T);   // bytes to shift by
#pragma unroll
        for (int k = 4 * D; k >= 2; k /= 2) {
          if (!(s & k)) continue;
#pragma unroll
          for (int i = 0; i < D; ++i) {
            const unsigned next = i + 1 < D ? d[i + 1] : 0;
            d[i] = k == 2 ? d[i] >> 16 | next << 16 : i + k / 4 < D ? d[i + k / 4] : 0;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void unpack(float* v) const {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (sizeof(T) == 2) v[e] = __builtin_bit_cast(float, e & 1 ? d[e / 2] & 0xffff0000u : d[e / 2] << 16);
      else v[e] = __builtin_bit_cast(float, d[e]);
    }
  }
  // What was computed from the piece is not kept for a second use (in two registers for every one of the piece's).
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < D; ++i) asm volatile("" : "+v"(d[i]));
  }
  static __device__ __forceinline__ void get(const T* row, int c, int C, float* v) {
    Piece q;
    q.load(row, c, C);
    q.shift(c, C);
    q.unpack(v);
  }
};

template <int VEC, class T>
__device__ __forceinline__ void store(T* row, int c, int C, const float* v) {
  constexpr bool bf = sizeof(T) == 2;
  if (VEC > 1 && c + VEC <= C) {
    typedef typename Piece<T, VEC>::raw raw;
    raw q;
#pragma unroll
    for (int i = 0; i < Piece<T, VEC>::D; ++i) {
      if constexpr (bf) q[i] = bits(__float2bfloat16(v[2 * i])) | bits(__float2bfloat16(v[2 * i + (VEC > 1)])) << 16;
      else q[i] = __builtin_bit_cast(unsigned, v[i]);
    }
    *reinterpret_cast<raw*>(row + c) = q;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (c + e < C) {
        if constexpr (bf) row[c + e] = __float2bfloat16(v[e]);
        else row[c + e] = v[e];
      }
  }
}

// A per-column parameter: fp32 or bf16, or absent.
struct Param {
  const void* p;
  int bf;
  // columns c .. c + VEC - 1; 0 past C
  template <int VEC>
  __device__ __forceinline__ void get(int c, int C, float none, float* v) const {
    constexpr int F = VEC > 4 ? 4 : VEC;
    if (!p) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = none;
    } else if (bf) {
      Piece<bf16, VEC>::get(reinterpret_cast<const bf16*>(p), c, C, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e += F) Piece<float, F>::get(reinterpret_cast<const float*>(p), c + e, C, v + e);
    }
  }
};

// Sum over at most 64 of G lanes (all of them get it): rotations inside 16 lanes, exchanges beyond.
template <int G>
__device__ __forceinline__ float lane_sum(float v) {
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
  return v;
}

// Sums of K values each over G lanes.  Beyond a wave they pass through red[K][16], which no lane may still be reading
// from the call before (one barrier a call: callers alternate between two).
template <int G, int K>
__device__ __forceinline__ void group_sums(float (&v)[K], float (*red)[16]) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lane_sum<G>(v[k]);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = red[k][0];
#pragma unroll
      for (int i = 1; i < G / 64; ++i) v[k] += red[k][i];
    }
  }
}
template <int G>
__device__ __forceinline__ float group_sum(float v, float (*red)[16]) {
  float w[1] = {v};
  group_sums<G>(w, red);
  return w[0];
}

// Grids of one workgroup per row (or few) have two dimensions: one holds at most 2^32 - 1 threads.
__device__ __forceinline__ long block_of() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }
static dim3 grid_of(long blocks) {
  const long x = std::min<long>(blocks, 1L << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

// The mean, corrected by the mean d of x - first, and the mean of the squares about it from q, that about first.  The first
// one is off by the roundings of a long sum and of 1 / C: of a row of equal values it would leave a difference that 1 / sqrt
// (eps) makes visible (30000 in 7 columns: 0.5).  Corrected, such a row's mean is its value.  Where the correction is not
// small beside the spread (again), the difference of the squares' means would cancel: they are summed once more.
struct Mean {
  float mu, shift, var;   // shift: mu - first
  bool again;
};
__device__ __forceinline__ Mean corrected(float first, float d, float q) {
  Mean m;
  m.mu = first + d;
  m.shift = m.mu - first;
  m.var = q - m.shift * (2.f * d - m.shift);
  m.again = m.shift * m.shift > q * (1.f / 1024.f);
  return m;
}

template <class T, int VEC, int G, int N>
__global__ __launch_bounds__(G > 256 ? G : 256) void fwd_kernel(const T* x, long ldx, Param w, Param b, T* y, float* mean,
                                                                float* rstd, long M, int C, float eps) {
  constexpr int NT = G > 256 ? G : 256, E = VEC * N;
  __shared__ float red[4][16];
  const int lane = threadIdx.x % G;
  const long row0 = block_of() * (NT / G) + threadIdx.x / G, row = row0 < M ? row0 : M - 1;
  const T* xr = x + row * ldx;
  Piece<T, VEC> raw[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
    raw[n].zero();
    if (c < C) raw[n].load(xr, c, C);
  }
  float v[E];
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
    if (c < C) raw[n].shift(c, C);
    raw[n].unpack(v + n * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[n * VEC + e];
  }
  const float inv = 1.f / (float)C, first = group_sum<G>(s, red) * inv;
  float sum[2] = {0.f, 0.f};   // of x - first and its square
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
    if (c >= C) break;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[n * VEC + e] -= first;
    if (c + VEC > C) {
#pragma unroll
      for (int e = 1; e < VEC; ++e) v[n * VEC + e] = c + e < C ? v[n * VEC + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum[0] += v[n * VEC + e];
      sum[1] += v[n * VEC + e] * v[n * VEC + e];
    }
  }
  group_sums<G>(sum, red + 1);
  const Mean m = corrected(first, sum[0] * inv, sum[1] * inv);
  float var = m.var;
  if (m.again) {
    float q = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * G + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = v[n * VEC + e] - m.shift;
        q += c + e < C ? d * d : 0.f;
      }
    }
    var = group_sum<G>(q, red + 3) * inv;
  }
  const float mu = m.mu, r = 1.f / sqrtf(var + eps);
  if (row0 >= M) return;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
    if (c >= C) break;
    float wv[VEC], bv[VEC];
    w.get<VEC>(c, C, 1.f, wv);
    b.get<VEC>(c, C, 0.f, bv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[n * VEC + e] = (v[n * VEC + e] - m.shift) * r * wv[e] + bv[e];
    store<VEC>(y + row * C, c, C, v + n * VEC);
  }
  if (lane == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

// Four waves a SIMD (128 registers) where bf16 pieces fit: 16384 x 8192 194 us without, 174 us with; fp32 pieces do not
// (8192 x 8192: 172 us, 178 us with the bound).
// dx (if not null) of rows i, i + groups, ..; part (if not null): part[block][0][c] = sum dy xh, part[block][1][c] = sum dy
// over the block's rows.
template <class T, int VEC, int G, int N>
__global__ __launch_bounds__(G > 256 ? G : 256, sizeof(T) == 2 ? 4 : 2) void bwd_kernel(const T* x, long ldx, const T* dy, long lddy, Param w,
                                                                const float* mean, const float* rstd, T* dx, float* part,
                                                                long M, int C) {
  constexpr int NT = G > 256 ? G : 256, E = VEC * N, WG = NT / G;   // groups of the workgroup
  __shared__ float red[2][2][16];
  int turn = 0;
  const int lane = threadIdx.x % G, grp = threadIdx.x / G;
  float wv[E], dw[E], db[E];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * G + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) wv[n * VEC + e] = dw[n * VEC + e] = db[n * VEC + e] = 0.f;
    if (c < C) w.get<VEC>(c, C, 1.f, wv + n * VEC);
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
    // where nothing is loaded dy is 0, whatever becomes of x
    Piece<T, VEC> rx[N], rg[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * G + lane) * VEC;
      rx[n].zero();
      rg[n].zero();
      if (in && c < C) {
        rx[n].load(xr, c, C);
        rg[n].load(gr, c, C);
      }
    }
    // xh and dy of piece n: unpacked again for dx, so that only the 16-byte pieces live across the sums
    auto get = [&](int n, float* xh, float* g) {
      rx[n].unpack(xh);
      rg[n].unpack(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) xh[e] = (xh[e] - mu) * r;
    };
    float sum[2] = {0.f, 0.f}, xh[VEC], g[VEC];   // of dy w, dy w xh
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * G + lane) * VEC;
      if (c < C) {
        rx[n].shift(c, C);
        rg[n].shift(c, C);
      }
      get(n, xh, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        dw[n * VEC + e] += g[e] * xh[e];
        db[n * VEC + e] += g[e];
        asm volatile("" : "+v"(dw[n * VEC + e]), "+v"(db[n * VEC + e]));   // here, not behind dx with xh and g kept for it
        g[e] *= wv[n * VEC + e];
        sum[0] += g[e];
        sum[1] += g[e] * xh[e];
      }
    }
    if (dx) {
      group_sums<G>(sum, red[turn ^= 1]);
      const float ms = sum[0] * inv, mq = sum[1] * inv;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * G + lane) * VEC;
        if (!in || c >= C) break;
        rx[n].forget();
        rg[n].forget();
        get(n, xh, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = r * (g[e] * wv[n * VEC + e] - ms - xh[e] * mq);
        store<VEC>(dx + row * C, c, C, g);
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
    __shared__ float all[2][K];
#pragma unroll
    for (int z = 0; z < W; ++z) {
      if ((int)(threadIdx.x >> 6) == z && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int k = i * G + lane;
          all[0][k] = z ? all[0][k] + dw[i] : dw[i];
          all[1][k] = z ? all[1][k] + db[i] : db[i];
        }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x; k < 2 * K; k += NT) {
      const int i = (k % K) / G, l = k % G, c = ((i / VEC) * G + l) * VEC + i % VEC;
      if (c < C) out[(long)(k / K) * C + c] = all[k / K][k % K];
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

// ---- rows too long for registers: three passes over a row by a workgroup, column sums by a kernel of their own.  All but
// the first pass read what the caches hold (8192 rows of bf16: 16,384 columns in registers 128 and 203 us, 16,392 so 160 and
// 341 us).

// f(c, left): the pieces of a row that this thread of 1024 takes, and how many of a piece's elements are inside.
template <int VEC, class F>
__device__ __forceinline__ void row_pieces(int C, F&& f) {
  for (int c = threadIdx.x * VEC; c < C; c += 1024 * VEC) f(c, min(VEC, C - c));
}

template <class T, int VEC>
__global__ __launch_bounds__(1024) void fwd_long_kernel(const T* x, long ldx, Param w, Param b, T* y, float* mean,
                                                        float* rstd, long M, int C, float eps) {
  __shared__ float red[4][16];
  const long row = block_of();
  if (row >= M) return;
  const T* xr = x + row * ldx;
  float v[VEC], wv[VEC], bv[VEC];
  float s = 0.f;
  row_pieces<VEC>(C, [&](int c, int) {
    Piece<T, VEC>::get(xr, c, C, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[e];
  });
  const float inv = 1.f / (float)C, first = group_sum<1024>(s, red) * inv;
  float sum[2] = {0.f, 0.f};
  row_pieces<VEC>(C, [&](int c, int left) {
    Piece<T, VEC>::get(xr, c, C, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = e < left ? v[e] - first : 0.f;
      sum[0] += d;
      sum[1] += d * d;
    }
  });
  group_sums<1024>(sum, red + 1);
  const Mean m = corrected(first, sum[0] * inv, sum[1] * inv);
  const float mu = m.mu;
  float var = m.var;
  if (m.again) {
    float q = 0.f;
    row_pieces<VEC>(C, [&](int c, int left) {
      Piece<T, VEC>::get(xr, c, C, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = e < left ? v[e] - mu : 0.f;
        q += d * d;
      }
    });
    var = group_sum<1024>(q, red + 3) * inv;
  }
  const float r = 1.f / sqrtf(var + eps);
  row_pieces<VEC>(C, [&](int c, int) {
    Piece<T, VEC>::get(xr, c, C, v);
    w.get<VEC>(c, C, 1.f, wv);
    b.get<VEC>(c, C, 0.f, bv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (v[e] - mu) * r * wv[e] + bv[e];
    store<VEC>(y + row * C, c, C, v);
  });
  if (threadIdx.x == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
}

template <class T, int VEC>
__global__ __launch_bounds__(1024) void bwd_long_kernel(const T* x, long ldx, const T* dy, long lddy, Param w,
                                                        const float* mean, const float* rstd, T* dx, long M, int C) {
  __shared__ float red[2][16];
  const long row = block_of();
  if (row >= M) return;
  const T *xr = x + row * ldx, *gr = dy + row * lddy;
  const float mu = mean[row], r = rstd[row];
  float xv[VEC], gv[VEC], wv[VEC];
  // xh and g of a piece (g is 0 past C)
  auto get = [&](int c) {
    Piece<T, VEC> rx, rg;
    rx.load(xr, c, C);
    rg.load(gr, c, C);
    rx.shift(c, C);
    rg.shift(c, C);
    rx.unpack(xv);
    rg.unpack(gv);
    w.get<VEC>(c, C, 1.f, wv);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      xv[e] = (xv[e] - mu) * r;
      gv[e] *= wv[e];
    }
  };
  float sum[2] = {0.f, 0.f};
  row_pieces<VEC>(C, [&](int c, int) {
    get(c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum[0] += gv[e];
      sum[1] += gv[e] * xv[e];
    }
  });
  group_sums<1024>(sum, red);
  const float ms = sum[0] / (float)C, mq = sum[1] / (float)C;
  row_pieces<VEC>(C, [&](int c, int) {
    get(c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) gv[e] = r * (gv[e] - ms - xv[e] * mq);
    store<VEC>(dx + row * C, c, C, gv);
  });
}

template <class T, int VEC>
__global__ __launch_bounds__(256) void bwd_long_sums_kernel(const T* x, long ldx, const T* dy, long lddy, const float* mean,
                                                            const float* rstd, float* part, long M, int C) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= C) return;
  float dw[VEC], db[VEC], xv[VEC], gv[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 2
  for (long m = blockIdx.y; m < M; m += gridDim.y) {
    Piece<T, VEC> rx, rg;
    rx.load(x + m * ldx, c, C);
    rg.load(dy + m * lddy, c, C);
    rx.shift(c, C);
    rg.shift(c, C);
    rx.unpack(xv);
    rg.unpack(gv);
    const float mu = mean[m], r = rstd[m];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      dw[e] += gv[e] * ((xv[e] - mu) * r);
      db[e] += gv[e];
    }
  }
  store<VEC>(part + (long)blockIdx.y * 2 * C, c, C, dw);
  store<VEC>(part + ((long)blockIdx.y * 2 + 1) * C, c, C, db);
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
// each -- the backward pass keeps five values an element in registers, and with 32 of them too few waves fit to cover the
// loads (16384 x 8192 bf16: 237 us with 256 lanes, 175 us with 512).
// g = 0: too long for registers.
struct Shape {
  int g, n;
};
static Shape shape_of(long C, int vec) {
  const long p = (C + vec - 1) / vec;   // pieces
  for (int g : {8, 16, 32, 64})
    if (p <= g) return {g, 1};
  const int most = vec == 8 ? 2 : 4;
  for (int g : {64, 256, 512, 1024})
    for (int n : {1, 2, 4})
      if (n <= most && (g == 256 || 2 * n >= most) && p <= (long)g * n) return {g, n};
  return {0, 0};
}

// Elements of a piece: 16 bytes, or one where a row is shorter.
static int vec_of(long C, int bf) {
  const int v = bf ? 8 : 4;
  return C >= v ? v : 1;
}

// Partial rows of the backward: workgroups, each over rows / workgroups rows: at most 1,024, and 8 MB of partial sums or 512
// (16384 x 8192 bf16: 361 us with 256 workgroups, 237 us with 512).
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
  GSC_SHAPE(8, 1)
  if constexpr (VEC > 1) {
    GSC_SHAPE(16, 1) GSC_SHAPE(32, 1) GSC_SHAPE(64, 1) GSC_SHAPE(64, 2) GSC_SHAPE(256, 2)
  }
  if constexpr (VEC == 8) {
    GSC_SHAPE(256, 1) GSC_SHAPE(512, 2) GSC_SHAPE(1024, 2)
  } else if constexpr (VEC == 4) {
    GSC_SHAPE(64, 4) GSC_SHAPE(256, 4) GSC_SHAPE(512, 4) GSC_SHAPE(1024, 4)
  }
#undef GSC_SHAPE
  GSC_CHECK(false, "layer_norm: no kernel for this shape");
}

template <class T, int VEC>
static void run_fwd(uintptr_t x, long ldx, Param w, Param b, uintptr_t y, uintptr_t mean, uintptr_t rstd, long M, int C,
                    float eps, hipStream_t s) {
  const Shape sh = shape_of(C, VEC);
  if (!sh.g) {
    if constexpr (VEC > 1)
      hipLaunchKernelGGL((fwd_long_kernel<T, VEC>), grid_of(M), dim3(1024), 0, s, ptr<const T>(x), ldx, w, b, ptr<T>(y),
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
    if constexpr (VEC > 1) {
      if (dx)
        hipLaunchKernelGGL((bwd_long_kernel<T, VEC>), grid_of(M), dim3(1024), 0, s, ptr<const T>(x), ldx, ptr<const T>(dy),
                           lddy, w, ptr<const float>(mean), ptr<const float>(rstd), ptr<T>(dx), M, C);
      if (part)
        hipLaunchKernelGGL((bwd_long_sums_kernel<T, VEC>), dim3((C + 256 * VEC - 1) / (256 * VEC), parts), dim3(256), 0, s,
                           ptr<const T>(x), ldx, ptr<const T>(dy), lddy, ptr<const float>(mean), ptr<const float>(rstd), ptr<float>(part), M, C);
    }
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
  const int vec = vec_of(C, bf);
  if (vec == 8) run_fwd<bf16, 8>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else if (bf) run_fwd<bf16, 1>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else if (vec == 4) run_fwd<float, 4>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
  else run_fwd<float, 1>(x, ldx, pw, pb, y, mean, rstd, M, (int)C, eps, s);
}

// fp32 elements of the backward's partial column sums.
static long workspace(long M, long C, int bf) {
  check_sizes(M, C);
  return 2 * C * parts_of(M, C, vec_of(C, bf));
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
  const int vec = vec_of(C, bf);
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
