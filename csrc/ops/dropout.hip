// Dropout from a counter-based generator: the mask is a function of (seed, offset, element index) and is never stored.
//
//   T = min(round(p 2^32), 2^32 - 1),  group g = i / 8 and lane j = i % 8 of element i (row-major)
//   A = Philox4x32-10(key = seed, counter = (g, offset)),  B the same with the counter's top bit set
//   u = (half j of A) 2^16 + (half j of B)          half j: bits 16 (j & 1) .. of word j / 2
//   y = u >= T ? x / (1 - p) : 0  (+ residual)
//
// The backward pass is the same kernel on dy.  p holds to 2^-32 at 16 random bits an element: B is drawn only where the
// upper half equals that of T (one element in 65,536).
#include <hip/hip_bf16.h>
#include <algorithm>
#include <pybind11/pybind11.h>

#include "../common.h"
#include "../sim/philox.h"

namespace py = pybind11;

namespace gsc {
namespace drop {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

__device__ __forceinline__ Philox4 block(uint64_t seed, uint64_t group, uint64_t offset) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c0, c1, c2, c3, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox4{{c0, c1, c2, c3}};
}

// Which of a group's 8 elements stay, one bit each.
__device__ __forceinline__ uint32_t keep_bits(uint64_t seed, uint64_t group, uint64_t offset, uint32_t thr) {
  const Philox4 a = block(seed, group, offset);
  const uint32_t th = thr >> 16, tl = thr & 0xffffu;
  uint32_t keep = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = (a.v[j >> 1] >> (16 * (j & 1))) & 0xffffu;
    keep |= (h > th ? 1u : 0u) << j;
    tie |= (h == th ? 1u : 0u) << j;
  }
  if (tie) {
    const Philox4 b = block(seed, group, offset | (1ull << 63));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t l = (b.v[j >> 1] >> (16 * (j & 1))) & 0xffffu;
      if (l >= tl) keep |= tie & (1u << j);
    }
  }
  return keep;
}

typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef short s16x8 __attribute__((ext_vector_type(8), aligned(2)));

// The 8 elements of a group, in 16-byte accesses at any element's alignment (52 M elements off 16-byte alignment: fp32
// 235 us element by element, 74 us so; bf16 80 and 38 us).
struct Eight {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  }
  __device__ __forceinline__ void load(const __hip_bfloat16* p) {
    const s16x8 a = *reinterpret_cast<const s16x8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __bfloat162float(__builtin_bit_cast(__hip_bfloat16, (short)a[e]));
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ void store(__hip_bfloat16* p) const {
    s16x8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = __builtin_bit_cast(short, __float2bfloat16(v[e]));
    *reinterpret_cast<s16x8*>(p) = a;
  }
};

// A thread takes whole groups.  The loads are sent before the generator runs (about 20 wide multiplies and 60 other
// instructions a group), so its arithmetic hides behind them: the kernel runs at the rate of the memory (25601 x 2047
// fp32: 72 us, 5.8 TB/s; 25600 x 256 bf16 with a residual: 8.7 us, 4.5 TB/s).
template <class T>
__global__ __launch_bounds__(256) void drop_kernel(const T* x, const T* res, T* y, long n, uint64_t seed, uint64_t offset,
                                                   const long long* offset_ptr, long long* offset_out, uint32_t thr,
                                                   float scale) {
  const long groups = (n + 7) / 8, first = (long)blockIdx.x * 256 + threadIdx.x;
  if (offset_ptr) offset = (uint64_t)*offset_ptr & ~(1ull << 63);
  if (offset_out && first == 0) *offset_out = (long long)offset;
  for (long g = first; g < groups; g += (long)gridDim.x * 256) {
    const long i0 = 8 * g;
    const bool whole = i0 + 8 <= n;
    Eight a, b;
    if (whole) {
      a.load(x + i0);
      if (res) b.load(res + i0);
    }
    const uint32_t keep = keep_bits(seed, (uint64_t)g, offset, thr);
    if (whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a.v[j] = (keep >> j) & 1u ? a.v[j] * scale : 0.f;
        if (res) a.v[j] += b.v[j];
      }
      a.store(y + i0);
    } else {
      for (int j = 0; j < 8 && i0 + j < n; ++j) {
        float v = (keep >> j) & 1u ? to_f(x[i0 + j]) * scale : 0.f;
        if (res) v += to_f(res[i0 + j]);
        y[i0 + j] = from_f<T>(v);
      }
    }
  }
}

void run(uintptr_t x, uintptr_t res, uintptr_t y, int bf16, long n, uint64_t seed, uint64_t offset, uintptr_t offset_ptr,
         uintptr_t offset_out, double p, uintptr_t stream) {
  GSC_CHECK(p >= 0.0 && p < 1.0, "dropout: p must be in [0, 1)");
  GSC_CHECK(n >= 1, "dropout: no elements");
  const uint32_t thr = (uint32_t)std::min(4294967295.0, __builtin_rint(p * 4294967296.0));
  const float scale = (float)(1.0 / (1.0 - p));
  const long groups = (n + 7) / 8;
  const unsigned grid = (unsigned)std::min<long>((groups + 255) / 256, 1 << 16);
  const hipStream_t s = stream_of(stream);
  auto go = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(drop_kernel<T>, dim3(grid), dim3(256), 0, s, ptr<const T>(x), ptr<const T>(res), ptr<T>(y), n, seed,
                       offset, ptr<const long long>(offset_ptr), ptr<long long>(offset_out), thr, scale);
  };
  if (bf16) go((__hip_bfloat16*)nullptr);
  else go((float*)nullptr);
  check_launch();
}

}  // namespace drop

void register_dropout(py::module_& m) {
  m.def("dropout", &drop::run, "y = keep(seed, offset, i) ? x / (1 - p) : 0 (+ residual), mask never stored");
}

}  // namespace gsc
