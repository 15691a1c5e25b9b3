// Residual add with dropout, and its backward:
//   out = residual + alpha m x,   dx = alpha m dout
// with m = keep ? scale : 0 of the counter-based generator (g5moe_dropout in g5moe.h; row =
// the row of x, column = the column).  The mask is never stored: the backward forms it again
// from the seed.  One fp32 multiply-add and one rounding per element.
//
// What bounds it: memory, two reads and one write (one and one in the backward) per element;
// a thread moves 16 bytes of each operand, and its hashes (one per two elements, two for the
// row) are hidden behind the loads.  36,400 x 768 bf16: 25.7 us, backward 19 us (6.5 and 5.9
// TB/s, where part of the operands is still in the last-level cache; a large copy reaches 4.9);
// 777 x 768 fp32 3.2 us each, launch and latency.
#include <algorithm>

#include "g5moe_internal.h"

namespace g5moe {
namespace {

// 16 bytes of T as floats and back.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void load(float (&f)[kN], const void* p) {
    const float4 v = *static_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  static __device__ __forceinline__ void store(void* p, const float (&f)[kN]) {
    *static_cast<float4*>(p) = float4{f[0], f[1], f[2], f[3]};
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct Vec<uint16_t> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void load(float (&f)[kN], const void* p) {
    const uint4 v = *static_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16_bits_to_f32(w[i] & 0xffffu);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(void* p, const float (&f)[kN]) {
    *static_cast<uint4*>(p) = uint4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                    pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  }
  static __device__ __forceinline__ float get(const uint16_t* p) { return bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
};

// up = alpha * scale.  ADD: out = residual + m x (forward); else out = m x (backward).
// Rows of whole 16-byte pieces (VEC), or element by element.
template <typename T, bool ADD, bool VEC>
__global__ __launch_bounds__(256) void dropout_add_kernel(const T* __restrict__ x,
                                                          const T* __restrict__ residual,
                                                          T* __restrict__ out, int64_t pieces,
                                                          uint32_t per_row, float up,
                                                          DropoutParams drop) {
  constexpr int N = VEC ? Vec<T>::kN : 1;
  for (int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x; u < pieces;
       u += int64_t(gridDim.x) * 256) {
    // 32-bit division where the numbers allow it
    const int64_t row =
        pieces <= int64_t(UINT32_MAX) ? int64_t(uint32_t(u) / per_row) : u / per_row;
    const uint32_t c0 = uint32_t(u - row * per_row) * N;
    const uint32_t key = dropout_row_key(uint32_t(row), drop.seed_lo, drop.seed_hi);
    if constexpr (VEC) {
      float v[N], r[N];
      Vec<T>::load(v, x + u * N);
      if constexpr (ADD) Vec<T>::load(r, residual + u * N);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint32_t bits = dropout_pair_bits(key, (c0 + i) >> 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool keep = (e == 0 ? bits & 0xffffu : bits >> 16) >= drop.thr;
          const float base = ADD ? r[i + e] : 0.0f;
          v[i + e] = keep ? __builtin_fmaf(v[i + e], up, base) : base;
        }
      }
      Vec<T>::store(out + u * N, v);
    } else {
      const uint32_t bits = dropout_pair_bits(key, c0 >> 1);
      const bool keep = ((c0 & 1) ? bits >> 16 : bits & 0xffffu) >= drop.thr;
      const float base = ADD ? Vec<T>::get(residual + u) : 0.0f;
      Vec<T>::put(out + u, keep ? __builtin_fmaf(Vec<T>::get(x + u), up, base) : base);
    }
  }
}

template <typename T>
hipError_t launch(const void* x, const void* residual, void* out, int64_t rows, int d, float up,
                  const DropoutParams& drop, hipStream_t st) {
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                          reinterpret_cast<uintptr_t>(out);
  const bool vec = d % Vec<T>::kN == 0 && align % 16 == 0;
  const int per_row = vec ? d / Vec<T>::kN : d;
  const int64_t pieces = rows * per_row;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(std::min<int64_t>((pieces + 255) / 256, 1 << 20))),
                       dim3(256), 0, st,
                       static_cast<const T*>(x), static_cast<const T*>(residual),
                       static_cast<T*>(out), pieces, uint32_t(per_row), up, drop);
    return hipGetLastError();
  };
  if (residual != nullptr)
    return vec ? go(dropout_add_kernel<T, true, true>) : go(dropout_add_kernel<T, true, false>);
  return vec ? go(dropout_add_kernel<T, false, true>) : go(dropout_add_kernel<T, false, false>);
}

}  // namespace

hipError_t launch_dropout_add(const void* x, const void* residual, void* out, int64_t rows, int d,
                              bool f32, float alpha, const DropoutParams& drop, hipStream_t st) {
  const float up = alpha * (drop.on ? drop.scale : 1.0f);
  return f32 ? launch<float>(x, residual, out, rows, d, up, drop, st)
             : launch<uint16_t>(x, residual, out, rows, d, up, drop, st);
}

}  // namespace g5moe
