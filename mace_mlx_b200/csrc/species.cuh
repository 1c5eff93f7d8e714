// Device helpers shared by the species operators (species.cu, species_linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace mace {

using bf16 = __nv_bfloat16;

// Programmatic dependent launch: a kernel of these operators may be resident while the one before it in its stream
// still runs; it touches nothing of the caller's before pdl_wait(), which returns when that one is complete.
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// an address that is not a multiple of its values' size
template <typename... P>
bool unaligned(int size, const P*... p) { return ((reinterpret_cast<uintptr_t>(p) % size != 0) || ...); }
inline int value_size(int32_t dtype) { return dtype == MACE_F32 ? 4 : 2; }

template <typename... P, typename... A>
int launch(const char* name, void (*kernel)(P...), dim3 grid, unsigned threads, unsigned smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) return fail(MACE_ERR_CUDA, std::string("launch ") + name + ": " + cudaGetErrorString(e));
  return MACE_OK;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(int8_t x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }

// Loads of what a kernel gets.  The kernel before it may have written it, and with a dependent launch that one still
// runs when this one starts: so these are plain loads (the read-only path is for data that nothing writes while the
// kernel lives), and volatile, which keeps them behind pdl_wait().  They depend on no store in the compiler's eyes, but
// the assembler keeps them behind the stores that come before them: load first, store afterwards.
__device__ __forceinline__ uint4 load_in(const uint4* a) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(a));
  return v;
}
__device__ __forceinline__ uint2 load_in(const uint2* a) {
  uint2 v;
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(a));
  return v;
}
__device__ __forceinline__ uint32_t load_in(const uint32_t* a) {
  uint32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(a));
  return v;
}
__device__ __forceinline__ int32_t load_in(const int32_t* a) {
  return (int32_t)load_in(reinterpret_cast<const uint32_t*>(a));
}
__device__ __forceinline__ float load_in(const float* a) {
  return __uint_as_float(load_in(reinterpret_cast<const uint32_t*>(a)));
}
__device__ __forceinline__ bf16 load_in(const bf16* a) {
  uint16_t v;
  asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(a));
  return __ushort_as_bfloat16(v);
}
__device__ __forceinline__ int8_t load_in(const int8_t* a) {
  int32_t v;
  asm volatile("ld.global.s8 %0, [%1];" : "=r"(v) : "l"(a));
  return (int8_t)v;
}

// V consecutive channels: one 16-byte store where they fill it, else one by one
template <typename T, int V>
__device__ __forceinline__ void store_channels(T* dst, const float* v) {
  if constexpr (V * sizeof(T) == 16) {
    uint4 u;
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int k = 0; k < V; ++k) t[k] = from_f32<T>(v[k]);
    *reinterpret_cast<uint4*>(dst) = u;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) dst[k] = from_f32<T>(v[k]);
  }
}

// four consecutive values, aligned to four
__device__ __forceinline__ void load4(const float* src, float* v) {
  const uint4 u = load_in(reinterpret_cast<const uint4*>(src));
  v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void load4(const bf16* src, float* v) {
  const uint2 u = load_in(reinterpret_cast<const uint2*>(src));
  v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
  v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* dst, const float* v) {
  *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(bf16* dst, const float* v) {
  bf16 t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = from_f32<bf16>(v[k]);
  *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(t);
}

// V channels as loaded: one 16-byte piece where they fill it, else single values; APART: never neighbours
template <typename T, int V, bool APART = false>
struct Raw {
  static constexpr bool PIECE = !APART && V * sizeof(T) == 16;
  uint4 piece;
  T one[PIECE ? 1 : V];
  __device__ __forceinline__ void zero() {
    if constexpr (PIECE)
      piece = make_uint4(0, 0, 0, 0);
    else
      for (int k = 0; k < V; ++k) one[k] = from_f32<T>(0.f);
  }
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (PIECE)
      piece = load_in(reinterpret_cast<const uint4*>(src));
    else
      for (int k = 0; k < V; ++k) one[k] = load_in(src + k);
  }
  // channels `hop` apart, those below `left`
  __device__ __forceinline__ void load(const T* src, int hop, int left) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k * hop < left) one[k] = load_in(src + k * hop);
  }
  __device__ __forceinline__ void values(float* v) const {
    if constexpr (!PIECE) {
      for (int k = 0; k < V; ++k) v[k] = to_f32(one[k]);
    } else {
      const uint32_t w[4] = {piece.x, piece.y, piece.z, piece.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          v[k] = __uint_as_float(w[k]);
        } else {
          v[2 * k] = __uint_as_float(w[k] << 16);
          v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ void add_to(float* acc) const {
    float v[V];
    values(v);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += v[k];
  }
};

// 8-bit value of x at scale s = max |x| fl(1 / 127) (0 where s is 0, infinite or NaN): the IEEE quotient rounded to
// the nearest, half to even; the clamp only acts where s is subnormal and the quotient may pass 127
__device__ __forceinline__ int quantise8(float x, float s) {
  if (!(s > 0.f) || s > 3.4028234e38f) return 0;
  return (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f);
}

// Four of them, one per byte.  x times the hardware's 1 / s (2 units in the last place, 2^-22 relative) is within 3.8e-5
// of the quotient, which is at most 127 in magnitude, so it rounds to the same number unless it lies within 6.2e-5 of a
// tie; only then are the four divided.
// Adding 1.5 2^23 rounds to a whole number, half to even, and leaves it in the low bits.
__device__ __forceinline__ uint32_t quantise8x4(const float* x, float s) {
  const float inv = __fdividef(1.0f, s);
  uint32_t w[4];
  bool tie = !(s > 1e-30f && s < 1e30f);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float r = x[k] * inv, t = r + 12582912.f;
    w[k] = __float_as_uint(t);
    tie |= fabsf(r - (t - 12582912.f)) > 0.5f - 6.2e-5f;
  }
  if (tie) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)quantise8(x[k], s);
  }
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

// rows [lo, hi) of `order` that belong to group g, kept inside [0, n] whatever offsets holds
struct Range {
  int64_t lo, hi;
};
__device__ __forceinline__ Range group_range(const int32_t* offsets, int g, int64_t n) {
  Range r;
  r.lo = min(max((int64_t)offsets[g], (int64_t)0), n);
  r.hi = min(max((int64_t)offsets[g + 1], r.lo), n);
  return r;
}

}  // namespace mace
