// Rows of elements of three types for the kernels that work channel by channel (gated scan, norms): vectors of VEC elements in registers
// as f32, and the place of a row in a strided tensor.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/tgdn.h"

namespace tgdn {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two 16-bit elements in a word.
template <typename T> __device__ __forceinline__ float2 word_to_f32(uint32_t w);
template <> __device__ __forceinline__ float2 word_to_f32<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 word_to_f32<__half>(uint32_t w) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
template <typename T> __device__ __forceinline__ uint32_t word_from_f32(float lo, float hi);
template <> __device__ __forceinline__ uint32_t word_from_f32<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &v, 4);
  return w;
}
template <> __device__ __forceinline__ uint32_t word_from_f32<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &v, 4);
  return w;
}

// VEC consecutive elements as they lie in memory, in whole words (a single 16-bit element in the low half of one): kept this way until
// they are worked on.  As an array of 16-bit values the compiler takes them apart at once, a register each (65536 x 32 heads of 128:
// 803 us for the gated norm).
template <typename T, int VEC>
struct Raw {
  static constexpr int BYTES = VEC * sizeof(T), WORDS = BYTES < 4 ? 1 : BYTES / 4;
  static_assert(BYTES == 2 || BYTES == 4 || BYTES == 8 || BYTES == 16 || BYTES == 32, "vector size");
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (BYTES == 2) w[0] = *static_cast<const uint16_t*>(p);
    if constexpr (BYTES == 4) w[0] = *static_cast<const uint32_t*>(p);
    if constexpr (BYTES == 8) {
      const uint2 v = *static_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    }
    if constexpr (BYTES >= 16)
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = static_cast<const uint4*>(p)[i / 4];
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (BYTES == 2) *static_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    if constexpr (BYTES == 4) *static_cast<uint32_t*>(p) = w[0];
    if constexpr (BYTES == 8) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    if constexpr (BYTES >= 16)
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) static_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
  // Element i read by itself (the ends of a row).
  __device__ __forceinline__ void load_one(const T* p, int i) {
    if constexpr (sizeof(T) == 4) w[i] = *reinterpret_cast<const uint32_t*>(p);
    else w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << (i % 2 * 16);
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const float2 v = word_to_f32<T>(w[i]);
        f[2 * i] = v.x;
        if constexpr (VEC > 1) f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void put(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = word_from_f32<T>(f[2 * i], VEC > 1 ? f[2 * i + 1] : 0.f);
    }
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_f32_as(T* p, const float* f) {
  Raw<T, VEC> raw;
  raw.put(f);
  raw.store(p);
}

// An element of a small vector whose type is known at run time only (weights, scales).
__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
  if (type == TGDN_F32) return static_cast<const float*>(p)[i];
  if (type == TGDN_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, int64_t i, float v) {
  if (type == TGDN_F32) static_cast<float*>(p)[i] = v;
  else if (type == TGDN_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

inline int type_bytes(int type) { return type == TGDN_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == TGDN_F32 || type == TGDN_BF16 || type == TGDN_F16; }

// True when every row of the tensor starts on a multiple of `vec` elements.
inline bool rows_in_vectors(const tgdn_rows& t, int vec) {
  const int64_t bytes = static_cast<int64_t>(vec) * type_bytes(t.type);
  return reinterpret_cast<uintptr_t>(t.data) % (bytes < 16 ? bytes : 16) == 0 && t.stride_outer % vec == 0 && t.stride_inner % vec == 0;
}

}  // namespace tgdn
