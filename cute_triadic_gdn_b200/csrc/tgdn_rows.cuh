// Rows of elements of three types for the kernels that work channel by channel (gated scan, norms): vectors of VEC elements in registers
// as f32, and the place of a row in a strided tensor.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tgdn.h"

namespace tgdn {

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
struct alignas(16) Raw32 { uint4 lo, hi; };
template <> struct RawOf<32> { using type = Raw32; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC elements of T as they lie in memory: what a thread loads or stores in one go (16 bytes at most an instruction).
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  using Raw = typename RawOf<VEC * sizeof(T)>::type;
  union { Raw raw; Pack<T, VEC> pack; } u;
  u.raw = *reinterpret_cast<const Raw*>(p);
  return u.pack;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> zero_pack() {
  Pack<T, VEC> z;
#pragma unroll
  for (int i = 0; i < VEC; ++i) z.v[i] = from_f32<T>(0.f);
  return z;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float* f) {
  using Raw = typename RawOf<VEC * sizeof(T)>::type;
  union { Raw raw; Pack<T, VEC> pack; } u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.pack.v[i] = from_f32<T>(f[i]);
  *reinterpret_cast<Raw*>(p) = u.raw;
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
