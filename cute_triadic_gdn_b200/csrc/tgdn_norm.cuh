// Norms before and after a block, fused with the residual stream, its scale and the block's gate.  Over rows of N channels:
//
//   before:  stream = residual + scale x,                y = n weight,               n = stream / sqrt(mean(stream^2) + eps)
//   after:   out = [residual +] scale (n weight act(gate)),                          n = x / sqrt(mean(x^2) + eps)
//
// act: SiLU or sigmoid, or no gate.  Backward, with inv = 1 / sqrt(...) kept from the forward (4 bytes a row) and v the gradient of n:
//   d(normed tensor) = inv (v - n mean(v n));
//   before:  v = dy weight, dresidual = dstream + that, dx = scale dresidual, dweight = sum_rows dy n, dscale = sum_rows dresidual x;
//   after:   v = scale dout weight act, dgate = scale dout n weight act', S = sum_rows dout n act, dweight = scale S, dscale = weight S.
//
// HBM streams: every input is read once, every output written once.  A row is held in registers by `tpr` threads, eight or sixteen
// channels each: part of a warp for a head's 128 channels, a block for a row of thousands.  The sums over rows are formed per thread over
// the rows that its block walks (a thread keeps its channels), left as one partial per block, and added up in a fixed order by a second
// small kernel: no atomics, the same bits every time.
//
// Sums, norms and products are f32; a rounding to the tensors' types happens once, at each store.  The norm before a block is taken of
// the sum before its rounding to the stream's type.
#pragma once

#include <initializer_list>

#include "tgdn_common.cuh"
#include "tgdn_host.h"
#include "tgdn_kernels.h"
#include "tgdn_rows.cuh"

namespace tgdn {

constexpr int NORM_BLOCK = 256;                  // threads of a block that holds several rows
constexpr int NORM_MAX_WARPS = 32;

struct RowsAt {                                  // row r of the tensor starts at (r / inner) * so + (r % inner) * si
  const void* p;
  int64_t so, si;
  uint32_t inner;
  __device__ __forceinline__ int64_t at(uint32_t r) const {
    const uint32_t o = r / inner;
    return o * so + (r - o * inner) * si;
  }
};

struct SmallVector {                             // weight or scale: N elements of a type, or none
  const void* p;
  int type;
  __device__ __forceinline__ float get(int i, float otherwise) const { return p ? load_any(p, type, i) : otherwise; }
};

struct NormParams {
  RowsAt x, other, dy, dstream;                  // other: residual (before), gate (after)
  RowsAt residual;                               // after: added to the output
  SmallVector weight, scale;
  void *out, *stream;
  float* rstd;
  void *dx, *dother;
  float *sums0, *sums1;                          // one partial of N per block
  float scale_value, eps, inv_n;
  int64_t rows;
  int N, tpr, act;
};

// Sum over the `tpr` threads of a row; every one of them gets it.  Rows of several warps are one per block: `red` is double-buffered by
// the caller (`phase`), so one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, int tpr, float (*red)[NORM_MAX_WARPS], int phase) {
  const int width = tpr < 32 ? tpr : 32;
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  if ((threadIdx.x & 31) == 0) red[phase][threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < tpr >> 5; ++w) s += red[phase][w];
  return s;
}

// A thread's channels of a row: K vectors of VEC, the k-th at ((k * tpr) + lane) * VEC.
template <typename T, int VEC, int K>
__device__ __forceinline__ void load_row(const T* row, bool ok, int lane, int tpr, int N, float (&out)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * tpr + lane) * VEC;
    const Pack<T, VEC> raw = ok && c < N ? load_pack<T, VEC>(row + c) : zero_pack<T, VEC>();
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[k][i] = to_f32(raw.v[i]);
  }
}
template <typename T, int VEC, int K>
__device__ __forceinline__ void store_row(T* row, bool ok, int lane, int tpr, int N, const float (&v)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * tpr + lane) * VEC;
    if (ok && c < N) store_pack<T, VEC>(row + c, v[k]);
  }
}
template <int VEC, int K>
__device__ __forceinline__ void load_small(const SmallVector& s, float otherwise, int lane, int tpr, int N, float (&out)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * tpr + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[k][i] = c < N ? s.get(c + i, otherwise) : 0.f;
  }
}

// The sums that the threads of a block hold for the same channels, added up over its groups in their order, and left as the block's partial.
template <int VEC, int K>
__device__ __forceinline__ void leave_sums(const float (&v)[K][VEC], float* partial, float* area, int lane, int group, int groups, int tpr, int N) {
  if (groups == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (k * tpr + lane) * VEC + i;
        if (c < N) partial[static_cast<int64_t>(blockIdx.x) * N + c] = v[k][i];
      }
    return;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) area[group * (tpr * K * VEC) + (k * tpr + lane) * VEC + i] = v[k][i];
  __syncthreads();
  for (int c = threadIdx.x; c < N; c += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < groups; ++g) s += area[g * (tpr * K * VEC) + c];
    partial[static_cast<int64_t>(blockIdx.x) * N + c] = s;
  }
}

// Column sums of the `blocks` partials of N: out0 = factor0 sum, out1 = factor1 sum (each where it is asked for).
int norm_add_up(const float* partials, int blocks, int N, const tgdn_vector* f0, float v0, void* out0, int t0, const tgdn_vector* f1, float v1, void* out1,
                int t1, cudaStream_t st);

}  // namespace tgdn

namespace tgdn {
namespace {

// How a row is laid over threads: `tpr` threads of K vectors each.  Part of a warp (a power of two) as far as one vector a thread goes,
// whole warps beyond; two vectors a thread above 128 threads, so that a block of a wide row has fewer warps to wait for.
struct NormShape {
  int vec, k, tpr, threads, groups;
};
NormShape norm_shape(int N, bool vectors, int vec_elements) {
  NormShape s;
  s.vec = vectors ? vec_elements : 1;
  const int per8 = 8 / s.vec, units = (N + s.vec - 1) / s.vec;         // vectors of eight channels' worth
  s.k = (units + per8 - 1) / per8 > 128 ? 2 * per8 : per8;
  const int need = (units + s.k - 1) / s.k;
  if (need <= 32) {
    s.tpr = 1;
    while (s.tpr < need) s.tpr *= 2;
    s.threads = NORM_BLOCK;
  } else {
    s.tpr = (need + 31) / 32 * 32;
    s.threads = s.tpr;
  }
  s.groups = s.threads / s.tpr;
  return s;
}

// Blocks of a pass: as many as hold the rows, at most two thousand threads' worth on every SM.
int norm_blocks(const NormShape& s, int64_t rows) {
  const int64_t want = (rows + s.groups - 1) / s.groups, most = static_cast<int64_t>(tgdn_sm_count()) * (2048 / s.threads > 0 ? 2048 / s.threads : 1);
  return static_cast<int>(want < most ? want : most);
}

bool vectors_ok(int N, int vec, std::initializer_list<const tgdn_rows*> tensors) {
  if (N % vec) return false;
  for (const tgdn_rows* t : tensors)
    if (t && t->data && !rows_in_vectors(*t, vec)) return false;
  return true;
}

RowsAt rows_at(const tgdn_rows* t) {
  if (!t || !t->data) return RowsAt{nullptr, 0, 0, 1u};
  return RowsAt{t->data, t->stride_outer, t->stride_inner, static_cast<uint32_t>(t->inner)};
}
tgdn_rows dense(const void* p, int type, int64_t rows, int N) { return tgdn_rows{p, rows > 0 ? rows : 1, 0, N, type}; }
SmallVector small(const tgdn_vector* v) { return v && v->data ? SmallVector{v->data, v->type} : SmallVector{nullptr, 0}; }

int check_rows(const tgdn_rows* t, bool needed) {
  if (!t || !t->data) return needed ? TGDN_ERR_NULL : 0;
  if (!type_known(t->type)) return TGDN_ERR_TYPE;
  return t->inner <= 0 || t->inner > 0x7fffffffLL ? TGDN_ERR_SHAPE : 0;
}
int check_vector(const tgdn_vector* v) { return v && v->data && !type_known(v->type) ? TGDN_ERR_TYPE : 0; }

#define TGDN_TRY(expr) do { if (const int rc_ = (expr)) return rc_; } while (0)

// The kernels by shape: 16-byte vectors (eight channels of 16 bits, four of 32) or single channels; eight channels a thread, or sixteen in
// blocks of up to 512 and of up to 1024 threads (whose registers differ).
template <typename TX, typename TR, template <typename, typename, int, int, int> class Launch>
int launch_shape(const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  constexpr int V = sizeof(TX) == 2 ? 8 : 4;
  if (s.vec == V) {
    if (s.k == 8 / V) Launch<TX, TR, V, 8 / V, NORM_BLOCK>::go(s, blocks, p, st);
    else if (s.threads <= 512) Launch<TX, TR, V, 16 / V, 512>::go(s, blocks, p, st);
    else Launch<TX, TR, V, 16 / V, 1024>::go(s, blocks, p, st);
  } else {
    if (s.k == 8) Launch<TX, TR, 1, 8, NORM_BLOCK>::go(s, blocks, p, st);
    else if (s.threads <= 512) Launch<TX, TR, 1, 16, 512>::go(s, blocks, p, st);
    else Launch<TX, TR, 1, 16, 1024>::go(s, blocks, p, st);
  }
  return tgdn_cuda_error(cudaGetLastError());
}
template <template <typename, typename, int, int, int> class Launch>
int launch_types(int xt, int rt, const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  if (xt == TGDN_F32 && rt == TGDN_F32) return launch_shape<float, float, Launch>(s, blocks, p, st);
  if (xt == TGDN_BF16 && rt == TGDN_BF16) return launch_shape<__nv_bfloat16, __nv_bfloat16, Launch>(s, blocks, p, st);
  if (xt == TGDN_BF16 && rt == TGDN_F32) return launch_shape<__nv_bfloat16, float, Launch>(s, blocks, p, st);
  if (xt == TGDN_F16 && rt == TGDN_F16) return launch_shape<__half, __half, Launch>(s, blocks, p, st);
  if (xt == TGDN_F16 && rt == TGDN_F32) return launch_shape<__half, float, Launch>(s, blocks, p, st);
  return TGDN_ERR_TYPE;
}

#define TGDN_LAUNCHER(name, kernel)                                                                    \
  template <typename TX, typename TR, int VEC, int K, int MAXT> struct name {                          \
    static void go(const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {             \
      kernel<TX, TR, VEC, K, MAXT><<<blocks, s.threads, 0, st>>>(p);                                   \
    }                                                                                                  \
  }

int check_norm(int64_t rows, int N) { return rows <= 0 || rows > 0x7fffffffLL || N <= 0 || N > TGDN_NORM_MAX_CHANNELS ? TGDN_ERR_SHAPE : 0; }

NormParams norm_params(int64_t rows, int N, float eps, const NormShape& s, const tgdn_vector* weight, const tgdn_vector* scale, float scale_value) {
  NormParams p{};
  p.weight = small(weight); p.scale = small(scale); p.scale_value = scale_value; p.eps = eps; p.inv_n = 1.f / static_cast<float>(N);
  p.rows = rows; p.N = N; p.tpr = s.tpr;
  return p;
}

int vec_of(int xt) { return xt == TGDN_F32 ? 4 : 8; }

}  // namespace
}  // namespace tgdn
