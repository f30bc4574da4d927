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
// the sum before its rounding to the stream's type.  Its backward forms n from the stream as stored, which saves reading x and the residual
// again: with a stream in 16 bits every n is off by up to half a step of that type, which gradients in 16 bits do not show, and which
// dweight and dscale in f32 carry as a mean over the rows.
#pragma once

#include <initializer_list>

#include "tgdn_common.cuh"
#include "tgdn_host.h"
#include "tgdn_kernels.h"
#include "tgdn_rows.cuh"

namespace tgdn {

constexpr int NORM_BLOCK = 256;                  // threads of a block that holds several rows
constexpr int NORM_MAX_WARPS = 32;
// How rows lie on blocks: several a block, or one a block of up to 512 or of up to 1024 threads.
enum NormSize { NORM_GROUPS, NORM_WIDE, NORM_WIDEST };
// Channels of a row a thread.  Sixteen, but for short rows of 32 bits, which would not fit the registers beside the next row's.
constexpr int norm_channels(int bytes, int size) { return bytes == 4 && size == NORM_GROUPS ? 8 : 16; }
// Threads of a block, and blocks an SM, that a kernel's registers are sized for, by time: as many bytes on their way as possible.  Rows of up to
// 8192 channels on vectors' borders spill nothing forward and up to 36 bytes a thread backward, but for the residual norm of heads (44 to 228);
// rows of odd length up to 336 bytes.  Above 8192 channels 64 registers a thread are too few for sixteen channels (up to 400 bytes forward, 328
// to 588 backward, rows of odd length up to 1420); most kernels of single channels spill too (up to 908).
// Forward, rows of up to 512 threads: 80 registers do where both types have 16 bits (65536 x 2048, gated: 189 us with 100 registers, 150 with
// 80 and the next round's gates on their way into L2), not with a stream in 32 bits (32768 x 4096: 264 us with 100 registers, 293 with 80).
constexpr int norm_threads(int size, bool backward, bool small) {
  return size == NORM_GROUPS ? NORM_BLOCK : size == NORM_WIDEST ? 1024 : backward || !small ? 512 : 768;
}
constexpr int norm_blocks_of(int size, bool backward, bool small) { return size != NORM_GROUPS ? 1 : backward || !small ? 2 : 3; }
#define TGDN_NORM_BOUNDS(backward)                                                                    \
  __launch_bounds__(norm_threads(SIZE, backward, sizeof(TX) + sizeof(TR) == 4), norm_blocks_of(SIZE, backward, sizeof(TX) + sizeof(TR) == 4))

struct RowsAt {                                  // row r of the tensor starts at (r / inner) * so + (r % inner) * si
  const void* p;
  int64_t so, si;
  uint32_t inner, magic, shift;                  // inner = 0: one level, r * si;  r / inner = (mulhi(r, magic) + r) >> shift for r < 2^31
  __device__ __forceinline__ int64_t at(uint32_t r) const {
    if (inner == 0) return r * si;
    const uint32_t o = (__umulhi(r, magic) + r) >> shift;
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
  int end_rows;                                  // so many rows at the end of a tensor have less than a vector behind them
};

// A thread's E channels of a row, worked on in pairs by the two-wide f32 instructions.
template <int E>
struct Row {
  float v[E];
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(v[i], v[i + 1]); }
  __device__ __forceinline__ void set(int i, float2 p) { v[i] = p.x, v[i + 1] = p.y; }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = f;
  }
};

// Which channels: its vectors of VEC, the k-th at ((k * tpr) + lane) * VEC - shift.  Rows of any length that follow one another densely start
// `shift` elements behind a vector's border, the same shift for all rows of a group (the rows of a group are multiples of eight apart), so
// that whole vectors are moved although N is no multiple of them; what sticks out at a row's two ends is left out, and written element by
// element.
template <int VEC, int K, bool EDGES>
struct Columns {
  int first, step, N;
  __device__ __forceinline__ Columns(int lane, int tpr, int shift, int N_) : first(lane * VEC - shift), step(tpr * VEC), N(N_) {}
  __device__ __forceinline__ int at(int k) const { return first + k * step; }
  __device__ __forceinline__ bool whole(int c) const { return EDGES ? c >= 0 && c + VEC <= N : c < N; }
  __device__ __forceinline__ bool part(int c) const { return EDGES && c + VEC > 0 && c < N; }
  __device__ __forceinline__ bool holds(int c) const { return (!EDGES || c >= 0) && c < N; }
};

template <typename T, int VEC, int K, bool EDGES>
struct RawRow {
  Raw<T, VEC> raw[K];
  // Vectors at a row's ends bring elements of its neighbours along, which get() leaves out; only the last rows, behind which the tensor
  // ends, take their ends element by element (those reads are waited for at once).
  __device__ __forceinline__ void load(const T* row, bool ok, bool last, const Columns<VEC, K, EDGES>& cols) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = cols.at(k);
      raw[k].zero();
      if (ok && (cols.whole(c) || (cols.part(c) && !last))) {
        raw[k].load(row + c);
      } else if (ok && cols.part(c)) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (cols.holds(c + i)) raw[k].load_one(row + c + i, i);
      }
    }
  }
  __device__ __forceinline__ Row<K * VEC> get(const Columns<VEC, K, EDGES>& cols) const {
    Row<K * VEC> r;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      raw[k].get(r.v + k * VEC);
      const int c = cols.at(k);
      if (EDGES && !cols.whole(c)) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[k * VEC + i] = cols.holds(c + i) ? r.v[k * VEC + i] : 0.f;
      }
    }
    return r;
  }
};
template <typename T, int VEC, int K, bool EDGES>
__device__ __forceinline__ void store_row(T* row, bool ok, const Columns<VEC, K, EDGES>& cols, const Row<K * VEC>& r) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = cols.at(k);
    if (ok && cols.whole(c)) {
      store_f32_as<T, VEC>(row + c, r.v + k * VEC);
    } else if (ok && cols.part(c)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (cols.holds(c + i)) row[c + i] = from_f32<T>(r.v[k * VEC + i]);
    }
  }
}
template <int VEC, int K, bool EDGES>
__device__ __forceinline__ Row<K * VEC> load_small(const SmallVector& s, float otherwise, const Columns<VEC, K, EDGES>& cols) {
  Row<K * VEC> r;
  auto take = [&](auto get) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) r.v[k * VEC + i] = cols.holds(cols.at(k) + i) ? get(cols.at(k) + i) : 0.f;
  };
  if (!s.p) take([&](int) { return otherwise; });
  else if (s.type == TGDN_F32) take([&](int i) { return static_cast<const float*>(s.p)[i]; });
  else if (s.type == TGDN_BF16) take([&](int i) { return to_f32(static_cast<const __nv_bfloat16*>(s.p)[i]); });
  else take([&](int i) { return to_f32(static_cast<const __half*>(s.p)[i]); });
  return r;
}

// A vector over the channels that every row needs, kept in shared memory: a slot per thread, which it alone writes and reads.
template <int E>
struct Held {
  float4* slot;
  int threads;
  __device__ __forceinline__ Held(float4* area, int which) : slot(area + which * (E / 4) * blockDim.x + threadIdx.x), threads(blockDim.x) {}
  __device__ __forceinline__ void put(const Row<E>& v) {
#pragma unroll
    for (int i = 0; i < E; i += 4) slot[i / 4 * threads] = make_float4(v.v[i], v.v[i + 1], v.v[i + 2], v.v[i + 3]);
  }
  __device__ __forceinline__ Row<E> get() const {
    Row<E> v;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 q = slot[i / 4 * threads];
      v.v[i] = q.x, v.v[i + 1] = q.y, v.v[i + 2] = q.z, v.v[i + 3] = q.w;
    }
    return v;
  }
};

// The walk of a thread over its rows: group `group` of the block takes row base + group of every base, all groups together (they meet in
// shuffles and barriers).
template <int VEC, int K, bool EDGES>
struct Walk {
  int tpr, lane, group, groups;
  int64_t base, step;
  Columns<VEC, K, EDGES> cols;
  __device__ __forceinline__ explicit Walk(const NormParams& p)
      : tpr(p.tpr), lane(threadIdx.x % p.tpr), group(threadIdx.x / p.tpr), groups(blockDim.x / p.tpr),
        base(static_cast<int64_t>(blockIdx.x) * groups), step(static_cast<int64_t>(gridDim.x) * groups),
        cols(lane, p.tpr, EDGES ? static_cast<int>((base + group) * p.N % VEC) : 0, p.N) {}
  __device__ __forceinline__ int64_t row() const { return base + group; }
};

// Asks for a row of the next round, on its way into L2 while this one is worked on (one thread; whole 16-byte pieces inside the row).
template <typename T>
__device__ __forceinline__ void pull_row(const T* row, int N) {
  const uintptr_t from = (reinterpret_cast<uintptr_t>(row) + 15) & ~static_cast<uintptr_t>(15), to = reinterpret_cast<uintptr_t>(row + N) & ~static_cast<uintptr_t>(15);
  if (to > from) bulk_prefetch(reinterpret_cast<const void*>(from), static_cast<uint32_t>(to - from));
}

// Sum over the `tpr` threads of a row; every one of them gets it.  Rows of several warps are one per block: `red` is double-buffered by
// the caller (`phase`), so one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float2 pair, int tpr, float (*red)[NORM_MAX_WARPS], int phase) {
  float v = pair.x + pair.y;
  const int width = tpr < 32 ? tpr : 32;
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  if ((threadIdx.x & 31) == 0) red[phase][threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < tpr >> 5; ++w) s += red[phase][w];
  return s;
}

// The sums that the threads of a block hold for the same channels, added up over its groups in their order, and left as the block's partial.
template <int VEC, int K, bool EDGES>
__device__ __forceinline__ void leave_sums(const Row<K * VEC>& s, float* partial, float* area, const Walk<VEC, K, EDGES>& walk, int N) {
  float* out = partial + static_cast<int64_t>(blockIdx.x) * N;
  if (walk.groups == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = walk.cols.at(k) + i;
        if (walk.cols.holds(c)) out[c] = s.v[k * VEC + i];
      }
    return;
  }
  const int pitch = walk.tpr * K * VEC;          // at least N
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = walk.cols.at(k) + i;
      if (walk.cols.holds(c)) area[walk.group * pitch + c] = s.v[k * VEC + i];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < N; c += blockDim.x) {
    float t = 0.f;
    for (int g = 0; g < walk.groups; ++g) t += area[g * pitch + c];
    out[c] = t;
  }
}

// Column sums of the `blocks` partials of N: out0 = factor0 sum, out1 = factor1 sum (each where it is asked for).
int norm_add_up(const float* partials, int blocks, int N, const tgdn_vector* f0, float v0, void* out0, int t0, const tgdn_vector* f1, float v1, void* out1,
                int t1, cudaStream_t st);

}  // namespace tgdn

namespace tgdn {
namespace {

// How a row is laid over threads: `tpr` threads, a power of two of a warp's lanes as far as they go and whole warps beyond.
struct NormShape {
  int vec, tpr, threads, groups, size;
  bool edges, small;
};
NormShape norm_shape(int N, bool vectors, int x_type, int other_type) {
  NormShape s;
  const int bytes = type_bytes(x_type);
  s.small = bytes + type_bytes(other_type) == 4;
  s.vec = vectors ? 16 / bytes : 1;
  s.edges = N % s.vec != 0;
  const int units = (N + (s.edges ? s.vec - 1 : 0) + s.vec - 1) / s.vec * s.vec;
  const int few = (units + norm_channels(bytes, NORM_GROUPS) - 1) / norm_channels(bytes, NORM_GROUPS), many = (units + 15) / 16;
  if (few <= 32) {
    s.size = NORM_GROUPS;
    s.tpr = 1;
    while (s.tpr < few) s.tpr *= 2;
    s.threads = NORM_BLOCK;
  } else {
    s.tpr = s.threads = (many + 31) / 32 * 32;
    s.size = s.threads <= 512 ? NORM_WIDE : NORM_WIDEST;
  }
  if (s.threads > 1024) return norm_shape(N, false, x_type, other_type);     // (the widest rows, where they do not start on a vector's border)
  s.groups = s.threads / s.tpr;
  return s;
}

// Blocks of a pass: as many as hold the rows, at most what the SMs hold at once (a block fetches the vectors over the channels first and
// leaves a partial of its sums last: 3000 rows of 2001 channels in 2368 blocks took 47 us backward, in 500 blocks 28), in whole rounds of
// equal length.  Where a block would walk 32 rows and more it takes a quarter of them and leaves the SMs to even out (forward, 32768 x 4096
// with an f32 stream: 264 -> 248 us; heads of 128 in 32 bits, backward: 442 -> 409 us); backward, one row a block, the partials cost what
// that gains (bf16, 32768 x 4096: 190 -> 210 us), and half is right with 32 bits (446 -> 420 us).  Rows of a group are multiples of eight
// apart.
int norm_blocks(const NormShape& s, int64_t rows, bool backward) {
  const int64_t want = (rows + s.groups - 1) / s.groups;
  const int per_sm = norm_blocks_of(s.size, backward, s.small) * (norm_threads(s.size, backward, s.small) / s.threads);
  int64_t most = static_cast<int64_t>(tgdn_sm_count()) * per_sm;
  if (want >= most * 32) most *= !backward || s.size == NORM_GROUPS ? 4 : s.small ? 1 : 2;
  const int64_t rounds = (want + most - 1) / most;
  const int multiple = !s.edges || s.groups >= 8 ? 1 : 8 / s.groups;
  return static_cast<int>(((want + rounds - 1) / rounds + multiple - 1) / multiple * multiple);
}

// True when the rows can be moved as vectors: every row starts as far behind a vector's border as row * N elements do, and what a vector
// at a row's end takes along lies in the rows behind it.
bool vectors_ok(int64_t rows, int N, int vec, std::initializer_list<const tgdn_rows*> tensors) {
  for (const tgdn_rows* t : tensors) {
    if (!t || !t->data) continue;
    if (reinterpret_cast<uintptr_t>(t->data) % 16) return false;
    if (t->stride_inner % vec != N % vec) return false;
    if (N % vec && (t->stride_inner < N || (t->inner < rows && t->stride_outer < t->inner * t->stride_inner))) return false;
    if (t->inner < rows && t->stride_outer % vec != static_cast<int64_t>(t->inner % vec) * (N % vec) % vec) return false;
  }
  return true;
}

RowsAt rows_at(const tgdn_rows* t, int64_t rows) {
  RowsAt r{};
  if (!t || !t->data) return r;
  r.p = t->data; r.so = t->stride_outer; r.si = t->stride_inner;
  if (r.so == r.si * t->inner || t->inner >= rows) return r;
  r.inner = static_cast<uint32_t>(t->inner);
  while ((uint64_t{1} << r.shift) < r.inner) ++r.shift;
  r.magic = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << r.shift) - r.inner)) / r.inner + 1);
  return r;
}
// (one level: rows of an outer stride that the kernels never read)
tgdn_rows dense(const void* p, int type, int64_t rows, int N) { return tgdn_rows{p, rows, rows * N, N, type}; }
SmallVector small(const tgdn_vector* v) { return v && v->data ? SmallVector{v->data, v->type} : SmallVector{nullptr, 0}; }

int check_rows(const tgdn_rows* t, bool needed) {
  if (!t || !t->data) return needed ? TGDN_ERR_NULL : 0;
  if (!type_known(t->type)) return TGDN_ERR_TYPE;
  return t->inner <= 0 || t->inner > 0x7fffffffLL ? TGDN_ERR_SHAPE : 0;
}
int check_vector(const tgdn_vector* v) { return v && v->data && !type_known(v->type) ? TGDN_ERR_TYPE : 0; }

#define TGDN_TRY(expr) do { if (const int rc_ = (expr)) return rc_; } while (0)

// The kernels by shape: 16-byte vectors (eight channels of 16 bits, four of 32), the same with rows that start inside one, or single
// channels, in the three sizes.
template <typename TX, typename TR, int VEC, bool EDGES, template <typename, typename, int, bool, int> class Launch>
int launch_size(const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  if (s.size == NORM_GROUPS) return Launch<TX, TR, VEC, EDGES, NORM_GROUPS>::go(s, blocks, p, st);
  return s.size == NORM_WIDE ? Launch<TX, TR, VEC, EDGES, NORM_WIDE>::go(s, blocks, p, st) : Launch<TX, TR, VEC, EDGES, NORM_WIDEST>::go(s, blocks, p, st);
}
template <typename TX, typename TR, template <typename, typename, int, bool, int> class Launch>
int launch_shape(const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  constexpr int V = sizeof(TX) == 2 ? 8 : 4;
  if (s.vec == 1) return launch_size<TX, TR, 1, false, Launch>(s, blocks, p, st);
  return s.edges ? launch_size<TX, TR, V, true, Launch>(s, blocks, p, st) : launch_size<TX, TR, V, false, Launch>(s, blocks, p, st);
}
// Dynamic shared memory: two vectors over the channels (which the sums over a block's groups use after them).
template <typename Kernel>
int launch_norm(Kernel kernel, bool* configured, const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  const int bytes = 2 * 16 * 4 * s.threads;
  if (const int rc = tgdn_dynamic_smem(reinterpret_cast<const void*>(kernel), 2 * 16 * 4 * 1024, configured)) return rc;
  kernel<<<blocks, s.threads, bytes, st>>>(p);
  return tgdn_cuda_error(cudaGetLastError());
}
template <template <typename, typename, int, bool, int> class Launch>
int launch_types(int xt, int rt, const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {
  if (xt == TGDN_F32 && rt == TGDN_F32) return launch_shape<float, float, Launch>(s, blocks, p, st);
  if (xt == TGDN_BF16 && rt == TGDN_BF16) return launch_shape<__nv_bfloat16, __nv_bfloat16, Launch>(s, blocks, p, st);
  if (xt == TGDN_BF16 && rt == TGDN_F32) return launch_shape<__nv_bfloat16, float, Launch>(s, blocks, p, st);
  if (xt == TGDN_F16 && rt == TGDN_F16) return launch_shape<__half, __half, Launch>(s, blocks, p, st);
  if (xt == TGDN_F16 && rt == TGDN_F32) return launch_shape<__half, float, Launch>(s, blocks, p, st);
  return TGDN_ERR_TYPE;
}

#define TGDN_LAUNCHER(name, kernel)                                                                    \
  template <typename TX, typename TR, int VEC, bool EDGES, int SIZE> struct name {                     \
    static int go(const NormShape& s, int blocks, const NormParams& p, cudaStream_t st) {              \
      static bool configured[64] = {false};                                                            \
      return launch_norm(kernel<TX, TR, VEC, EDGES, SIZE>, configured, s, blocks, p, st);              \
    }                                                                                                  \
  }

int check_norm(int64_t rows, int N) { return rows <= 0 || rows > 0x7fffffffLL || N <= 0 || N > TGDN_NORM_MAX_CHANNELS ? TGDN_ERR_SHAPE : 0; }

NormParams norm_params(int64_t rows, int N, float eps, const NormShape& s, const tgdn_vector* weight, const tgdn_vector* scale, float scale_value) {
  NormParams p{};
  p.weight = small(weight); p.scale = small(scale); p.scale_value = scale_value; p.eps = eps; p.inv_n = 1.f / static_cast<float>(N);
  p.rows = rows; p.N = N; p.tpr = s.tpr; p.end_rows = (s.vec - 1 + N - 1) / N;
  return p;
}

int vec_of(int xt) { return xt == TGDN_F32 ? 4 : 8; }

}  // namespace
}  // namespace tgdn
