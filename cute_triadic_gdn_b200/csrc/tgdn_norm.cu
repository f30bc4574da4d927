// The norm before a block (tgdn_norm.cuh): residual stream, norm and weight in one pass, and the sums over rows that both norms leave.
#include "tgdn_norm.cuh"

namespace tgdn {

template <typename TX, typename TR, int VEC, bool EDGES, int SIZE>
__global__ void TGDN_NORM_BOUNDS(false) residual_fwd_kernel(NormParams p) {
  constexpr int E = norm_channels(sizeof(TX), SIZE), K = E / VEC;
  extern __shared__ float4 vectors[];
  __shared__ float red[2][NORM_MAX_WARPS];
  Walk<VEC, K, EDGES> walk(p);
  RawRow<TX, VEC, K, EDGES> xr;
  RawRow<TR, VEC, K, EDGES> rr;
  auto request = [&](int64_t row) {              // the next row is on its way while this one is worked on
    const bool ok = row < p.rows;
    const bool last = row >= p.rows - p.end_rows;
    const uint32_t r = ok ? static_cast<uint32_t>(row) : 0u;
    xr.load(static_cast<const TX*>(p.x.p) + p.x.at(r), ok, last, walk.cols);
    rr.load(static_cast<const TR*>(p.other.p) + p.other.at(r), ok, last, walk.cols);
  };
  request(walk.row());
  Held<E> weight(vectors, 0), scale(vectors, 1);
  weight.put(load_small<VEC, K, EDGES>(p.weight, 1.f, walk.cols));
  scale.put(load_small<VEC, K, EDGES>(p.scale, p.scale_value, walk.cols));
  for (int phase = 0; walk.base < p.rows; walk.base += walk.step, phase ^= 1) {
    const int64_t row = walk.row();
    const bool ok = row < p.rows;
    const Row<E> x = xr.get(walk.cols);
    Row<E> r = rr.get(walk.cols);
    request(row + walk.step);
    const Row<E> c = scale.get();
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      r.set(i, __ffma2_rn(c.pair(i), x.pair(i), r.pair(i)));
      ss = __ffma2_rn(r.pair(i), r.pair(i), ss);
    }
    store_row<TR, VEC, K, EDGES>(static_cast<TR*>(p.stream) + row * p.N, ok, walk.cols, r);
    const float inv = rsqrtf(fmaf(row_sum(ss, walk.tpr, red, phase), p.inv_n, p.eps));
    const Row<E> w = weight.get();
#pragma unroll
    for (int i = 0; i < E; i += 2) r.set(i, __fmul2_rn(__fmul2_rn(r.pair(i), make_float2(inv, inv)), w.pair(i)));
    store_row<TX, VEC, K, EDGES>(static_cast<TX*>(p.out) + row * p.N, ok, walk.cols, r);
    if (ok && walk.lane == 0 && p.rstd) p.rstd[row] = inv;
  }
}

template <typename TX, typename TR, int VEC, bool EDGES, int SIZE>
__global__ void TGDN_NORM_BOUNDS(true) residual_bwd_kernel(NormParams p) {
  constexpr int E = norm_channels(sizeof(TX), SIZE), K = E / VEC;
  extern __shared__ float4 vectors[];
  __shared__ float red[2][NORM_MAX_WARPS];
  Walk<VEC, K, EDGES> walk(p);
  RawRow<TR, VEC, K, EDGES> nr, sr;
  RawRow<TX, VEC, K, EDGES> yr, xr;
  constexpr bool AHEAD = SIZE == NORM_GROUPS;   // (one wide row a block: registers are short, and several blocks take turns)
  float next_inv;
  auto request = [&](int64_t row) {
    const bool ok = row < p.rows;
    const bool last = row >= p.rows - p.end_rows;
    const uint32_t r = ok ? static_cast<uint32_t>(row) : 0u;
    nr.load(static_cast<const TR*>(p.stream) + r * static_cast<int64_t>(p.N), ok, last, walk.cols);
    yr.load(static_cast<const TX*>(p.dy.p) + p.dy.at(r), ok && p.dy.p, last, walk.cols);
    sr.load(static_cast<const TR*>(p.dstream.p) + p.dstream.at(r), ok && p.dstream.p, last, walk.cols);
    if (p.sums1) xr.load(static_cast<const TX*>(p.x.p) + p.x.at(r), ok, last, walk.cols);
    next_inv = ok ? p.rstd[row] : 0.f;
  };
  if (AHEAD) request(walk.row());
  Held<E> weight(vectors, 0), scale(vectors, 1);
  weight.put(load_small<VEC, K, EDGES>(p.weight, 1.f, walk.cols));
  scale.put(load_small<VEC, K, EDGES>(p.scale, p.scale_value, walk.cols));
  Row<E> dw, dc;
  dw.fill(0.f);
  dc.fill(0.f);
  for (int phase = 0; walk.base < p.rows; walk.base += walk.step, phase ^= 1) {
    const int64_t row = walk.row();
    const bool ok = row < p.rows;
    if (!AHEAD) {
      request(row);
      if (threadIdx.x == 0 && row + walk.step < p.rows) {
        const uint32_t r = static_cast<uint32_t>(row + walk.step);
        pull_row(static_cast<const TR*>(p.stream) + r * static_cast<int64_t>(p.N), p.N);
        if (p.dy.p) pull_row(static_cast<const TX*>(p.dy.p) + p.dy.at(r), p.N);
        if (p.dstream.p) pull_row(static_cast<const TR*>(p.dstream.p) + p.dstream.at(r), p.N);
        if (p.sums1) pull_row(static_cast<const TX*>(p.x.p) + p.x.at(r), p.N);
      }
    }
    Row<E> n = nr.get(walk.cols), dy = yr.get(walk.cols), ds = sr.get(walk.cols), x;
    if (p.sums1) x = xr.get(walk.cols);
    const float inv = next_inv;
    if (AHEAD) request(row + walk.step);
    const Row<E> w = weight.get();
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      n.set(i, __fmul2_rn(n.pair(i), make_float2(inv, inv)));
      dw.set(i, __ffma2_rn(dy.pair(i), n.pair(i), dw.pair(i)));
      dy.set(i, __fmul2_rn(dy.pair(i), w.pair(i)));
      sum = __ffma2_rn(dy.pair(i), n.pair(i), sum);
    }
    const float s = -row_sum(sum, walk.tpr, red, phase) * p.inv_n;
    const Row<E> c = scale.get();
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      ds.set(i, __ffma2_rn(make_float2(inv, inv), __ffma2_rn(n.pair(i), make_float2(s, s), dy.pair(i)), ds.pair(i)));
      if (p.sums1) dc.set(i, __ffma2_rn(ds.pair(i), x.pair(i), dc.pair(i)));
      dy.set(i, __fmul2_rn(ds.pair(i), c.pair(i)));
    }
    store_row<TR, VEC, K, EDGES>(static_cast<TR*>(p.dother) + row * p.N, ok, walk.cols, ds);
    if (p.dx) store_row<TX, VEC, K, EDGES>(static_cast<TX*>(p.dx) + row * p.N, ok, walk.cols, dy);
  }
  if (p.sums0) leave_sums<VEC, K, EDGES>(dw, p.sums0, reinterpret_cast<float*>(vectors), walk, p.N);
  if (p.sums1) leave_sums<VEC, K, EDGES>(dc, p.sums1, reinterpret_cast<float*>(vectors), walk, p.N);
}

// Column sums of the partials, in the order of the blocks: thread (i, j) adds up every 32nd partial of channel j from the i-th on, then
// the 32 of a channel are added up in order.  out0 = factor0 sum, out1 = factor1 sum (one or both).
constexpr int SUM_ROWS = 32;
struct SumParams {
  const float* partials;
  int blocks, N;
  SmallVector factor0, factor1;
  float value0, value1;
  void *out0, *out1;
  int type0, type1;
};
__global__ void __launch_bounds__(32 * SUM_ROWS) norm_sums_kernel(SumParams p) {
  __shared__ float part[SUM_ROWS][33];
  const int j = threadIdx.x & 31, i = threadIdx.x >> 5, c = blockIdx.x * 32 + j;
  float s = 0.f;
  if (c < p.N)
#pragma unroll 8
    for (int b = i; b < p.blocks; b += SUM_ROWS) s += p.partials[static_cast<int64_t>(b) * p.N + c];
  part[i][j] = s;
  __syncthreads();
  if (i == 0 && c < p.N) {
    s = 0.f;
    for (int k = 0; k < SUM_ROWS; ++k) s += part[k][j];
    if (p.out0) store_any(p.out0, p.type0, c, s * p.factor0.get(c, p.value0));
    if (p.out1) store_any(p.out1, p.type1, c, s * p.factor1.get(c, p.value1));
  }
}

int norm_add_up(const float* partials, int blocks, int N, const tgdn_vector* f0, float v0, void* out0, int t0, const tgdn_vector* f1, float v1, void* out1,
           int t1, cudaStream_t st) {
  SumParams q{partials, blocks, N, small(f0), small(f1), v0, v1, out0, out1, t0, t1};
  norm_sums_kernel<<<(N + 31) / 32, 32 * SUM_ROWS, 0, st>>>(q);
  return tgdn_cuda_error(cudaGetLastError());
}

}  // namespace tgdn

using namespace tgdn;

namespace {
TGDN_LAUNCHER(ResidualFwd, residual_fwd_kernel);
TGDN_LAUNCHER(ResidualBwd, residual_bwd_kernel);
}  // namespace

extern "C" int64_t tgdn_norm_scratch_floats(int64_t rows, int N) {
  if (check_norm(rows, N)) return 0;
  int most = 0;
  for (const int x_type : {TGDN_F32, TGDN_BF16})         // whichever types and layout the call comes with
    for (const int other : {TGDN_F32, TGDN_BF16})
      for (const bool vectors : {true, false}) {
        const int b = norm_blocks(norm_shape(N, vectors, x_type, other), rows, true);
        if (b > most) most = b;
      }
  return 2 * static_cast<int64_t>(most) * N;
}

extern "C" int tgdn_residual_norm_fwd(const tgdn_rows* host_x, const tgdn_rows* host_residual, const tgdn_vector* host_weight,
                                      const tgdn_vector* host_scale, float scale_value, int64_t rows, int N, float eps, void* y,
                                      void* stream_out, float* rstd, void* stream) {
  TGDN_TRY(check_rows(host_x, true)); TGDN_TRY(check_rows(host_residual, true));
  TGDN_TRY(check_vector(host_weight)); TGDN_TRY(check_vector(host_scale)); TGDN_TRY(check_norm(rows, N));
  if (!y || !stream_out) return TGDN_ERR_NULL;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  const int xt = host_x->type, rt = host_residual->type;
  const tgdn_rows yo = dense(y, xt, rows, N), so = dense(stream_out, rt, rows, N);
  const NormShape s = norm_shape(N, vectors_ok(rows, N, vec_of(xt), {host_x, host_residual, &yo, &so}), xt, rt);
  NormParams p = norm_params(rows, N, eps, s, host_weight, host_scale, scale_value);
  p.x = rows_at(host_x, rows); p.other = rows_at(host_residual, rows); p.out = y; p.stream = stream_out; p.rstd = rstd;
  return launch_types<ResidualFwd>(xt, rt, s, norm_blocks(s, rows, false), p, static_cast<cudaStream_t>(stream));
}

extern "C" int tgdn_residual_norm_bwd(const void* stream_in, int stream_type, const tgdn_rows* host_x, int x_type, const tgdn_rows* host_dy,
                                      const tgdn_rows* host_dstream, const tgdn_vector* host_weight, const tgdn_vector* host_scale,
                                      float scale_value, const float* rstd, int64_t rows, int N, void* dresidual, void* dx,
                                      const tgdn_vector* host_dweight, const tgdn_vector* host_dscale, float* scratch, int64_t scratch_floats,
                                      void* stream) {
  TGDN_TRY(check_rows(host_dy, false)); TGDN_TRY(check_rows(host_dstream, false));
  TGDN_TRY(check_vector(host_weight)); TGDN_TRY(check_vector(host_scale)); TGDN_TRY(check_vector(host_dweight)); TGDN_TRY(check_vector(host_dscale));
  TGDN_TRY(check_norm(rows, N));
  const bool want_w = host_dweight && host_dweight->data, want_c = host_dscale && host_dscale->data;
  TGDN_TRY(check_rows(host_x, want_c));
  if (!stream_in || !rstd || !dresidual) return TGDN_ERR_NULL;
  if (!type_known(stream_type) || !type_known(x_type)) return TGDN_ERR_TYPE;
  if (want_c && host_x->type != x_type) return TGDN_ERR_TYPE;
  if ((host_dy && host_dy->data && host_dy->type != x_type) || (host_dstream && host_dstream->data && host_dstream->type != stream_type)) return TGDN_ERR_TYPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  const tgdn_rows si = dense(stream_in, stream_type, rows, N), dr = dense(dresidual, stream_type, rows, N), dxo = dense(dx, x_type, rows, N);
  const NormShape s = norm_shape(N, vectors_ok(rows, N, vec_of(x_type), {&si, &dr, &dxo, host_dy, host_dstream, want_c ? host_x : nullptr}), x_type, stream_type);
  const int blocks = norm_blocks(s, rows, true);
  if ((want_w || want_c) && (!scratch || scratch_floats < 2 * static_cast<int64_t>(blocks) * N)) return TGDN_ERR_SCRATCH;
  NormParams p = norm_params(rows, N, 0.f, s, host_weight, host_scale, scale_value);
  p.x = rows_at(want_c ? host_x : nullptr, rows); p.dy = rows_at(host_dy, rows); p.dstream = rows_at(host_dstream, rows);
  p.stream = const_cast<void*>(stream_in); p.rstd = const_cast<float*>(rstd); p.dother = dresidual; p.dx = dx;
  p.sums0 = want_w ? scratch : nullptr;
  p.sums1 = want_c ? scratch + static_cast<int64_t>(blocks) * N : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TGDN_TRY(launch_types<ResidualBwd>(x_type, stream_type, s, blocks, p, st));
  if (want_w) TGDN_TRY(norm_add_up(p.sums0, blocks, N, nullptr, 1.f, const_cast<void*>(host_dweight->data), host_dweight->type, nullptr, 1.f, nullptr, 0, st));
  if (want_c) TGDN_TRY(norm_add_up(p.sums1, blocks, N, nullptr, 1.f, const_cast<void*>(host_dscale->data), host_dscale->type, nullptr, 1.f, nullptr, 0, st));
  return 0;
}

