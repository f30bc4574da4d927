// The norm after a block (tgdn_norm.cuh), with its gate and, where asked for, the scaled sum into the residual stream.
#include "tgdn_norm.cuh"

namespace tgdn {

__device__ __forceinline__ float power_of_two(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The gate's activation and, where asked for, its slope, two channels at a time.  sigmoid(z) = 1 / (1 + 2^(-z log2 e)): the power of two
// overflows to infinity below z = -88.7 and its reciprocal is zero there, as it should be; a quarter of the sum keeps the reciprocal in the
// range that the hardware does not flush to zero.  Both hardware functions err by two units at most; a
// division in full precision is eight instructions an element more in kernels that are bound by their issue.
template <bool SLOPE>
__device__ __forceinline__ float2 gate_act(bool silu, float2 z, float2& slope) {
  const float2 t = __fmul2_rn(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 quarter = make_float2(0.25f, 0.25f), d = __ffma2_rn(make_float2(power_of_two(t.x), power_of_two(t.y)), quarter, quarter);
  const float2 sig = __fmul2_rn(make_float2(reciprocal(d.x), reciprocal(d.y)), quarter);
  const float2 zs = __fmul2_rn(z, sig);
  if (SLOPE) {                                   // silu: sig (1 + z (1 - sig));  sigmoid: sig (1 - sig)
    const float2 rest = __ffma2_rn(sig, make_float2(-1.f, -1.f), make_float2(1.f, 1.f));
    const float2 f = silu ? __ffma2_rn(z, rest, make_float2(1.f, 1.f)) : rest;
    slope = __fmul2_rn(sig, f);
  }
  return silu ? zs : sig;
}

template <typename TX, typename TR, int VEC, bool EDGES, int SIZE>
__global__ void TGDN_NORM_BOUNDS(false) gated_fwd_kernel(NormParams p) {
  constexpr int E = norm_channels(sizeof(TX), SIZE), K = E / VEC;
  extern __shared__ float4 vectors[];
  __shared__ float red[2][NORM_MAX_WARPS];
  Walk<VEC, K, EDGES> walk(p);
  RawRow<TX, VEC, K, EDGES> xr, zr;
  RawRow<TR, VEC, K, EDGES> rr;
  // The next row is on its way while this one is worked on: x from the start, gate and residual from where this row's are used up.
  auto request = [&](int64_t row, bool front) {
    const bool ok = row < p.rows, last = row >= p.rows - p.end_rows;
    const uint32_t r = ok ? static_cast<uint32_t>(row) : 0u;
    if (front) {
      xr.load(static_cast<const TX*>(p.x.p) + p.x.at(r), ok, last, walk.cols);
      return;
    }
    if (p.act) zr.load(static_cast<const TX*>(p.other.p) + p.other.at(r), ok, last, walk.cols);
    if (p.residual.p) rr.load(static_cast<const TR*>(p.residual.p) + p.residual.at(r), ok, last, walk.cols);
  };
  request(walk.row(), true);
  request(walk.row(), false);
  Held<E> weight(vectors, 0);                    // weight and scale in one
  {
    Row<E> w = load_small<VEC, K, EDGES>(p.weight, 1.f, walk.cols);
    const Row<E> c = load_small<VEC, K, EDGES>(p.scale, p.scale_value, walk.cols);
#pragma unroll
    for (int i = 0; i < E; ++i) w.v[i] *= c.v[i];
    weight.put(w);
  }
  const bool silu = p.act == TGDN_ACT_SILU;
  for (int phase = 0; walk.base < p.rows; walk.base += walk.step, phase ^= 1) {
    const int64_t row = walk.row();
    const bool ok = row < p.rows;
    Row<E> x = xr.get(walk.cols);
    request(row + walk.step, true);
    if (SIZE != NORM_GROUPS && threadIdx.x == 0 && row + walk.step < p.rows) {
      const uint32_t r = static_cast<uint32_t>(row + walk.step);
      if (p.act) pull_row(static_cast<const TX*>(p.other.p) + p.other.at(r), p.N);
      if (p.residual.p) pull_row(static_cast<const TR*>(p.residual.p) + p.residual.at(r), p.N);
    }
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) ss = __ffma2_rn(x.pair(i), x.pair(i), ss);
    const float inv = rsqrtf(fmaf(row_sum(ss, walk.tpr, red, phase), p.inv_n, p.eps));
    const Row<E> w = weight.get();
#pragma unroll
    for (int i = 0; i < E; i += 2) x.set(i, __fmul2_rn(__fmul2_rn(x.pair(i), make_float2(inv, inv)), w.pair(i)));
    if (p.act) {
      const Row<E> z = zr.get(walk.cols);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        float2 slope;
        x.set(i, __fmul2_rn(x.pair(i), gate_act<false>(silu, z.pair(i), slope)));
      }
    }
    if (p.residual.p) {
      const Row<E> r = rr.get(walk.cols);
#pragma unroll
      for (int i = 0; i < E; i += 2) x.set(i, __fadd2_rn(r.pair(i), x.pair(i)));
    }
    request(row + walk.step, false);
    store_row<TR, VEC, K, EDGES>(static_cast<TR*>(p.out) + row * p.N, ok, walk.cols, x);
    if (ok && walk.lane == 0 && p.rstd) p.rstd[row] = inv;
  }
}

template <typename TX, typename TR, int VEC, bool EDGES, int SIZE>
__global__ void TGDN_NORM_BOUNDS(true) gated_bwd_kernel(NormParams p) {
  constexpr int E = norm_channels(sizeof(TX), SIZE), K = E / VEC;
  extern __shared__ float4 vectors[];
  __shared__ float red[2][NORM_MAX_WARPS];
  Walk<VEC, K, EDGES> walk(p);
  RawRow<TX, VEC, K, EDGES> xr, zr;
  RawRow<TR, VEC, K, EDGES> yr;
  constexpr bool AHEAD = SIZE == NORM_GROUPS;   // (one wide row a block: registers are short, and several blocks take turns)
  float next_inv;
  auto request = [&](int64_t row) {
    const bool ok = row < p.rows;
    const bool last = row >= p.rows - p.end_rows;
    const uint32_t r = ok ? static_cast<uint32_t>(row) : 0u;
    xr.load(static_cast<const TX*>(p.x.p) + p.x.at(r), ok, last, walk.cols);
    if (p.act) zr.load(static_cast<const TX*>(p.other.p) + p.other.at(r), ok, last, walk.cols);
    yr.load(static_cast<const TR*>(p.dy.p) + p.dy.at(r), ok, last, walk.cols);
    next_inv = ok ? p.rstd[row] : 0.f;
  };
  if (AHEAD) request(walk.row());
  Held<E> weight(vectors, 0);
  Row<E> sums;
  sums.fill(0.f);
  {
    Row<E> w = load_small<VEC, K, EDGES>(p.weight, 1.f, walk.cols);
    const Row<E> c = load_small<VEC, K, EDGES>(p.scale, p.scale_value, walk.cols);
#pragma unroll
    for (int i = 0; i < E; ++i) w.v[i] *= c.v[i];
    weight.put(w);
  }
  const bool silu = p.act == TGDN_ACT_SILU;
  for (int phase = 0; walk.base < p.rows; walk.base += walk.step, phase ^= 1) {
    const int64_t row = walk.row();
    const bool ok = row < p.rows;
    if (!AHEAD) {
      request(row);
      if (threadIdx.x == 0 && row + walk.step < p.rows) {
        const uint32_t r = static_cast<uint32_t>(row + walk.step);
        pull_row(static_cast<const TX*>(p.x.p) + p.x.at(r), p.N);
        if (p.act) pull_row(static_cast<const TX*>(p.other.p) + p.other.at(r), p.N);
        pull_row(static_cast<const TR*>(p.dy.p) + p.dy.at(r), p.N);
      }
    }
    Row<E> n = xr.get(walk.cols), z, dy = yr.get(walk.cols);
    if (p.act) z = zr.get(walk.cols);
    const float inv = next_inv;
    if (AHEAD) request(row + walk.step);
    const Row<E> w = weight.get();
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      float2 slope, act = make_float2(1.f, 1.f);
      if (p.act) act = gate_act<true>(silu, z.pair(i), slope);
      n.set(i, __fmul2_rn(n.pair(i), make_float2(inv, inv)));
      const float2 dn = __fmul2_rn(dy.pair(i), n.pair(i)), wa = __fmul2_rn(w.pair(i), act);
      sums.set(i, __ffma2_rn(dn, act, sums.pair(i)));
      if (p.act) z.set(i, __fmul2_rn(__fmul2_rn(dn, w.pair(i)), slope));
      dy.set(i, __fmul2_rn(dy.pair(i), wa));
      sum = __ffma2_rn(dy.pair(i), n.pair(i), sum);
    }
    if (p.act) store_row<TX, VEC, K, EDGES>(static_cast<TX*>(p.dother) + row * p.N, ok, walk.cols, z);
    const float s = -row_sum(sum, walk.tpr, red, phase) * p.inv_n;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      n.set(i, __fmul2_rn(make_float2(inv, inv), __ffma2_rn(n.pair(i), make_float2(s, s), dy.pair(i))));
    }
    store_row<TX, VEC, K, EDGES>(static_cast<TX*>(p.dx) + row * p.N, ok, walk.cols, n);
  }
  if (p.sums0) leave_sums<VEC, K, EDGES>(sums, p.sums0, reinterpret_cast<float*>(vectors), walk, p.N);
}

}  // namespace tgdn

using namespace tgdn;

namespace {
TGDN_LAUNCHER(GatedFwd, gated_fwd_kernel);
TGDN_LAUNCHER(GatedBwd, gated_bwd_kernel);
}  // namespace

extern "C" int tgdn_gated_norm_fwd(const tgdn_rows* host_x, const tgdn_rows* host_gate, int activation, const tgdn_vector* host_weight,
                                   const tgdn_rows* host_residual, const tgdn_vector* host_scale, float scale_value, int64_t rows, int N,
                                   float eps, void* out, int out_type, float* rstd, void* stream) {
  TGDN_TRY(check_rows(host_x, true)); TGDN_TRY(check_rows(host_gate, activation != TGDN_ACT_NONE)); TGDN_TRY(check_rows(host_residual, false));
  TGDN_TRY(check_vector(host_weight)); TGDN_TRY(check_vector(host_scale)); TGDN_TRY(check_norm(rows, N));
  if (!out) return TGDN_ERR_NULL;
  const int xt = host_x->type;
  const bool gated = activation != TGDN_ACT_NONE;
  if (activation < TGDN_ACT_NONE || activation > TGDN_ACT_SIGMOID) return TGDN_ERR_SHAPE;
  if (!type_known(out_type) || (gated && host_gate->type != xt) || (host_residual && host_residual->data && host_residual->type != out_type)) return TGDN_ERR_TYPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  const tgdn_rows oo = dense(out, out_type, rows, N);
  const NormShape s = norm_shape(N, vectors_ok(rows, N, vec_of(xt), {host_x, gated ? host_gate : nullptr, host_residual, &oo}), xt, out_type);
  NormParams p = norm_params(rows, N, eps, s, host_weight, host_scale, scale_value);
  p.x = rows_at(host_x, rows); p.other = rows_at(gated ? host_gate : nullptr, rows); p.residual = rows_at(host_residual, rows); p.out = out; p.rstd = rstd; p.act = activation;
  const int blocks = norm_blocks(s, rows, false);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launch_types<GatedFwd>(xt, out_type, s, blocks, p, st);
}

extern "C" int tgdn_gated_norm_bwd(const tgdn_rows* host_x, const tgdn_rows* host_gate, int activation, const tgdn_rows* host_dout,
                                   const tgdn_vector* host_weight, const tgdn_vector* host_scale, float scale_value, const float* rstd,
                                   int64_t rows, int N, void* dx, void* dgate, const tgdn_vector* host_dweight, const tgdn_vector* host_dscale,
                                   float* scratch, int64_t scratch_floats, void* stream) {
  const bool gated = activation != TGDN_ACT_NONE;
  TGDN_TRY(check_rows(host_x, true)); TGDN_TRY(check_rows(host_gate, gated)); TGDN_TRY(check_rows(host_dout, true));
  TGDN_TRY(check_vector(host_weight)); TGDN_TRY(check_vector(host_scale)); TGDN_TRY(check_vector(host_dweight)); TGDN_TRY(check_vector(host_dscale));
  TGDN_TRY(check_norm(rows, N));
  if (activation < TGDN_ACT_NONE || activation > TGDN_ACT_SIGMOID) return TGDN_ERR_SHAPE;
  if (!rstd || !dx || (gated && !dgate)) return TGDN_ERR_NULL;
  const int xt = host_x->type, ot = host_dout->type;
  if (gated && host_gate->type != xt) return TGDN_ERR_TYPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  const tgdn_rows dxo = dense(dx, xt, rows, N), dzo = dense(gated ? dgate : nullptr, xt, rows, N);
  const NormShape s = norm_shape(N, vectors_ok(rows, N, vec_of(xt), {host_x, gated ? host_gate : nullptr, host_dout, &dxo, &dzo}), xt, ot);
  const int blocks = norm_blocks(s, rows, true);
  const bool want_w = host_dweight && host_dweight->data, want_c = host_dscale && host_dscale->data;
  if ((want_w || want_c) && (!scratch || scratch_floats < static_cast<int64_t>(blocks) * N)) return TGDN_ERR_SCRATCH;
  NormParams p = norm_params(rows, N, 0.f, s, host_weight, host_scale, scale_value);
  p.x = rows_at(host_x, rows); p.other = rows_at(gated ? host_gate : nullptr, rows); p.dy = rows_at(host_dout, rows);
  p.rstd = const_cast<float*>(rstd); p.dx = dx; p.dother = dgate; p.act = activation;
  p.sums0 = want_w || want_c ? scratch : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TGDN_TRY(launch_types<GatedBwd>(xt, ot, s, blocks, p, st));
  if (!p.sums0) return 0;
  return norm_add_up(p.sums0, blocks, N, host_scale, scale_value, want_w ? const_cast<void*>(host_dweight->data) : nullptr, want_w ? host_dweight->type : 0,
                host_weight, 1.f, want_c ? const_cast<void*>(host_dscale->data) : nullptr, want_c ? host_dscale->type : 0, st);
}
