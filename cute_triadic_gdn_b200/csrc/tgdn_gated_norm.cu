// The norm after a block (tgdn_norm.cuh), with its gate and, where asked for, the scaled sum into the residual stream.
#include "tgdn_norm.cuh"

namespace tgdn {

// act(z) and its slope.  1 / (1 + exp(-z)) in f32: exp(-z) overflows to infinity below -88 and the quotient is zero there, as it should be.
__device__ __forceinline__ float gate_act(int act, float z, float& slope) {
  const float sig = 1.f / (1.f + __expf(-z));
  const bool silu = act == TGDN_ACT_SILU;
  slope = silu ? sig * fmaf(z, 1.f - sig, 1.f) : sig * (1.f - sig);
  return silu ? z * sig : sig;
}

template <typename TX, typename TR, int VEC, int K, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_fwd_kernel(NormParams p) {
  __shared__ float red[2][NORM_MAX_WARPS];
  const int tpr = p.tpr, lane = threadIdx.x % tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
  float w[K][VEC];
  {
    float c[K][VEC];
    load_small<VEC, K>(p.weight, 1.f, lane, tpr, p.N, w);
    load_small<VEC, K>(p.scale, p.scale_value, lane, tpr, p.N, c);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[k][i] *= c[k][i];
  }
  int phase = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups; base < p.rows; base += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t row = base + group;
    const bool ok = row < p.rows;
    const uint32_t rr = ok ? static_cast<uint32_t>(row) : 0u;
    float x[K][VEC], z[K][VEC], r[K][VEC];
    load_row<TX, VEC, K>(static_cast<const TX*>(p.x.p) + p.x.at(rr), ok, lane, tpr, p.N, x);
    if (p.act) load_row<TX, VEC, K>(static_cast<const TX*>(p.other.p) + p.other.at(rr), ok, lane, tpr, p.N, z);
    load_row<TR, VEC, K>(static_cast<const TR*>(p.residual.p) + p.residual.at(rr), ok && p.residual.p, lane, tpr, p.N, r);
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(x[k][i], x[k][i], ss);
    const float inv = rsqrtf(fmaf(row_sum(ss, tpr, red, phase), p.inv_n, p.eps));
    phase ^= 1;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float slope = 0.f, act = 1.f;
        if (p.act) act = gate_act(p.act, z[k][i], slope);
        r[k][i] = fmaf(x[k][i] * inv * w[k][i], act, r[k][i]);
      }
    store_row<TR, VEC, K>(static_cast<TR*>(p.out) + row * p.N, ok, lane, tpr, p.N, r);
    if (ok && lane == 0 && p.rstd) p.rstd[row] = inv;
  }
}

template <typename TX, typename TR, int VEC, int K, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_bwd_kernel(NormParams p) {
  __shared__ float red[2][NORM_MAX_WARPS];
  __shared__ float area[NORM_BLOCK * VEC * K];
  const int tpr = p.tpr, lane = threadIdx.x % tpr, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
  float w[K][VEC], sum[K][VEC];
  {
    float c[K][VEC];
    load_small<VEC, K>(p.weight, 1.f, lane, tpr, p.N, w);
    load_small<VEC, K>(p.scale, p.scale_value, lane, tpr, p.N, c);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[k][i] *= c[k][i], sum[k][i] = 0.f;
  }
  int phase = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups; base < p.rows; base += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t row = base + group;
    const bool ok = row < p.rows;
    const uint32_t rr = ok ? static_cast<uint32_t>(row) : 0u;
    float n[K][VEC], z[K][VEC], dy[K][VEC];
    load_row<TX, VEC, K>(static_cast<const TX*>(p.x.p) + p.x.at(rr), ok, lane, tpr, p.N, n);
    if (p.act) load_row<TX, VEC, K>(static_cast<const TX*>(p.other.p) + p.other.at(rr), ok, lane, tpr, p.N, z);
    load_row<TR, VEC, K>(static_cast<const TR*>(p.dy.p) + p.dy.at(rr), ok, lane, tpr, p.N, dy);
    const float inv = ok ? p.rstd[row] : 0.f;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float slope = 0.f, act = 1.f;
        if (p.act) act = gate_act(p.act, z[k][i], slope);
        n[k][i] *= inv;
        const float dn = dy[k][i] * n[k][i];
        sum[k][i] = fmaf(dn, act, sum[k][i]);
        if (p.act) z[k][i] = dn * w[k][i] * slope;
        dy[k][i] *= w[k][i] * act;
        s = fmaf(dy[k][i], n[k][i], s);
      }
    if (p.act) store_row<TX, VEC, K>(static_cast<TX*>(p.dother) + row * p.N, ok, lane, tpr, p.N, z);
    s = row_sum(s, tpr, red, phase) * p.inv_n;
    phase ^= 1;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[k][i] = inv * fmaf(-n[k][i], s, dy[k][i]);
    store_row<TX, VEC, K>(static_cast<TX*>(p.dx) + row * p.N, ok, lane, tpr, p.N, n);
  }
  if (p.sums0) leave_sums<VEC, K>(sum, p.sums0, area, lane, group, groups, tpr, p.N);
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
  const NormShape s = norm_shape(N, vectors_ok(N, vec_of(xt), {host_x, gated ? host_gate : nullptr, host_residual, &oo}), vec_of(xt));
  NormParams p = norm_params(rows, N, eps, s, host_weight, host_scale, scale_value);
  p.x = rows_at(host_x); p.other = rows_at(gated ? host_gate : nullptr); p.residual = rows_at(host_residual); p.out = out; p.rstd = rstd; p.act = activation;
  const int blocks = norm_blocks(s, rows);
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
  const NormShape s = norm_shape(N, vectors_ok(N, vec_of(xt), {host_x, gated ? host_gate : nullptr, host_dout, &dxo, &dzo}), vec_of(xt));
  const int blocks = norm_blocks(s, rows);
  const bool want_w = host_dweight && host_dweight->data, want_c = host_dscale && host_dscale->data;
  if ((want_w || want_c) && (!scratch || scratch_floats < static_cast<int64_t>(blocks) * N)) return TGDN_ERR_SCRATCH;
  NormParams p = norm_params(rows, N, 0.f, s, host_weight, host_scale, scale_value);
  p.x = rows_at(host_x); p.other = rows_at(gated ? host_gate : nullptr); p.dy = rows_at(host_dout);
  p.rstd = const_cast<float*>(rstd); p.dx = dx; p.dother = dgate; p.act = activation;
  p.sums0 = want_w || want_c ? scratch : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TGDN_TRY(launch_types<GatedBwd>(xt, ot, s, blocks, p, st));
  if (!p.sums0) return 0;
  return norm_add_up(p.sums0, blocks, N, host_scale, scale_value, want_w ? const_cast<void*>(host_dweight->data) : nullptr, want_w ? host_dweight->type : 0,
                host_weight, 1.f, want_c ? const_cast<void*>(host_dscale->data) : nullptr, want_c ? host_dscale->type : 0, st);
}
