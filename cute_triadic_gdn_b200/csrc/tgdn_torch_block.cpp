// Host path of the operators that stand around the core in a block: the gated scan and its decode step, the norms before and after a
// block.  Same division of labour as in tgdn_torch.cpp: operators in the namespace tgdn_b200 with autograd kernels of their own, checks and
// launches here, the fake implementations in Python beside the calls (gated_scan.py, block_norm.py).
#include "tgdn_torch.h"

#include <ATen/cuda/EmptyTensor.h>

namespace {

using namespace tgdn_torch;
using std::nullopt;

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TGDN_F32;
    case at::kBFloat16: return TGDN_BF16;
    case at::kHalf: return TGDN_F16;
    default: return -1;
  }
}

bool floating(const Tensor& t) { return type_of(t) >= 0; }

void check_place(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == x.device(), name, ": every tensor must live on x's CUDA device");
}

void check_sm100(const Tensor& x, const char* call) {
  TORCH_CHECK_VALUE(at::cuda::getDeviceProperties(x.device().index())->major == 10, call, " requires an sm_100 device");
}

// Outputs straight from the allocator: a small call is the host's time, and the dispatcher's part of an allocation is half of it.
Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}
Tensor none(const Tensor& like) { return fresh({0}, like, at::kFloat); }

// ---- gated scan -------------------------------------------------------------------------------------------------------
// A (B, T, D) tensor as the library reads it; an axis of size one may carry any stride.  Channels apart, or tokens that are 2^31 elements
// apart, are copied together.
struct SequenceRows {
  Tensor held;
  tgdn_rows rows;
  explicit SequenceRows(const Tensor& t)
      : held((t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) == 1 || t.stride(1) < (int64_t{1} << 31)) ? t : t.contiguous()) {
    rows = {held.data_ptr(), held.size(1), held.size(0) == 1 ? 0 : held.stride(0), held.size(1) == 1 ? 0 : held.stride(1), type_of(held)};
  }
};

void check_pair(const Tensor& x, const Tensor& g) {
  TORCH_CHECK_VALUE(floating(x) && (g.scalar_type() == at::kFloat || g.scalar_type() == x.scalar_type()),
                    "x must be float32, bfloat16 or float16 and g float32 or of x's type; got ", x.scalar_type(), " and ", g.scalar_type());
}

void check_scan(const Tensor& x, const Tensor& g, const OptTensor& initial, const OptTensor& map, int64_t documents) {
  TORCH_CHECK_VALUE(x.dim() == 3 && g.sizes() == x.sizes(), "x and g must be (B, T, D) and agree; got ", shape_of(x), " and ", shape_of(g));
  check_pair(x, g);
  check_place(x, x, "x");
  check_place(g, x, "g");
  TORCH_CHECK_VALUE(x.size(0) < (int64_t{1} << 31) && x.size(1) < (int64_t{1} << 31) && x.size(2) < (int64_t{1} << 31),
                    "gated_scan: an axis is limited to 2^31 - 1 elements");
  const int64_t sequences = has(map) ? documents : x.size(0);
  if (has(map))
    TORCH_CHECK_VALUE(x.size(0) == 1 && documents >= 1 && map->dim() == 1 && map->size(0) == x.size(1) && map->scalar_type() == at::kInt &&
                          map->is_contiguous() && map->device() == x.device(),
                      "doc_map: int32 (T), from gated_scan_map, for a packed row (1, T, D)");
  if (has(initial))
    TORCH_CHECK_VALUE(initial->dim() == 2 && initial->size(0) == sequences && initial->size(1) == x.size(2) &&
                          initial->scalar_type() == at::kFloat && initial->device() == x.device(),
                      "initial_state must be an f32 tensor of shape (", sequences, ", ", x.size(2), ") on x's device");
  check_sm100(x, "gated_scan");
}

std::tuple<Tensor, Tensor> scan_map(const Tensor& cu, int64_t tokens) {
  const c10::cuda::CUDAGuard guard(cu.device());
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 2 && cu.is_contiguous() && (cu.scalar_type() == at::kInt || cu.scalar_type() == at::kLong),
                    "cu_seqlens: a contiguous vector of int32 or int64 document offsets, at least [0, T]");
  Tensor map = fresh({tokens}, cu, at::kInt), valid = fresh({1}, cu, at::kBool);
  check_rc(tgdn_scan_map(ptr(cu), cu.scalar_type() == at::kLong ? 1 : 0, static_cast<int>(cu.numel() - 1), static_cast<int>(tokens),
                         ptr<int32_t>(map), ptr<uint8_t>(valid), stream_of(cu)),
           "tgdn_scan_map");
  return {map, valid};
}

Tensor scan_scratch(const Tensor& x) {
  const int64_t floats = tgdn_scan_scratch_floats(static_cast<int>(x.size(0)), static_cast<int>(x.size(1)), static_cast<int>(x.size(2)));
  return floats > 0 ? fresh({floats}, x, at::kFloat) : Tensor();
}

// (h, final state, the state before every tile): the last two are empty unless asked for.
std::tuple<Tensor, Tensor, Tensor> scan_fwd(const Tensor& x, const Tensor& g, const OptTensor& initial, const OptTensor& map, int64_t documents,
                                            bool output_final_state, bool save) {
  check_scan(x, g, initial, map, documents);
  const c10::cuda::CUDAGuard guard(x.device());
  const int B = static_cast<int>(x.size(0)), T = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2));
  const SequenceRows xr(x), gr(g);
  Tensor h = fresh(x.sizes(), x, x.scalar_type()), final_state = none(x), carry = none(x), start;
  if (output_final_state) final_state = fresh({has(map) ? documents : x.size(0), x.size(2)}, x, at::kFloat);
  if (save) carry = fresh({tgdn_scan_carry_floats(B, T, D)}, x, at::kFloat);
  if (has(initial)) start = initial->contiguous();
  const Tensor scratch = scan_scratch(x);
  check_rc(tgdn_scan_fwd(&xr.rows, &gr.rows, ptr<int32_t>(map), static_cast<int>(documents), B, T, D, ptr<float>(start), ptr(h),
                         output_final_state ? ptr<float>(final_state) : nullptr, save ? ptr<float>(carry) : nullptr, ptr<float>(scratch), scratch.defined() ? scratch.numel() : 0,
                         stream_of(x)),
           "tgdn_scan_fwd");
  return {h, final_state, carry};
}

// (dx, dg, dinitial); the last is empty without an initial state.
std::tuple<Tensor, Tensor, Tensor> scan_bwd(const Tensor& x, const Tensor& g, const Tensor& dh, const Tensor& carry, const OptTensor& initial,
                                            const OptTensor& map, int64_t documents, const OptTensor& dfinal) {
  check_scan(x, g, initial, map, documents);
  const c10::cuda::CUDAGuard guard(x.device());
  const int B = static_cast<int>(x.size(0)), T = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2));
  TORCH_CHECK_VALUE(dh.sizes() == x.sizes() && dh.scalar_type() == x.scalar_type() && dh.device() == x.device(), "dh must be like x");
  TORCH_CHECK_VALUE(carry.scalar_type() == at::kFloat && carry.is_contiguous() && carry.device() == x.device() &&
                        carry.numel() == tgdn_scan_carry_floats(B, T, D),
                    "carry must be what gated_scan_fwd saved");
  const int64_t sequences = has(map) ? documents : x.size(0);
  if (has(dfinal))
    TORCH_CHECK_VALUE(dfinal->dim() == 2 && dfinal->size(0) == sequences && dfinal->size(1) == x.size(2) && dfinal->scalar_type() == at::kFloat &&
                          dfinal->device() == x.device(),
                      "dfinal must be like the final state");
  const SequenceRows xr(x), gr(g), hr(dh);
  Tensor dx = fresh(x.sizes(), x, x.scalar_type()), dg = fresh(x.sizes(), x, g.scalar_type()), dinitial = none(x), start, end;
  if (has(initial)) {
    start = initial->contiguous();
    dinitial = fresh({sequences, x.size(2)}, x, at::kFloat);
  }
  if (has(dfinal)) end = dfinal->contiguous();
  const Tensor scratch = scan_scratch(x);
  check_rc(tgdn_scan_bwd(&xr.rows, &gr.rows, &hr.rows, ptr<int32_t>(map), static_cast<int>(documents), B, T, D, ptr<float>(start),
                         ptr<float>(carry), ptr<float>(end), ptr(dx), ptr(dg), has(initial) ? ptr<float>(dinitial) : nullptr, ptr<float>(scratch),
                         scratch.defined() ? scratch.numel() : 0, stream_of(x)),
           "tgdn_scan_bwd");
  return {dx, dg, dinitial};
}

using ScanOut = std::tuple<Tensor, Tensor, Tensor>;
ScanOut call_scan_fwd(const Tensor& x, const Tensor& g, const OptTensor& initial, const OptTensor& map, int64_t documents, bool final_state,
                      bool save) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::gated_scan_fwd", "").typed<decltype(scan_fwd)>();
  return op.call(x, g, initial, map, documents, final_state, save);
}

struct ScanSteps {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const OptTensor& initial, const OptTensor& map,
                               int64_t documents, bool output_final_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [h, final_state, carry] = call_scan_fwd(x, g, initial, map, documents, output_final_state, true);
    ctx->save_for_backward({x, g, carry, or_undefined(initial), or_undefined(map)});
    ctx->saved_data["documents"] = documents;
    if (output_final_state) ctx->mark_non_differentiable({carry});
    else ctx->mark_non_differentiable({final_state, carry});
    ctx->set_materialize_grads(false);
    return {h, final_state, carry};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(6);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    variable_list s = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::gated_scan_bwd", "").typed<decltype(scan_bwd)>();
    const Tensor dh = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
    auto [dx, dg, dinitial] = op.call(s[0], s[1], dh, s[2], or_nullopt(s[3]), or_nullopt(s[4]), ctx->saved_data["documents"].toInt(),
                                      or_nullopt(grads[1]));
    res[0] = dx;
    res[1] = dg;
    if (s[3].defined()) res[2] = dinitial;
    return res;
  }
};
using ScanFunction = Differentiable<ScanSteps>;

ScanOut scan_fwd_autograd(const Tensor& x, const Tensor& g, const OptTensor& initial, const OptTensor& map, int64_t documents,
                          bool output_final_state, bool save) {
  const Tensor undefined, &start = has(initial) ? *initial : undefined;
  if (!any_grad({&x, &g}) && !(start.defined() && any_grad({&start}))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_scan_fwd(x, g, initial, map, documents, output_final_state, save);
  }
  variable_list out = ScanFunction::apply(x, g, initial, map, documents, output_final_state);
  return {out[0], out[1], out[2]};
}

// The calls' way in: the packed row's rules are those of the core (what can be checked without reading the offsets here, the offsets
// themselves on the device).
std::tuple<Tensor, OptTensor> scan_call(const Tensor& x, const Tensor& g, const OptTensor& cu, const OptTensor& initial, bool output_final_state) {
  OptTensor map;
  int64_t documents = 0;
  if (has(cu)) {
    TORCH_CHECK_VALUE(x.dim() == 3 && x.size(0) == 1 && x.size(1) >= 1, "a packed row has shape (1, T, D) with T >= 1; got ", shape_of(x));
    TORCH_CHECK_VALUE(cu->dim() == 1 && cu->numel() >= 2, "cu_seqlens: a vector of document offsets, at least [0, T]");
    TORCH_CHECK_VALUE(cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong, "cu_seqlens: int32 or int64 offsets, got ", cu->scalar_type());
    TORCH_CHECK_VALUE(cu->is_contiguous() && cu->device() == x.device(), "cu_seqlens: must be contiguous and live on the device of the inputs");
    TORCH_CHECK_VALUE(x.size(1) < (int64_t{1} << 31), "a packed row is limited to 2^31 - 1 tokens (offsets are 32-bit on the device)");
    documents = cu->numel() - 1;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::gated_scan_map", "").typed<decltype(scan_map)>();
    auto [built, valid] = op.call(*cu, x.size(1));
    at::_assert_async(valid, "cu_seqlens must start at 0, end at T, and strictly increase");
    map = built;
  }
  auto [h, final_state, carry] = call_scan_fwd(x, g, initial, map, documents, output_final_state, false);
  return {h, output_final_state ? OptTensor(final_state) : OptTensor()};
}

// One token per sequence on a resident state, which is updated in place.
Tensor scan_decode(const Tensor& x, const Tensor& g, const Tensor& state) {
  TORCH_CHECK_VALUE(!any_grad({&x, &g, &state}), "gated_scan_decode is forward-only: run it under torch.no_grad()");
  at::AutoDispatchBelowADInplaceOrView below;
  const bool squeeze = x.dim() == 3;
  TORCH_CHECK_VALUE((squeeze || x.dim() == 2) && g.sizes() == x.sizes(), "x and g must be (B, 1, D) or (B, D) and agree; got ", shape_of(x), " and ",
                    shape_of(g));
  TORCH_CHECK_VALUE(!squeeze || x.size(1) == 1, "gated_scan_decode takes one token per sequence: T must be 1");
  check_pair(x, g);
  check_place(x, x, "x");
  check_place(g, x, "g");
  const int64_t B = x.size(0), D = x.size(-1);
  TORCH_CHECK_VALUE(state.dim() == 2 && state.size(0) == B && state.size(1) == D && state.scalar_type() == at::kFloat && state.device() == x.device() &&
                        state.is_contiguous(),
                    "state must be a contiguous f32 tensor of shape (", B, ", ", D, ") on x's device");
  TORCH_CHECK_VALUE(B < (int64_t{1} << 31) && D < (int64_t{1} << 31), "gated_scan_decode: an axis is limited to 2^31 - 1 elements");
  check_sm100(x, "gated_scan_decode");
  const c10::cuda::CUDAGuard guard(x.device());
  const SequenceRows xr(squeeze ? x : x.unsqueeze(1)), gr(squeeze ? g : g.unsqueeze(1));
  Tensor h = fresh(x.sizes(), x, x.scalar_type());
  check_rc(tgdn_scan_step(&xr.rows, &gr.rows, static_cast<int>(B), static_cast<int>(D), ptr<float>(state), ptr(h), stream_of(x)), "tgdn_scan_step");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();      // a backward that still needs the state of before says so
  return h;
}

// ---- norms ------------------------------------------------------------------------------------------------------------
// A (..., N) tensor as rows in two levels of strides; what does not fit into two is copied.
struct NormRows {
  Tensor held;
  tgdn_rows rows{nullptr, 1, 0, 0, 0};
  explicit NormRows(const OptTensor& t) {
    if (!has(t)) return;
    held = *t;
    if (!fill()) {
      held = held.contiguous();
      fill();
    }
  }
  bool fill() {
    rows = {held.data_ptr(), 1, 0, 0, type_of(held)};
    if (held.size(-1) != 1 && held.stride(-1) != 1) return false;
    int64_t size[2] = {1, 1}, stride[2] = {0, 0};          // innermost first
    int levels = 0;
    for (int64_t d = held.dim() - 2; d >= 0; --d) {
      if (held.size(d) == 1) continue;
      if (levels > 0 && held.stride(d) == stride[levels - 1] * size[levels - 1]) {
        size[levels - 1] *= held.size(d);
        continue;
      }
      if (levels == 2) return false;
      size[levels] = held.size(d);
      stride[levels++] = held.stride(d);
    }
    rows.inner = size[0];
    rows.stride_inner = stride[0];
    rows.stride_outer = stride[1];
    return true;
  }
};

struct Vector {
  Tensor held;
  tgdn_vector v{nullptr, 0};
  explicit Vector(const OptTensor& t) {
    if (!has(t)) return;
    held = t->contiguous();
    v = {held.data_ptr(), type_of(held)};
  }
};

int64_t rows_of(const Tensor& x) {
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  return rows;
}

void check_vector(const OptTensor& v, const Tensor& x, const char* name) {
  if (!has(v)) return;
  TORCH_CHECK_VALUE(v->dim() == 1 && v->size(0) == x.size(-1) && floating(*v), name, " must be a float32, bfloat16 or float16 vector of the ", x.size(-1),
                    " channels; got ", shape_of(*v), " of ", v->scalar_type());
  check_place(*v, x, name);
}

void check_norm(const Tensor& x, const OptTensor& weight, const OptTensor& scale, const char* call) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && floating(x), call, ": x must be (..., N), float32, bfloat16 or float16; got ", shape_of(x), " of ", x.scalar_type());
  check_place(x, x, "x");
  TORCH_CHECK_VALUE(x.size(-1) <= TGDN_NORM_MAX_CHANNELS && rows_of(x) < (int64_t{1} << 31), call, ": at most ", TGDN_NORM_MAX_CHANNELS,
                    " channels and 2^31 - 1 rows; got ", shape_of(x));
  check_vector(weight, x, "weight");
  check_vector(scale, x, "scale");
  check_sm100(x, call);
}

void check_stream(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == x.sizes() && (t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type()), name,
                    " must have x's shape and be float32 or of x's type; got ", shape_of(t), " of ", t.scalar_type());
  check_place(t, x, name);
}

Tensor scratch_for(const Tensor& x, bool wanted) {
  return wanted ? fresh({tgdn_norm_scratch_floats(rows_of(x), static_cast<int>(x.size(-1)))}, x, at::kFloat) : Tensor();
}

// (y, stream, rstd); the last is empty unless a backward follows.
std::tuple<Tensor, Tensor, Tensor> residual_fwd(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& scale,
                                                double scale_value, double eps, bool save) {
  check_norm(x, weight, scale, "residual_norm");
  check_stream(residual, x, "residual");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = rows_of(x);
  const NormRows xr(x), rr(residual);
  const Vector w(weight), c(scale);
  Tensor y = fresh(x.sizes(), x, x.scalar_type()), stream = fresh(x.sizes(), x, residual.scalar_type()),
         rstd = fresh({save ? rows : 0}, x, at::kFloat);
  check_rc(tgdn_residual_norm_fwd(&xr.rows, &rr.rows, &w.v, &c.v, static_cast<float>(scale_value), rows, static_cast<int>(x.size(-1)),
                                  static_cast<float>(eps), ptr(y), ptr(stream), save ? ptr<float>(rstd) : nullptr, stream_of(x)),
           "tgdn_residual_norm_fwd");
  return {y, stream, rstd};
}

// (dresidual, dx, dweight, dscale).  x: only where dscale is wanted.  dx is empty where it is the same tensor as dresidual: no scale, one type.
std::tuple<Tensor, Tensor, Tensor, Tensor> residual_bwd(const Tensor& stream, const OptTensor& x, at::ScalarType x_type, const OptTensor& dy,
                                                        const OptTensor& dstream, const OptTensor& weight, const OptTensor& scale,
                                                        double scale_value, const Tensor& rstd, bool want_weight, bool want_scale) {
  check_norm(stream, weight, scale, "residual_norm");
  if (has(dy)) TORCH_CHECK_VALUE(dy->sizes() == stream.sizes() && dy->scalar_type() == x_type && dy->device() == stream.device(), "dy must be like x");
  if (has(dstream))
    TORCH_CHECK_VALUE(dstream->sizes() == stream.sizes() && dstream->scalar_type() == stream.scalar_type() && dstream->device() == stream.device(),
                      "dstream must be like the stream");
  TORCH_CHECK_VALUE(!want_weight || has(weight), "no weight to differentiate");
  TORCH_CHECK_VALUE(!want_scale || (has(scale) && has(x) && x->sizes() == stream.sizes() && x->scalar_type() == x_type && x->device() == stream.device()),
                    "the gradient of the scale needs the scale and x");
  const int64_t rows = rows_of(stream);
  TORCH_CHECK_VALUE(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == rows && rstd.device() == stream.device(),
                    "rstd must be what residual_norm_fwd saved");
  const c10::cuda::CUDAGuard guard(stream.device());
  const Tensor st = stream.contiguous();
  const NormRows xr(want_scale ? x : OptTensor()), yr(dy), sr(dstream);
  const Vector w(weight), c(scale);
  const bool same = !has(scale) && scale_value == 1.0 && x_type == stream.scalar_type();
  Tensor dresidual = fresh(stream.sizes(), stream, stream.scalar_type()), dx = same ? none(stream) : fresh(stream.sizes(), stream, x_type);
  Tensor dweight = want_weight ? fresh(weight->sizes(), stream, weight->scalar_type()) : none(stream);
  Tensor dscale = want_scale ? fresh(scale->sizes(), stream, scale->scalar_type()) : none(stream);
  const Vector dw(want_weight ? OptTensor(dweight) : OptTensor()), dc(want_scale ? OptTensor(dscale) : OptTensor());
  const Tensor scratch = scratch_for(stream, want_weight || want_scale);
  const int xt = x_type == at::kFloat ? TGDN_F32 : x_type == at::kBFloat16 ? TGDN_BF16 : x_type == at::kHalf ? TGDN_F16 : -1;
  check_rc(tgdn_residual_norm_bwd(ptr(st), type_of(st), &xr.rows, xt, &yr.rows, &sr.rows, &w.v, &c.v, static_cast<float>(scale_value),
                                  ptr<float>(rstd), rows, static_cast<int>(stream.size(-1)), ptr(dresidual), same ? nullptr : ptr(dx), &dw.v,
                                  &dc.v, ptr<float>(scratch), scratch.defined() ? scratch.numel() : 0, stream_of(stream)),
           "tgdn_residual_norm_bwd");
  return {dresidual, dx, dweight, dscale};
}

// (out, rstd); the last is empty unless a backward follows.
std::tuple<Tensor, Tensor> gated_fwd(const Tensor& x, const OptTensor& gate, const OptTensor& weight, const OptTensor& residual,
                                     const OptTensor& scale, double scale_value, int64_t activation, double eps, bool save) {
  check_norm(x, weight, scale, "gated_norm");
  TORCH_CHECK_VALUE(has(gate) == (activation != TGDN_ACT_NONE), "gated_norm: a gate comes with an activation");
  if (has(gate)) {
    TORCH_CHECK_VALUE(gate->sizes() == x.sizes() && gate->scalar_type() == x.scalar_type(), "gate must have x's shape and type; got ", shape_of(*gate),
                      " of ", gate->scalar_type());
    check_place(*gate, x, "gate");
  }
  if (has(residual)) check_stream(*residual, x, "residual");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = rows_of(x);
  const NormRows xr(x), zr(gate), rr(residual);
  const Vector w(weight), c(scale);
  Tensor out = fresh(x.sizes(), x, has(residual) ? residual->scalar_type() : x.scalar_type()), rstd = fresh({save ? rows : 0}, x, at::kFloat);
  check_rc(tgdn_gated_norm_fwd(&xr.rows, &zr.rows, static_cast<int>(activation), &w.v, &rr.rows, &c.v, static_cast<float>(scale_value), rows,
                               static_cast<int>(x.size(-1)), static_cast<float>(eps), ptr(out), type_of(out), save ? ptr<float>(rstd) : nullptr, stream_of(x)),
           "tgdn_gated_norm_fwd");
  return {out, rstd};
}

// (dx, dgate, dweight, dscale); what is not there or not wanted is empty.
std::tuple<Tensor, Tensor, Tensor, Tensor> gated_bwd(const Tensor& x, const OptTensor& gate, const Tensor& dout, const OptTensor& weight,
                                                     const OptTensor& scale, double scale_value, int64_t activation, const Tensor& rstd,
                                                     bool want_weight, bool want_scale) {
  check_norm(x, weight, scale, "gated_norm");
  TORCH_CHECK_VALUE(has(gate) == (activation != TGDN_ACT_NONE), "gated_norm: a gate comes with an activation");
  if (has(gate))
    TORCH_CHECK_VALUE(gate->sizes() == x.sizes() && gate->scalar_type() == x.scalar_type() && gate->device() == x.device(), "gate must be like x");
  check_stream(dout, x, "dout");
  TORCH_CHECK_VALUE((!want_weight || has(weight)) && (!want_scale || has(scale)), "no such vector to differentiate");
  const int64_t rows = rows_of(x);
  TORCH_CHECK_VALUE(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == rows && rstd.device() == x.device(),
                    "rstd must be what gated_norm_fwd saved");
  const c10::cuda::CUDAGuard guard(x.device());
  const NormRows xr(x), zr(gate), yr(dout);
  const Vector w(weight), c(scale);
  Tensor dx = fresh(x.sizes(), x, x.scalar_type()), dgate = has(gate) ? fresh(x.sizes(), x, x.scalar_type()) : none(x);
  Tensor dweight = want_weight ? fresh(weight->sizes(), x, weight->scalar_type()) : none(x);
  Tensor dscale = want_scale ? fresh(scale->sizes(), x, scale->scalar_type()) : none(x);
  const Vector dw(want_weight ? OptTensor(dweight) : OptTensor()), dc(want_scale ? OptTensor(dscale) : OptTensor());
  const Tensor scratch = scratch_for(x, want_weight || want_scale);
  check_rc(tgdn_gated_norm_bwd(&xr.rows, &zr.rows, static_cast<int>(activation), &yr.rows, &w.v, &c.v, static_cast<float>(scale_value),
                               ptr<float>(rstd), rows, static_cast<int>(x.size(-1)), ptr(dx), has(gate) ? ptr(dgate) : nullptr, &dw.v, &dc.v,
                               ptr<float>(scratch), scratch.defined() ? scratch.numel() : 0, stream_of(x)),
           "tgdn_gated_norm_bwd");
  return {dx, dgate, dweight, dscale};
}

using Three = std::tuple<Tensor, Tensor, Tensor>;
using Two = std::tuple<Tensor, Tensor>;
Three call_residual_fwd(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& scale, double scale_value, double eps,
                        bool save) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::residual_norm_fwd", "").typed<decltype(residual_fwd)>();
  return op.call(x, residual, weight, scale, scale_value, eps, save);
}
Two call_gated_fwd(const Tensor& x, const OptTensor& gate, const OptTensor& weight, const OptTensor& residual, const OptTensor& scale,
                   double scale_value, int64_t activation, double eps, bool save) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::gated_norm_fwd", "").typed<decltype(gated_fwd)>();
  return op.call(x, gate, weight, residual, scale, scale_value, activation, eps, save);
}

bool wants_grad(const OptTensor& t) { return has(t) && at::GradMode::is_enabled() && t->requires_grad(); }

struct ResidualSteps {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& scale,
                               double scale_value, double eps, bool want_weight, bool want_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, stream, rstd] = call_residual_fwd(x, residual, weight, scale, scale_value, eps, true);
    ctx->save_for_backward({stream, rstd, or_undefined(weight), or_undefined(scale), want_scale ? x : Tensor()});
    ctx->saved_data["value"] = scale_value;
    ctx->saved_data["type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["want_weight"] = want_weight;
    ctx->saved_data["want_scale"] = want_scale;
    ctx->mark_non_differentiable({rstd});
    ctx->set_materialize_grads(false);
    return {y, stream, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(8);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    variable_list s = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::residual_norm_bwd", "").typed<decltype(residual_bwd)>();
    const bool want_weight = ctx->saved_data["want_weight"].toBool(), want_scale = ctx->saved_data["want_scale"].toBool();
    const double value = ctx->saved_data["value"].toDouble();
    const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    auto [dresidual, dx, dweight, dscale] = op.call(s[0], or_nullopt(s[4]), x_type, or_nullopt(grads[0]), or_nullopt(grads[1]), or_nullopt(s[2]),
                                                    or_nullopt(s[3]), value, s[1], want_weight, want_scale);
    res[0] = !s[3].defined() && value == 1.0 && x_type == s[0].scalar_type() ? dresidual : dx;
    res[1] = dresidual;
    if (want_weight) res[2] = dweight;
    if (want_scale) res[3] = dscale;
    return res;
  }
};
using ResidualFunction = Differentiable<ResidualSteps>;

Three residual_fwd_autograd(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& scale, double scale_value, double eps,
                            bool save) {
  if (!any_grad({&x, &residual}) && !wants_grad(weight) && !wants_grad(scale)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_residual_fwd(x, residual, weight, scale, scale_value, eps, save);
  }
  variable_list o = ResidualFunction::apply(x, residual, weight, scale, scale_value, eps, wants_grad(weight), wants_grad(scale));
  return {o[0], o[1], o[2]};
}

struct GatedSteps {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gate, const OptTensor& weight, const OptTensor& residual,
                               const OptTensor& scale, double scale_value, int64_t activation, double eps, bool want_weight, bool want_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, rstd] = call_gated_fwd(x, gate, weight, residual, scale, scale_value, activation, eps, true);
    ctx->save_for_backward({x, rstd, or_undefined(gate), or_undefined(weight), or_undefined(scale)});
    ctx->saved_data["value"] = scale_value;
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["residual"] = has(residual);
    ctx->saved_data["want_weight"] = want_weight;
    ctx->saved_data["want_scale"] = want_scale;
    ctx->mark_non_differentiable({rstd});
    ctx->set_materialize_grads(false);
    return {out, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(10);
    if (!grads[0].defined()) return res;
    variable_list s = ctx->get_saved_variables();
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("tgdn_b200::gated_norm_bwd", "").typed<decltype(gated_bwd)>();
    const bool want_weight = ctx->saved_data["want_weight"].toBool(), want_scale = ctx->saved_data["want_scale"].toBool();
    auto [dx, dgate, dweight, dscale] = op.call(s[0], or_nullopt(s[2]), grads[0], or_nullopt(s[3]), or_nullopt(s[4]), ctx->saved_data["value"].toDouble(),
                                                ctx->saved_data["activation"].toInt(), s[1], want_weight, want_scale);
    res[0] = dx;
    if (s[2].defined()) res[1] = dgate;
    if (want_weight) res[2] = dweight;
    if (ctx->saved_data["residual"].toBool()) res[3] = grads[0];
    if (want_scale) res[4] = dscale;
    return res;
  }
};
using GatedFunction = Differentiable<GatedSteps>;

Two gated_fwd_autograd(const Tensor& x, const OptTensor& gate, const OptTensor& weight, const OptTensor& residual, const OptTensor& scale,
                       double scale_value, int64_t activation, double eps, bool save) {
  if (!any_grad({&x}) && !wants_grad(gate) && !wants_grad(weight) && !wants_grad(residual) && !wants_grad(scale)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_gated_fwd(x, gate, weight, residual, scale, scale_value, activation, eps, save);
  }
  variable_list o = GatedFunction::apply(x, gate, weight, residual, scale, scale_value, activation, eps, wants_grad(weight), wants_grad(scale));
  return {o[0], o[1]};
}

Two residual_call(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& scale, double scale_value, double eps) {
  auto [y, stream, rstd] = call_residual_fwd(x, residual, weight, scale, scale_value, eps, false);
  return {y, stream};
}

Tensor gated_call(const Tensor& x, const OptTensor& gate, const OptTensor& weight, const OptTensor& residual, const OptTensor& scale,
                  double scale_value, int64_t activation, double eps) {
  return std::get<0>(call_gated_fwd(x, gate, weight, residual, scale, scale_value, activation, eps, false));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tgdn_b200, m) {
  m.def("gated_scan_map(Tensor cu_seqlens, SymInt tokens) -> (Tensor, Tensor)");
  m.def("gated_scan_fwd(Tensor x, Tensor g, Tensor? initial_state=None, Tensor? doc_map=None, SymInt documents=0, bool output_final_state=False, "
        "bool save=False) -> (Tensor, Tensor, Tensor)");
  m.def("gated_scan_bwd(Tensor x, Tensor g, Tensor dh, Tensor carry, Tensor? initial_state=None, Tensor? doc_map=None, SymInt documents=0, "
        "Tensor? dfinal=None) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm_fwd(Tensor x, Tensor residual, Tensor? weight, Tensor? scale, float scale_value, float eps, "
        "bool save=False) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm_bwd(Tensor stream, Tensor? x, ScalarType x_type, Tensor? dy, Tensor? dstream, Tensor? weight, Tensor? scale, "
        "float scale_value, Tensor rstd, bool want_weight, bool want_scale) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_norm_fwd(Tensor x, Tensor? gate, Tensor? weight, Tensor? residual, Tensor? scale, float scale_value, int activation, float eps, "
        "bool save=False) -> (Tensor, Tensor)");
  m.def("gated_norm_bwd(Tensor x, Tensor? gate, Tensor dout, Tensor? weight, Tensor? scale, float scale_value, int activation, Tensor rstd, "
        "bool want_weight, bool want_scale) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(tgdn_b200, CUDA, m) {
  m.impl("gated_scan_map", TORCH_FN(scan_map));
  m.impl("gated_scan_fwd", TORCH_FN(scan_fwd));
  m.impl("gated_scan_bwd", TORCH_FN(scan_bwd));
  m.impl("residual_norm_fwd", TORCH_FN(residual_fwd));
  m.impl("residual_norm_bwd", TORCH_FN(residual_bwd));
  m.impl("gated_norm_fwd", TORCH_FN(gated_fwd));
  m.impl("gated_norm_bwd", TORCH_FN(gated_bwd));
}

TORCH_LIBRARY_IMPL(tgdn_b200, Autograd, m) {
  m.impl("gated_scan_fwd", TORCH_FN(scan_fwd_autograd));
  m.impl("residual_norm_fwd", TORCH_FN(residual_fwd_autograd));
  m.impl("gated_norm_fwd", TORCH_FN(gated_fwd_autograd));
  m.impl("gated_scan_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("residual_norm_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("gated_norm_bwd", torch::autograd::autogradNotImplementedFallback());
}

void tgdn_torch::bind_block_operators(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> nogil;
  m.def("scan_call", &scan_call, nogil);
  m.def("scan_decode", &scan_decode, nogil);
  m.def("residual_norm", &residual_call, nogil);
  m.def("gated_norm", &gated_call, nogil);
}
