// Torch wrappers of the gated recurrent block's kernels: gated linear recurrence, norms
// around a block, 8-bit activations.
#include "host_common.h"
#include "recurrence.h"

using namespace su;

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool is_float_type(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Numbers go into messages as text: an integer put into the stream of TORCH_CHECK crashes
// where the interpreter brings a C++ library of its own.
std::string str(int64_t v) { return std::to_string(v); }
std::string str(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

// (of a tensor without values any stride will do: torch gives such tensors any)
bool unit_last(const at::Tensor& t) { return t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1; }

// rows that start on multiples of n values: base and strides of a tensor with unit last stride
bool rows_of(int n, const at::Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % (n * t.element_size()) != 0) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) % n != 0) return false;
  return t.size(-1) % n == 0;
}
bool rows_of_four(const at::Tensor& t) { return rows_of(4, t); }
// 4, 2 or 1: values that rows of t, and of vectors `width` wide, start on multiples of
int row_unit(const at::Tensor& t, int64_t width) {
  for (int n : {4, 2})
    if (width % n == 0 && rows_of(n, t)) return n;
  return 1;
}

void check_param(const at::Tensor& t, const char* name, int64_t width, const at::Device& dev) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(is_float_type(t), name, " must be float32 or bfloat16");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == width && t.is_contiguous(), name, " must be a contiguous vector of ",
              str(width));
}

void check_rows(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must be ", like.scalar_type());
  TORCH_CHECK(t.sizes() == like.sizes(), name, " must have the shape ", str(like.sizes()), ", got ", str(t.sizes()));
  TORCH_CHECK(unit_last(t), name, " must have unit stride along its last dimension");
}

// a rate or eps that kernels hold in fp32
float positive(double v, const char* name) {
  const float f = static_cast<float>(v);
  TORCH_CHECK(f > 0 && std::isfinite(f), name, " must be positive and finite in float32");
  return f;
}

struct ScanSizes {
  bool packed;
  int64_t batch, steps, width;
};
ScanSizes scan_sizes(at::IntArrayRef shape, const OptTensor& offsets, int64_t per_row) {
  ScanSizes s;
  s.packed = given(offsets);
  TORCH_CHECK(static_cast<int64_t>(shape.size()) == (s.packed ? 2 : 3),
              "gated_scan: p must be [batch, steps, 3H], or [rows, 3H] with offsets");
  TORCH_CHECK(shape.back() > 0 && shape.back() % per_row == 0, "gated_scan: the last dimension of p must be 3H, H > 0");
  s.width = shape.back() / per_row;
  TORCH_CHECK(s.width <= (1 << 18), "gated_scan: H above 2^18");
  s.steps = s.packed ? shape[0] : shape[1];
  if (s.packed) TORCH_CHECK(offsets->dim() == 1, "gated_scan: offsets must be a vector of sequences + 1");
  s.batch = s.packed ? offsets->size(0) - 1 : shape[0];
  // (the offsets' values are checked on the device, in a kernel over the sequences)
  TORCH_CHECK(!s.packed || s.batch != 0 || s.steps == 0, "gated_scan: offsets must rise from 0 to the number of rows, ",
              "but there are rows and no sequence");
  return s;
}

// what forward and backward share: sequences, mask, decay, first states, layout of the dense rows
ScanArgs scan_args(const ScanSizes& z, const at::Tensor& decay, const OptTensor& h0, const OptTensor& mask,
                   const OptTensor& offsets, double rate, bool time_major, bool codes, const at::Device& dev) {
  ScanArgs a;
  a.batch = z.batch;
  a.steps = z.steps;
  a.width = static_cast<int>(z.width);
  a.rate = positive(rate, "gated_scan: rate");
  check_param(decay, "gated_scan: decay", z.width, dev);
  a.decay = decay.data_ptr();
  a.decay_bf16 = decay.scalar_type() == at::kBFloat16;
  if (given(h0)) {
    TORCH_CHECK(h0->device() == dev && h0->scalar_type() == at::kFloat && h0->is_contiguous(),
                "gated_scan: h0 must be contiguous float32 on ", dev);
    TORCH_CHECK(h0->dim() == 2 && h0->size(0) == z.batch && h0->size(1) == z.width, "gated_scan: h0 must be [",
                str(z.batch), ", ", str(z.width), "]");
    a.h0 = h0->data_ptr<float>();
  }
  if (z.packed) {
    TORCH_CHECK(offsets->device() == dev && offsets->scalar_type() == at::kLong && offsets->dim() == 1 &&
                    offsets->size(0) >= 1 && offsets->is_contiguous(),
                "gated_scan: offsets must be a contiguous int64 vector of sequences + 1 on ", dev);
    a.offsets = offsets->data_ptr<int64_t>();
  }
  if (given(mask)) {
    TORCH_CHECK(mask->device() == dev && mask->scalar_type() == at::kBool, "gated_scan: mask must be bool on ", dev);
    const bool fits = z.packed ? mask->dim() == 1 && mask->size(0) == z.steps
                               : mask->dim() == 2 && mask->size(0) == z.batch && mask->size(1) == z.steps;
    TORCH_CHECK(fits, "gated_scan: mask must have the shape of p without its last dimension");
    a.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr<bool>());
    a.m_sb = z.packed ? 0 : mask->stride(0);
    a.m_st = mask->stride(z.packed ? 0 : 1);
  }
  a.row_sb = z.packed ? 0 : (time_major ? 1 : z.steps);
  a.row_st = z.packed ? 1 : (time_major ? z.batch : 1);
  a.state_every = codes ? kStateEvery : kStateShort;
  a.n_states = z.steps > 0 ? (z.steps - 1) / a.state_every : 0;
  a.status = device_status_ptr(dev.index());
  return a;
}

// [batch, steps, width] (packed: [rows, width]) over dense rows in the order of the layout
at::Tensor dense_rows(const ScanSizes& z, int64_t width, bool time_major, const at::TensorOptions& o) {
  if (z.packed) return at::empty({z.steps, width}, o);
  if (time_major) return at::empty({z.steps, z.batch, width}, o).transpose(0, 1);
  return at::empty({z.batch, z.steps, width}, o);
}

// stream-ordered, as every temporary here: the caching allocator reuses it after the call
at::Tensor scan_workspace_of(const ScanArgs& a, int sms, const at::TensorOptions& o) {
  const size_t bytes = scan_workspace(a, sms);
  return bytes == 0 ? at::Tensor() : at::empty({static_cast<int64_t>(bytes)}, o.dtype(at::kByte));
}

int64_t groups_of(int64_t width) { return (width + kGroup8 - 1) / kGroup8; }

}  // namespace

// -> h, last state, kept states, codes, scales (those three undefined where not kept), marks of
// packed sequences
static std::vector<at::Tensor> gated_scan_fwd(const at::Tensor& p, const at::Tensor& decay, const OptTensor& h0,
                                       const OptTensor& mask, const OptTensor& offsets, double rate, bool time_major,
                                       bool keep_states, bool keep8) {
  SU_CHECK_CUDA(p);
  TORCH_CHECK(is_float_type(p), "gated_scan: p must be float32 or bfloat16");
  const ScanSizes z = scan_sizes(p.sizes(), offsets, 3);
  TORCH_CHECK(unit_last(p), "gated_scan: p must have unit stride along its last dimension");
  c10::cuda::CUDAGuard guard(p.device());
  ScanArgs a = scan_args(z, decay, h0, mask, offsets, rate, time_major, keep8, p.device());
  a.bf16 = p.scalar_type() == at::kBFloat16;
  a.p = p.data_ptr();
  a.p_sb = z.packed ? 0 : p.stride(0);
  a.p_st = p.stride(z.packed ? 0 : 1);
  a.vec = row_unit(p, z.width);
  const auto f32 = p.options().dtype(at::kFloat);
  at::Tensor h = dense_rows(z, z.width, time_major, p.options());
  at::Tensor last = at::empty({z.batch, z.width}, f32);
  at::Tensor states, codes, scales, marks;
  a.h = h.data_ptr();
  a.last = last.data_ptr<float>();
  if (keep_states) {
    states = at::empty({z.packed ? 1 : z.batch, a.n_states, z.width}, f32);
    if (a.n_states > 0) a.states = states.data_ptr<float>();
  }
  if (keep8) {
    codes = dense_rows(z, 3 * z.width, time_major, p.options().dtype(at::kChar));
    scales = dense_rows(z, 3 * groups_of(z.width), time_major, f32);
    a.codes = codes.data_ptr<int8_t>();
    a.scales = scales.data_ptr<float>();
  }
  if (z.packed) {
    TORCH_CHECK(z.batch < (1ll << 29), "gated_scan: 2^29 sequences or more");
    marks = at::empty({z.steps}, p.options().dtype(at::kInt));
    a.marks = marks.data_ptr<int>();
  }
  if (z.batch > 0) {
    const int sms = num_sms(p.get_device());
    at::Tensor work = scan_workspace_of(a, sms, p.options());
    launch_scan_fwd(a, sms, work.defined() ? work.data_ptr() : nullptr, cur_stream());
    SU_LAUNCH_CHECK();
  }
  return {h, last, states, codes, scales, marks};
}

// `like`: p, or its 8-bit codes with `scales` (then the gradients have the type of h, `bf16`)
// -> dp, ddecay, dh0
static std::vector<at::Tensor> gated_scan_bwd(const at::Tensor& like, const OptTensor& scales, const at::Tensor& states,
                                       const at::Tensor& decay, const OptTensor& h0, const OptTensor& mask,
                                       const OptTensor& offsets, const OptTensor& marks, const OptTensor& dh,
                                       const OptTensor& dlast, double rate, bool time_major, bool bf16, bool need_dh0) {
  SU_CHECK_CUDA(like);
  const ScanSizes z = scan_sizes(like.sizes(), offsets, 3);
  const auto dev = like.device();
  c10::cuda::CUDAGuard guard(dev);
  ScanArgs a = scan_args(z, decay, h0, mask, offsets, rate, time_major, given(scales), dev);
  const auto f32 = like.options().dtype(at::kFloat);
  const auto type = bf16 ? at::kBFloat16 : at::kFloat;
  a.bf16 = bf16;
  a.vec = z.width % 4 == 0 ? 4 : z.width % 2 == 0 ? 2 : 1;
  if (given(scales)) {
    TORCH_CHECK(like.scalar_type() == at::kChar, "gated_scan: 8-bit codes must be int8");
    TORCH_CHECK(scales->device() == dev && scales->numel() == like.numel() / (3 * z.width) * 3 * groups_of(z.width),
                "gated_scan: scales do not fit the 8-bit codes");
    a.codes = like.data_ptr<int8_t>();
    a.scales = scales->data_ptr<float>();
  } else {
    TORCH_CHECK(like.scalar_type() == type, "gated_scan: p must have the type of h");
    TORCH_CHECK(unit_last(like), "gated_scan: p must have unit stride along its last dimension");
    a.p = like.data_ptr();
    a.p_sb = z.packed ? 0 : like.stride(0);
    a.p_st = like.stride(z.packed ? 0 : 1);
    a.vec = std::min(a.vec, row_unit(like, z.width));
  }
  TORCH_CHECK(states.device() == dev && states.is_contiguous() &&
                  states.numel() == (z.packed ? 1 : z.batch) * a.n_states * z.width,
              "gated_scan: kept states do not fit");
  a.states = const_cast<float*>(states.data_ptr<float>());
  if (z.packed) {
    TORCH_CHECK(given(marks) && marks->device() == dev && marks->is_contiguous() && marks->numel() == z.steps,
                "gated_scan: packed sequences need the forward's marks");
    a.marks = marks->data_ptr<int>();
  }
  if (given(dh)) {
    TORCH_CHECK(dh->device() == dev && dh->scalar_type() == type && dh->dim() == like.dim() &&
                    dh->sizes().slice(0, like.dim() - 1) == like.sizes().slice(0, like.dim() - 1) &&
                    dh->size(-1) == z.width && unit_last(*dh),
                "gated_scan: the gradient of h must have its type, shape and unit last stride");
    a.dh = dh->data_ptr();
    a.dh_sb = z.packed ? 0 : dh->stride(0);
    a.dh_st = dh->stride(z.packed ? 0 : 1);
    a.vec = std::min(a.vec, row_unit(*dh, z.width));
  }
  if (given(dlast)) {
    TORCH_CHECK(dlast->device() == dev && dlast->scalar_type() == at::kFloat && dlast->is_contiguous() &&
                    dlast->numel() == z.batch * z.width,
                "gated_scan: the gradient of the last state must be contiguous float32");
    a.dlast = dlast->data_ptr<float>();
  }
  at::Tensor dp = dense_rows(z, 3 * z.width, time_major, like.options().dtype(type));
  at::Tensor ddecay = at::empty_like(decay);
  at::Tensor dh0 = need_dh0 ? at::empty({z.batch, z.width}, f32) : at::Tensor();
  a.dp = dp.data_ptr();
  a.dh0 = need_dh0 ? dh0.data_ptr<float>() : nullptr;
  if (z.batch == 0) {
    ddecay.zero_();
    return {dp, ddecay, dh0};
  }
  const int sms = num_sms(like.get_device());
  at::Tensor partial = at::empty({scan_partials(a, sms), z.width}, f32);
  a.partial = partial.data_ptr<float>();
  at::Tensor work = scan_workspace_of(a, sms, like.options());
  launch_scan_bwd(a, sms, work.defined() ? work.data_ptr() : nullptr, ddecay.data_ptr(), cur_stream());
  SU_LAUNCH_CHECK();
  return {dp, ddecay, dh0};
}

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A tensor that saved-tensor hooks leave alone: its bits as int32 (hooks that compress
// activations take floating tensors).
at::Tensor hidden(const at::Tensor& t) { return t.defined() ? t.view(at::kInt) : t; }
at::Tensor shown(const at::Tensor& t) { return t.defined() ? t.view(at::kFloat) : t; }
OptTensor maybe(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
at::Tensor value(const OptTensor& t) { return given(t) ? *t : at::Tensor(); }

// What was saved comes back from a user's saved-tensor hooks with its values, but in any layout (pinned
// copies on the host are contiguous).
at::Tensor plain(const at::Tensor& t) { return t.defined() ? t.contiguous() : t; }
// dense rows in the order of the layout (see dense_rows)
at::Tensor dense(const at::Tensor& t, bool time_major) {
  return time_major && t.defined() ? t.transpose(0, 1).contiguous().transpose(0, 1) : plain(t);
}

void check_once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": its gradient cannot be differentiated again (create_graph)");
}

struct GatedScan : public torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& p, const at::Tensor& decay,
                               const OptTensor& h0, const OptTensor& mask, const OptTensor& offsets, double rate,
                               bool time_major, bool keep8) {
    auto out = gated_scan_fwd(p, decay, h0, mask, offsets, rate, time_major, true, keep8);
    ctx->save_for_backward({keep8 ? out[3] : p, hidden(out[4]), hidden(out[2]), decay, hidden(value(h0)), value(mask),
                            value(offsets), out[5]});
    ctx->saved_data["rate"] = rate;
    ctx->saved_data["time_major"] = time_major;
    ctx->saved_data["bf16"] = p.scalar_type() == at::kBFloat16;
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_scan");
    const auto v = ctx->get_saved_variables();
    at::Tensor dh = grads[0], dlast = grads[1];
    if (dh.defined() && !unit_last(dh)) dh = dh.contiguous();
    dlast = plain(dlast);
    const bool time_major = ctx->saved_data["time_major"].toBool();
    const bool keep8 = v[1].defined();
    const at::Tensor in = keep8 ? dense(v[0], time_major) : unit_last(v[0]) ? v[0] : v[0].contiguous();
    auto g = gated_scan_bwd(in, maybe(shown(dense(v[1], time_major))), shown(plain(v[2])), plain(v[3]),
                            maybe(shown(plain(v[4]))), maybe(v[5]), maybe(plain(v[6])), maybe(plain(v[7])), maybe(dh),
                            maybe(dlast), ctx->saved_data["rate"].toDouble(), time_major,
                            ctx->saved_data["bf16"].toBool(),
                            v[4].defined() && ctx->needs_input_grad(2));  // p, decay, h0: the tensors given
    return {g[0], g[1], g[2], {}, {}, {}, {}, {}};
  }
};

// Nothing here carries a tangent on: refused, as a second derivative is.
void check_no_tangent(const char* name, std::initializer_list<at::Tensor> ts) {
  for (const auto& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name,
                ": forward-mode differentiation is not supported on CUDA");
}

bool wants_grad(std::initializer_list<at::Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

}  // namespace

// The op as the Python package calls it: layout of the dense rows, autograd.
std::tuple<at::Tensor, at::Tensor> gated_scan(const at::Tensor& p_in, const at::Tensor& decay_in,
                                              const OptTensor& h0_in, const OptTensor& mask, const OptTensor& offsets,
                                              double rate, bool keep8) {
  scan_sizes(p_in.sizes(), offsets, 3);
  const at::Tensor p = unit_last(p_in) ? p_in : p_in.contiguous();
  const at::Tensor decay = decay_in.contiguous();
  const at::Tensor h0 = given(h0_in) ? h0_in->to(at::kFloat).contiguous() : at::Tensor();
  const bool time_major = !given(offsets) && p.stride(1) > p.stride(0);
  check_no_tangent("gated_scan", {p, decay, h0});
  if (wants_grad({p, decay, h0})) {
    auto out = GatedScan::apply(p, decay, maybe(h0), mask, offsets, rate, time_major, keep8);
    return {out[0], out[1]};
  }
  auto out = gated_scan_fwd(p, decay, maybe(h0), mask, offsets, rate, time_major, false, false);
  return {out[0], out[1]};
}

at::Tensor gated_scan_step(const at::Tensor& p_in, const at::Tensor& decay, at::Tensor& state, const OptTensor& rows,
                           double rate) {
  SU_CHECK_CUDA(p_in);
  const at::Tensor p = unit_last(p_in) ? p_in : p_in.detach().contiguous();
  TORCH_CHECK(is_float_type(p), "gated_scan_step: p must be float32 or bfloat16");
  TORCH_CHECK(p.dim() == 2 && p.size(1) > 0 && p.size(1) % 3 == 0 && unit_last(p),
              "gated_scan_step: p must be [rows, 3H] with unit stride along its last dimension");
  const int64_t n = p.size(0), H = p.size(1) / 3;
  TORCH_CHECK(H <= (1 << 18), "gated_scan_step: H above 2^18");
  const float rate32 = positive(rate, "gated_scan_step: rate");
  c10::cuda::CUDAGuard guard(p.device());
  check_param(decay, "gated_scan_step: decay", H, p.device());
  TORCH_CHECK(state.device() == p.device() && state.scalar_type() == at::kFloat && state.dim() == 2 &&
                  state.size(1) == H && unit_last(state),
              "gated_scan_step: state must be float32 [table rows, ", str(H), "] on ", p.device());
  TORCH_CHECK(state.size(0) <= 1 || state.stride(0) >= H, "gated_scan_step: the rows of state must not overlap");
  ScanStepArgs a;
  if (given(rows)) {
    TORCH_CHECK(rows->device() == p.device() && rows->scalar_type() == at::kLong && rows->dim() == 1 &&
                    rows->size(0) == n && rows->is_contiguous(),
                "gated_scan_step: rows must be a contiguous int64 vector, one place per row of p");
    a.index = rows->data_ptr<int64_t>();
  } else {
    TORCH_CHECK(state.size(0) == n, "gated_scan_step: without rows, state must have one row per row of p");
  }
  at::Tensor h = at::empty({n, H}, p.options());
  if (n == 0) return h;
  a.bf16 = p.scalar_type() == at::kBFloat16;
  // four channels a thread once single ones would fill the SMs: 70,915 x 260 bf16 61 us against
  // 121, and 600 x 100 fp32 2.6 against 2.2, where one thread's four gates take longer
  const bool many = n * H > static_cast<int64_t>(num_sms(p.get_device())) * 2048;
  a.vec = many && H % 4 == 0 && rows_of_four(p) && rows_of_four(state) ? 4 : 1;
  a.rows = n;
  a.table_rows = state.size(0);
  a.width = static_cast<int>(H);
  a.rate = rate32;
  a.p = p.data_ptr();
  a.p_sb = p.stride(0);
  a.decay = decay.data_ptr();
  a.decay_bf16 = decay.scalar_type() == at::kBFloat16;
  a.state = state.data_ptr<float>();
  a.state_sb = state.stride(0);
  a.h = h.data_ptr();
  a.status = device_status_ptr(p.get_device());
  // autograd refuses a backward pass over a table that it saved and this overwrites (tensors of
  // inference mode are never saved, and have no version)
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  launch_scan_step(a, cur_stream());
  SU_LAUNCH_CHECK();
  return h;
}

namespace {

NormArgs norm_args(const at::Tensor& x, int64_t width, const OptTensor& w_post, const OptTensor& w_pre,
                   const OptTensor& scale, double eps) {
  TORCH_CHECK(width >= 1 && width <= kNormMaxWidth, "norm_residual: the width must be 1 to ", str(kNormMaxWidth));
  NormArgs a;
  a.width = static_cast<int>(width);
  a.eps = positive(eps, "norm_residual: eps");
  auto param = [&](const OptTensor& t, const char* name, const void*& ptr, int& bf16) {
    if (!given(t)) return;
    check_param(*t, name, width, x.device());
    ptr = t->data_ptr();
    bf16 = t->scalar_type() == at::kBFloat16;
  };
  param(w_post, "norm_residual: w_post", a.w_post, a.post_bf16);
  param(w_pre, "norm_residual: w_pre", a.w_pre, a.pre_bf16);
  param(scale, "norm_residual: scale", a.scale, a.scale_bf16);
  return a;
}

}  // namespace

// x, u, gate [rows, H] -> y (undefined without u), n (undefined without w_pre), codes, scales
static std::vector<at::Tensor> norm_residual_fwd(const at::Tensor& x, const OptTensor& u, const OptTensor& gate,
                                          const OptTensor& w_post, const OptTensor& w_pre, const OptTensor& scale,
                                          double eps, bool keep8) {
  SU_CHECK_CUDA(x);
  TORCH_CHECK(is_float_type(x) && x.dim() == 2, "norm_residual: x must be float32 or bfloat16 rows");
  TORCH_CHECK(unit_last(x), "norm_residual: x must have unit stride along its last dimension");
  c10::cuda::CUDAGuard guard(x.device());
  NormArgs a = norm_args(x, x.size(1), w_post, w_pre, scale, eps);
  a.bf16 = x.scalar_type() == at::kBFloat16;
  a.rows = x.size(0);
  a.x = x.data_ptr();
  a.x_ld = x.stride(0);
  a.vec = rows_of_four(x);
  a.vec8 = rows_of(8, x);
  int64_t parts = 1;
  if (given(u)) {
    check_rows(*u, "norm_residual: u", x);
    a.u = u->data_ptr();
    a.u_ld = u->stride(0);
    a.vec = a.vec && rows_of_four(*u);
    a.vec8 = a.vec8 && rows_of(8, *u);
    ++parts;
  }
  if (given(gate)) {
    TORCH_CHECK(given(u), "norm_residual: a gate needs u");
    check_rows(*gate, "norm_residual: gate", x);
    a.gate = gate->data_ptr();
    a.gate_ld = gate->stride(0);
    a.vec = a.vec && rows_of_four(*gate);
    a.vec8 = a.vec8 && rows_of(8, *gate);
    ++parts;
  }
  const int64_t H = a.width;
  at::Tensor y, n, codes, scales;
  // (an empty tensor's address is null: what takes part goes by the arguments)
  if (given(u)) {
    y = at::empty({a.rows, H}, x.options());
    a.y = y.data_ptr();
  }
  if (given(w_pre)) {
    n = at::empty({a.rows, H}, x.options());
    a.n = n.data_ptr();
  }
  if (keep8) {
    codes = at::empty({parts, a.rows, H}, x.options().dtype(at::kChar));
    scales = at::empty({parts, a.rows, groups_of(H)}, x.options().dtype(at::kFloat));
    a.codes = codes.data_ptr<int8_t>();
    a.scales = scales.data_ptr<float>();
  }
  if (a.rows > 0) {
    launch_norm_fwd(a, num_sms(x.get_device()), cur_stream());
    SU_LAUNCH_CHECK();
  }
  return {y, n, codes, scales};
}

// x, u, gate: the forward's rows, or (keep8) undefined u and gate with x = codes and `scales`
// -> dx, du, dgate, dw_post, dw_pre, dscale (undefined where there is nothing to differentiate)
static std::vector<at::Tensor> norm_residual_bwd(const at::Tensor& x, const OptTensor& u, const OptTensor& gate,
                                          const OptTensor& scales, const OptTensor& w_post, const OptTensor& w_pre,
                                          const OptTensor& scale, double eps, const OptTensor& dy, const OptTensor& dn,
                                          bool bf16) {
  SU_CHECK_CUDA(x);
  c10::cuda::CUDAGuard guard(x.device());
  NormArgs a = norm_args(x, x.size(-1), w_post, w_pre, scale, eps);
  const int64_t H = a.width;
  const auto type = bf16 ? at::kBFloat16 : at::kFloat;
  const auto opt = x.options().dtype(type);
  a.bf16 = bf16;
  a.rows = x.size(-2);
  a.vec = H % 4 == 0;
  a.vec8 = H % 8 == 0;
  bool has_u, has_gate;
  if (given(scales)) {
    TORCH_CHECK(x.scalar_type() == at::kChar && x.dim() == 3 && x.is_contiguous() && scales->device() == x.device() &&
                    scales->is_contiguous() && scales->numel() == x.size(0) * x.size(1) * groups_of(H),
                "norm_residual: malformed 8-bit inputs");
    a.codes = x.data_ptr<int8_t>();
    a.scales = scales->data_ptr<float>();
    a.x = x.data_ptr();
    has_u = x.size(0) > 1;
    has_gate = x.size(0) > 2;
    if (has_u) a.u = a.x;  // only whether they exist is read
    if (has_gate) a.gate = a.x;
  } else {
    TORCH_CHECK(x.scalar_type() == type && x.dim() == 2 && unit_last(x), "norm_residual: x must have the type of y");
    a.x = x.data_ptr();
    a.x_ld = x.stride(0);
    a.vec = a.vec && rows_of_four(x);
    a.vec8 = a.vec8 && rows_of(8, x);
    has_u = given(u);
    has_gate = given(gate);
    if (has_u) {
      check_rows(*u, "norm_residual: u", x);
      a.u = u->data_ptr();
      a.u_ld = u->stride(0);
      a.vec = a.vec && rows_of_four(*u);
      a.vec8 = a.vec8 && rows_of(8, *u);
    }
    if (has_gate) {
      check_rows(*gate, "norm_residual: gate", x);
      a.gate = gate->data_ptr();
      a.gate_ld = gate->stride(0);
      a.vec = a.vec && rows_of_four(*gate);
      a.vec8 = a.vec8 && rows_of(8, *gate);
    }
  }
  auto grad = [&](const OptTensor& t, const void*& ptr, int64_t& ld) {
    if (!given(t)) return;
    TORCH_CHECK(t->device() == x.device() && t->scalar_type() == type && t->dim() == 2 && t->size(0) == a.rows &&
                    t->size(1) == H && unit_last(*t),
                "norm_residual: gradients must have the type and shape of the outputs and unit last stride");
    ptr = t->data_ptr();
    ld = t->stride(0);
    a.vec = a.vec && rows_of_four(*t);
    a.vec8 = a.vec8 && rows_of(8, *t);
  };
  grad(dy, a.dy, a.dy_ld);
  if (given(w_pre)) grad(dn, a.dn, a.dn_ld);
  at::Tensor dx = at::empty({a.rows, H}, opt), du, dgate, dw_post, dw_pre, dscale;
  a.dx = dx.data_ptr();
  if (has_u) {
    du = at::empty({a.rows, H}, opt);
    a.du = du.data_ptr();
  }
  if (has_gate) {
    dgate = at::empty({a.rows, H}, opt);
    a.dgate = dgate.data_ptr();
  }
  auto param = [&](const OptTensor& t, bool used, at::Tensor& g, void*& ptr) {
    if (!given(t) || !used) return;
    g = at::empty_like(*t);
    ptr = g.data_ptr();
    if (a.rows == 0) g.zero_();
  };
  param(w_post, has_u, dw_post, a.dw_post);
  param(w_pre, true, dw_pre, a.dw_pre);
  param(scale, has_u, dscale, a.dscale);
  if (a.rows > 0) {
    const int sms = num_sms(x.get_device());
    a.n_partial = norm_partials(a, sms);
    at::Tensor partial = at::empty({a.n_partial, 3, H}, x.options().dtype(at::kFloat));
    a.partial = partial.data_ptr<float>();
    launch_norm_bwd(a, sms, cur_stream());
    SU_LAUNCH_CHECK();
  }
  return {dx, du, dgate, dw_post, dw_pre, dscale};
}

namespace {

// [rows, H] of any shape, unit last stride (a copy where the rows cannot be one dimension)
at::Tensor as_rows(const at::Tensor& t, int64_t width) {
  if (!t.defined()) return t;
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  return unit_last(r) ? r : r.contiguous();
}
at::Tensor like_shape(const at::Tensor& t, at::IntArrayRef shape) {
  return !t.defined() || t.sizes() == shape ? t : t.view(shape);
}

struct NormResidual : public torch::autograd::Function<NormResidual> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& u, const OptTensor& gate,
                               const OptTensor& w_post, const OptTensor& w_pre, const OptTensor& scale, double eps,
                               bool keep8) {
    const int64_t H = x.size(-1);
    auto out = norm_residual_fwd(as_rows(x, H), maybe(as_rows(value(u), H)), maybe(as_rows(value(gate), H)), w_post,
                                 w_pre, scale, eps, keep8);
    if (keep8)
      ctx->save_for_backward({out[2], {}, {}, hidden(out[3]), value(w_post), value(w_pre), value(scale)});
    else
      ctx->save_for_backward({x, value(u), value(gate), {}, value(w_post), value(w_pre), value(scale)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["bf16"] = x.scalar_type() == at::kBFloat16;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["has_y"] = out[0].defined();
    ctx->set_materialize_grads(false);
    variable_list both;
    for (int k = 0; k < 2; ++k)
      if (out[k].defined()) both.push_back(like_shape(out[k], x.sizes()));
    return both;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("norm_residual");
    const auto v = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t H = shape.back();
    const bool keep8 = v[3].defined();
    const bool has_y = ctx->saved_data["has_y"].toBool();
    const at::Tensor dy = has_y ? grads[0] : at::Tensor();
    const at::Tensor dn = has_y ? (grads.size() > 1 ? grads[1] : at::Tensor()) : grads[0];
    auto g = norm_residual_bwd(keep8 ? plain(v[0]) : as_rows(v[0], H), maybe(as_rows(v[1], H)), maybe(as_rows(v[2], H)),
                               maybe(shown(plain(v[3]))), maybe(plain(v[4])), maybe(plain(v[5])), maybe(plain(v[6])),
                               ctx->saved_data["eps"].toDouble(), maybe(as_rows(dy, H)), maybe(as_rows(dn, H)),
                               ctx->saved_data["bf16"].toBool());
    return {like_shape(g[0], shape), like_shape(g[1], shape), like_shape(g[2], shape), g[3], g[4], g[5], {}, {}};
  }
};

}  // namespace

// The op as the Python package calls it: any shape [.., H], autograd. -> y (None without u), n (None
// without w_pre)
std::tuple<OptTensor, OptTensor> norm_residual(const at::Tensor& x, const OptTensor& u_in, const OptTensor& gate_in,
                                               const OptTensor& post_in, const OptTensor& pre_in,
                                               const OptTensor& scale_in, double eps, bool keep8) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "norm_residual: x needs a last dimension of at least one value");
  const at::Tensor u = value(u_in), gate = value(gate_in);
  const auto vec = [](const OptTensor& t) { return given(t) ? t->contiguous() : at::Tensor(); };
  const at::Tensor w_post = vec(post_in), w_pre = vec(pre_in), scale = vec(scale_in);
  for (const auto& t : {u, gate})
    TORCH_CHECK(!t.defined() || (t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device()),
                "norm_residual: u and gate must have x's shape, type and device");
  check_no_tangent("norm_residual", {x, u, gate, w_post, w_pre, scale});
  at::Tensor y, n;
  if (wants_grad({x, u, gate, w_post, w_pre, scale})) {
    auto out = NormResidual::apply(x, maybe(u), maybe(gate), maybe(w_post), maybe(w_pre), maybe(scale), eps, keep8);
    size_t k = 0;
    if (u.defined()) y = out[k++];
    if (w_pre.defined()) n = out[k];
  } else {
    const int64_t H = x.size(-1);
    auto out = norm_residual_fwd(as_rows(x, H), maybe(as_rows(u, H)), maybe(as_rows(gate, H)), maybe(w_post),
                                 maybe(w_pre), maybe(scale), eps, false);
    y = like_shape(out[0], x.sizes());
    n = like_shape(out[1], x.sizes());
  }
  return {maybe(y), maybe(n)};
}

// x [.., H] -> codes [rows, H], scales [rows, ceil(H / 32)]
std::tuple<at::Tensor, at::Tensor> quantize8(const at::Tensor& x_in) {
  SU_CHECK_CUDA(x_in);
  TORCH_CHECK(is_float_type(x_in) && x_in.dim() >= 1 && x_in.size(-1) > 0,
              "quantize8: x must be float32 or bfloat16 with a last dimension of at least one value");
  TORCH_CHECK(x_in.size(-1) <= INT32_MAX, "quantize8: rows of at most 2^31 - 1 values");
  c10::cuda::CUDAGuard guard(x_in.device());
  at::AutoDispatchBelowADInplaceOrView below;  // the codes have no gradient
  const at::Tensor x = as_rows(x_in, x_in.size(-1));
  const int64_t rows = x.size(0), H = x.size(1);
  at::Tensor codes = at::empty({rows, H}, x.options().dtype(at::kChar));
  at::Tensor scales = at::empty({rows, groups_of(H)}, x.options().dtype(at::kFloat));
  if (rows == 0) return {codes, scales};
  launch_quantize8(x.data_ptr(), x.scalar_type() == at::kBFloat16, x.stride(0), rows, static_cast<int>(H),
                   codes.data_ptr<int8_t>(), scales.data_ptr<float>(), rows_of_four(x), num_sms(x.get_device()),
                   cur_stream());
  SU_LAUNCH_CHECK();
  return {codes, scales};
}

at::Tensor dequantize8(const at::Tensor& codes, const at::Tensor& scales, bool bf16) {
  SU_CHECK_CUDA(codes);
  SU_CHECK_CUDA(scales);
  SU_CHECK_CONTIG(codes);
  SU_CHECK_CONTIG(scales);
  SU_CHECK_F32(scales);
  TORCH_CHECK(codes.scalar_type() == at::kChar && codes.dim() == 2, "dequantize8: codes must be int8 rows");
  const int64_t rows = codes.size(0), H = codes.size(1);
  TORCH_CHECK(scales.dim() == 2 && scales.size(0) == rows && scales.size(1) == groups_of(H) &&
                  scales.device() == codes.device() && H <= INT32_MAX,
              "dequantize8: one scale per row and group of ", str(kGroup8), " values");
  c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor x = at::empty({rows, H}, codes.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  if (x.numel() == 0) return x;
  const bool vec = H % 4 == 0 && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 4 == 0;
  launch_dequantize8(codes.data_ptr<int8_t>(), scales.data_ptr<float>(), rows, static_cast<int>(H), x.data_ptr(), bf16,
                     vec, num_sms(codes.get_device()), cur_stream());
  SU_LAUNCH_CHECK();
  return x;
}
