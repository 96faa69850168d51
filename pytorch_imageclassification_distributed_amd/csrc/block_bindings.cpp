// The pre-norm 8-bit linear block (block_ops.hip, fp8_gemm.hip) as autograd operators.  Every argument a kernel's
// indexing relies on is checked here, the launch goes to the current stream of the tensors' own device, and outputs and
// workspaces come from the caching allocator (they live as long as the call, or as what it saves for backward).
//
// The autograd nodes are C++: a small call is bound by the host, and a Python node costs it twice the time of one of
// torch's own (4 x 2048 dropout, forward and backward: 70 us with a Python node, 46 us for torch's product).
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <optional>

using at::Tensor;
using OT = std::optional<Tensor>;
typedef uint16_t bf16_t;

int dropout_counter_launch(const void*, const void*, void*, long, int, const long long*, unsigned long long,
                           unsigned long long, int, hipStream_t);
int rms_max_cols();
int rms_fwd_launch(const void*, const void*, const float*, void*, void*, uint8_t*, uint8_t*, float*, long, int, long,
                   int, float, int, const long long*, unsigned long long, unsigned long long, int, hipStream_t);
int rms_bwd_blocks(long, int);
int rms_bwd_launch(const void*, const void*, const void*, const float*, const float*, void*, void*, float*, int, long,
                   int, int, const long long*, unsigned long long, unsigned long long, int, hipStream_t);
int rows_sum_launch(const float*, float*, int, int, hipStream_t);
int quant_rows_chunk(long, int);
int quant_rows_launch(const void*, const void*, uint8_t*, uint8_t*, bf16_t*, float*, long, int, int, long, int, int,
                      int, hipStream_t);
int quant_tiles_launch(const void*, uint8_t*, uint8_t*, uint8_t*, uint8_t*, int, int, long, int, long, int, int,
                       hipStream_t);
int dequant_launch(const uint8_t*, const uint8_t*, void*, long, int, long, int, int, int, hipStream_t);
void rows_grad_force(int);
int rows_grad_forced();
int rows_grad_plan(int, int, int, int, int, int*);
int rows_grad_launch(const bf16_t*, const bf16_t*, float*, float*, int, int, int, int, int, int, int, hipStream_t);
void fp8_gemm_force(int);
int fp8_gemm_plan(int, int, int, int);
int fp8_gemm_launch(const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, const float*, int, int, int,
                    int, long, long, int, int, int, long, int, int, hipStream_t);

namespace {

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void ok(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " launch failed: ", hipGetErrorString((hipError_t)rc));
}

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, name, " has dtype ", t.scalar_type(), ", expected bfloat16, float16 or float32");
  }
}

// dense, 16-byte aligned, on x's device
void dense(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name, " must be on ", x.device());
  TORCH_CHECK(t.is_contiguous() && ((uintptr_t)t.data_ptr() & 15) == 0, name, " must be contiguous and 16-byte aligned");
}

void like(const OT& t, const Tensor& x, const char* name) {
  if (!t.has_value() || !t->defined()) return;
  dense(*t, x, name);
  TORCH_CHECK(t->scalar_type() == x.scalar_type() && t->numel() == x.numel(), name, " must have x's type and size");
}

void typed(const OT& t, const Tensor& x, at::ScalarType st, int64_t least, const char* name) {
  if (!t.has_value() || !t->defined()) return;
  dense(*t, x, name);
  TORCH_CHECK(t->scalar_type() == st && t->numel() >= least, name, " must be ", st, " with at least ", least, " values");
}

void* raw(const OT& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

const long long* state_of(const OT& st, const Tensor& x) {
  typed(st, x, at::kLong, 2, "seed");
  return (const long long*)raw(st);
}

void threshold(int t) { TORCH_CHECK(t >= 0 && t <= 65536, "drop threshold out of range"); }

// a copy where t does not begin at a multiple of `bytes` (a user's blocks may be slices of a checkpoint's buffer)
Tensor aligned(const Tensor& t, uintptr_t bytes) { return ((uintptr_t)t.data_ptr() & (bytes - 1)) == 0 ? t : t.clone(); }

// [rows, cols] e4m3 with cols a multiple of 128, and its scales
void blocks(const Tensor& q, const Tensor& sc, const Tensor& x, int64_t rows, int64_t cols, int64_t tile) {
  dense(q, x, "q");
  TORCH_CHECK(sc.is_cuda() && sc.device() == x.device() && sc.is_contiguous() && ((uintptr_t)sc.data_ptr() & 3) == 0,
              "scale must be contiguous, 4-byte aligned and on ", x.device());
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2 && q.size(0) == rows && q.size(1) % 128 == 0 &&
                  q.size(1) >= cols && q.size(1) < cols + 128,
              "q must be float8_e4m3fn [rows, cols rounded up to 128]");
  TORCH_CHECK(sc.scalar_type() == at::kByte && sc.dim() == 2 && sc.size(0) == (rows + tile - 1) / tile &&
                  sc.size(1) == (q.size(1) / 128 + 3) / 4 * 4,
              "scale must be uint8 [rows / tile, 128-column blocks rounded up to 4]");
}

void dropout_counter(Tensor x, OT res, Tensor y, OT state, uint64_t seed, uint64_t offset, int t) {
  const c10::DeviceGuard guard(x.device());
  const int code = type_code(x, "x");
  dense(x, x, "x");
  like(res, x, "residual");
  like(y, x, "y");
  threshold(t);
  ok(dropout_counter_launch(x.data_ptr(), raw(res), y.data_ptr(), x.numel(), code, state_of(state, x), seed, offset, t,
                            stream_of(x)),
     "dropout_counter");
}

void rms_rows(const Tensor& x, int64_t rows, int64_t N) {
  TORCH_CHECK(rows >= 0 && N >= 1 && N <= rms_max_cols() && x.numel() == rows * N, "rms_norm: rows of 1..", rms_max_cols(),
              " columns");
  TORCH_CHECK(rows < (1LL << 31), "rms_norm: too many rows");
}

void rms_fwd(Tensor x, OT res, OT w, OT h, Tensor y, OT rstd, int64_t rows, int64_t N, double eps, OT state,
             uint64_t seed, uint64_t offset, int t) {
  const c10::DeviceGuard guard(x.device());
  const int code = type_code(x, "x");
  dense(x, x, "x");
  rms_rows(x, rows, N);
  like(res, x, "residual"); like(h, x, "h"); like(y, x, "y");
  typed(w, x, at::kFloat, N, "weight"); typed(rstd, x, at::kFloat, rows, "rstd");
  threshold(t);
  ok(rms_fwd_launch(x.data_ptr(), raw(res), (const float*)raw(w), raw(h), y.data_ptr(), nullptr, nullptr,
                    (float*)raw(rstd), rows, (int)N, 0, 0, (float)eps, code, state_of(state, x), seed, offset, t,
                    stream_of(x)),
     "rms_norm");
}

void rms_fwd_fp8(Tensor x, OT res, OT w, OT h, Tensor q, Tensor sc, int64_t rows, int64_t N, double eps) {
  const c10::DeviceGuard guard(x.device());
  const int code = type_code(x, "x");
  dense(x, x, "x");
  rms_rows(x, rows, N);
  like(res, x, "residual"); like(h, x, "h");
  typed(w, x, at::kFloat, N, "weight");
  blocks(q, sc, x, rows, N, 1);
  ok(rms_fwd_launch(x.data_ptr(), raw(res), (const float*)raw(w), raw(h), nullptr, (uint8_t*)q.data_ptr(),
                    sc.data_ptr<uint8_t>(), nullptr, rows, (int)N, q.size(1), (int)sc.size(1), (float)eps, code, nullptr,
                    0, 0, 0, stream_of(x)),
     "rms_norm_fp8");
}

void rms_bwd(Tensor dy, Tensor h, OT dh, OT w, Tensor rstd, OT dx, OT dres, OT part, int64_t rows, int64_t N, OT state,
             uint64_t seed, uint64_t offset, int t) {
  const c10::DeviceGuard guard(dy.device());
  const int code = type_code(dy, "dy");
  dense(dy, dy, "dy");
  rms_rows(dy, rows, N);
  like(h, dy, "h"); like(dh, dy, "dh"); like(dx, dy, "dx"); like(dres, dy, "dres");
  const int nb = rms_bwd_blocks(rows, (int)N);
  typed(w, dy, at::kFloat, N, "weight"); typed(rstd, dy, at::kFloat, rows, "rstd");
  typed(part, dy, at::kFloat, (int64_t)nb * N, "part");
  threshold(t);
  ok(rms_bwd_launch(dy.data_ptr(), h.data_ptr(), raw(dh), (const float*)raw(w), rstd.data_ptr<float>(), raw(dx), raw(dres),
                    (float*)raw(part), nb, rows, (int)N, code, state_of(state, dy), seed, offset, t, stream_of(dy)),
     "rms_norm backward");
}

// out[c] = sum_i part[i][c]; out may be any dense fp32 tensor of N values
void rows_sum(Tensor part, Tensor out, int64_t G, int64_t N) {
  const c10::DeviceGuard guard(part.device());
  typed(part, part, at::kFloat, G * N, "part");
  TORCH_CHECK(out.device() == part.device() && out.scalar_type() == at::kFloat && out.is_contiguous() && out.numel() == N &&
                  G >= 0 && G < (1LL << 31) && N < (1LL << 31),
              "rows_sum: out must be contiguous float32 [N]");
  ok(rows_sum_launch(part.data_ptr<float>(), out.data_ptr<float>(), (int)G, (int)N, stream_of(part)), "rows_sum");
}

void quant_rows(Tensor x, Tensor q, Tensor sc, int64_t M, int64_t N) {
  const c10::DeviceGuard guard(x.device());
  const int code = type_code(x, "x");
  dense(x, x, "x");
  TORCH_CHECK(M >= 0 && N >= 1 && N < (1LL << 30) && x.numel() == M * N, "quantize_fp8: shape");
  blocks(q, sc, x, M, N, 1);
  ok(quant_rows_launch(x.data_ptr(), nullptr, (uint8_t*)q.data_ptr(), sc.data_ptr<uint8_t>(), nullptr, nullptr, M, (int)N,
                       quant_rows_chunk(M, (int)N), q.size(1), (int)sc.size(1), 0, code, stream_of(x)),
     "quantize_fp8");
}

void quant_tiles(Tensor w, Tensor q, Tensor sc) {
  const c10::DeviceGuard guard(w.device());
  const int code = type_code(w, "w");
  dense(w, w, "w");
  TORCH_CHECK(w.dim() == 2 && w.size(0) < (1LL << 23) - 128 && w.size(1) >= 1 && w.size(1) < (1LL << 30),
              "quantize_fp8_weight: shape");
  blocks(q, sc, w, w.size(0), w.size(1), 128);
  ok(quant_tiles_launch(w.data_ptr(), (uint8_t*)q.data_ptr(), sc.data_ptr<uint8_t>(), nullptr, nullptr, (int)w.size(0),
                        (int)w.size(1), q.size(1), (int)sc.size(1), 0, 0, code, stream_of(w)),
     "quantize_fp8_weight");
}

void fp8_dequant(Tensor q, Tensor sc, Tensor y, int64_t tile) {
  const c10::DeviceGuard guard(q.device());
  q = aligned(q, 16);
  sc = aligned(sc, 4);
  const int code = type_code(y, "y");
  dense(y, q, "y");
  TORCH_CHECK(y.dim() == 2 && (tile == 1 || tile == 128) && y.size(1) < (1LL << 31), "dequantize: shape");
  blocks(q, sc, q, y.size(0), y.size(1), tile);
  ok(dequant_launch((const uint8_t*)q.data_ptr(), sc.data_ptr<uint8_t>(), y.data_ptr(), y.size(0), (int)y.size(1),
                    q.size(1), (int)sc.size(1), (int)tile, code, stream_of(q)),
     "dequantize");
}

void fp8_gemm(Tensor a, Tensor as, Tensor b, Tensor bs, Tensor c, OT bias, int64_t K, int64_t btile, int act) {
  const c10::DeviceGuard guard(a.device());
  const int code = type_code(c, "out");
  TORCH_CHECK(c.dim() == 2 && c.device() == a.device() && c.is_contiguous(), "matmul_fp8: out must be contiguous [M, N]");
  const int64_t M = c.size(0), N = c.size(1);
  TORCH_CHECK(btile == 1 || btile == 128, "matmul_fp8: b's tile");
  TORCH_CHECK(K >= 1 && K < (1LL << 30) && M < (1LL << 30) && N < (1LL << 30), "matmul_fp8: size");
  TORCH_CHECK(act >= 0 && act <= 2, "matmul_fp8: act");
  blocks(a, as, a, M, K, 1);
  blocks(b, bs, a, N, K, btile);
  typed(bias, a, at::kFloat, N, "bias");
  TORCH_CHECK(M * N == 0 || fp8_gemm_plan((int)M, (int)N, (int)(a.size(1) / 128), btile == 128 ? 7 : 0) >= 0,
              "matmul_fp8: no kernel takes [", M, ", ", K, "] x [", N, ", ", K, "]: too large");
  ok(fp8_gemm_launch((const uint8_t*)a.data_ptr(), as.data_ptr<uint8_t>(), (const uint8_t*)b.data_ptr(),
                     bs.data_ptr<uint8_t>(), c.data_ptr(), (const float*)raw(bias), (int)M, (int)N, (int)(a.size(1) / 128),
                     (int)(K % 128), a.size(1), b.size(1), (int)as.size(1), (int)bs.size(1), btile == 128 ? 7 : 0, N, act, code,
                     stream_of(a)),
     "matmul_fp8");
}

// ---------------------------------------------------------------------------------------------------------------------
// operators
// ---------------------------------------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// row-major and 16-byte aligned (the kernels move whole 16-byte vectors); a copy where it is not
Tensor dense16(const Tensor& t) {
  Tensor c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15) == 0 ? c : c.clone();
}
OT dense16(const OT& t) { return t.has_value() && t->defined() ? OT(dense16(*t)) : OT(); }
// a float32 copy where it is not float32 already (only read through its pointer: no gradient flows here)
OT f32(const OT& t) {
  if (!t.has_value() || !t->defined()) return OT();
  return t->scalar_type() == at::kFloat ? dense16(*t) : dense16(t->detach().to(at::kFloat));
}
OT some(const Tensor& t) { return t.defined() ? OT(t) : OT(); }
bool has(const OT& t) { return t.has_value() && t->defined(); }
Tensor or_undefined(const OT& t) { return has(t) ? *t : Tensor(); }
bool wants(const OT& t) { return has(t) && t->requires_grad(); }

// The operators have no forward-mode derivative.  Their nodes refuse one, but a dual tensor need not ask for a gradient
// (and may come under no_grad), and then no node is made: without this the tangent would be lost without an error.
void no_tangent(const char* what, std::initializer_list<Tensor> in) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : in)
    TORCH_CHECK_NOT_IMPLEMENTED(!(t.defined() && t._fw_grad(/*level=*/0).defined()), what,
                                " has no forward-mode derivative, and an input carries a tangent");
}

Tensor fresh(at::IntArrayRef size, const Tensor& like, at::ScalarType st) { return at::empty(size, like.options().dtype(st)); }

struct Blocks {
  Tensor q, sc;
};
Blocks empty_blocks(int64_t rows, int64_t cols, int64_t tile, const Tensor& like) {
  const int64_t nb = (cols + 127) / 128;
  return {fresh({rows, nb * 128}, like, at::kFloat8_e4m3fn), fresh({(rows + tile - 1) / tile, (nb + 3) / 4 * 4}, like, at::kByte)};
}

// A Python callable that hands out the tensor for a parameter's float32 gradient (its gradient-arena slot)
struct Slot : torch::CustomClassHolder {
  py::object fn;
  explicit Slot(py::object f) : fn(std::move(f)) {}
  ~Slot() override {
    if (!Py_IsInitialized()) {  // a graph that outlives the interpreter
      fn.release();
      return;
    }
    py::gil_scoped_acquire gil;
    fn = py::object();
  }
};
c10::IValue slot_value(const py::object& fn) {
  if (fn.is_none()) return c10::IValue();
  return c10::IValue::make_capsule(c10::make_intrusive<Slot>(fn));
}
Tensor slot_or_empty(const c10::IValue& v, at::IntArrayRef size, const Tensor& like) {
  if (v.isNone()) return fresh(size, like, at::kFloat);
  auto slot = c10::static_intrusive_pointer_cast<Slot>(v.toCapsule());
  py::gil_scoped_acquire gil;
  return py::cast<Tensor>(slot->fn());
}

// The kernels' gradients have no second derivative: differentiating them again raises
variable_list no_second(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "the gradients of the dropout / RMS norm / 8-bit linear operators cannot be differentiated again", (int64_t)in.size());
  variable_list out = (*err)(std::move(in));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// drop arguments that travel through the nodes: threshold, seed, offset (64-bit patterns), and the device state
struct DropArgs {
  int64_t t;
  uint64_t seed, offset;
  void save(AutogradContext* ctx) const {
    ctx->saved_data["t"] = t;
    ctx->saved_data["seed"] = (int64_t)seed;
    ctx->saved_data["offset"] = (int64_t)offset;
  }
  static DropArgs load(AutogradContext* ctx) {
    return {ctx->saved_data["t"].toInt(), (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt()};
  }
};

Tensor drop_forward(const Tensor& x, const OT& residual, const OT& state, const DropArgs& d) {
  Tensor xd = dense16(x), y = at::empty_like(xd);
  dropout_counter(xd, dense16(residual), y, state, d.seed, d.offset, (int)d.t);
  return y;
}

struct DropoutCounterNode : torch::autograd::Function<DropoutCounterNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OT& residual, const OT& state, int64_t t,
                        int64_t seed, int64_t offset) {
    const DropArgs d{t, (uint64_t)seed, (uint64_t)offset};
    ctx->save_for_backward({or_undefined(state)});
    d.save(ctx);
    ctx->saved_data["res"] = has(residual);
    return drop_forward(x, residual, state, d);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const OT state = some(ctx->get_saved_variables()[0]);
    const DropArgs d = DropArgs::load(ctx);
    Tensor dx;
    if (ctx->needs_input_grad(0)) dx = d.t == 0 ? g[0] : no_second({drop_forward(g[0].detach(), OT(), state, d)})[0];
    return {dx, ctx->saved_data["res"].toBool() ? g[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor op_dropout_counter(const Tensor& x, const OT& residual, const OT& state, uint64_t seed, uint64_t offset, int64_t t) {
  no_tangent("dropout_counter", {x, or_undefined(residual)});
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || wants(residual)))  // nothing asks for a gradient
    return drop_forward(x, residual, state, {t, seed, offset});
  return DropoutCounterNode::apply(x, residual, state, t, (int64_t)seed, (int64_t)offset);
}

// y (and h): one pass over x and residual; h and one float a row are kept for the backward pass, which makes the dropout
// mask again
struct RmsOut {
  Tensor y, h, w, rstd;  // h undefined where it equals x
};
RmsOut rms_forward(const Tensor& x, const OT& residual, const OT& weight, const OT& state, const DropArgs& d, double eps,
                   bool need) {
  const int64_t n = x.size(-1), rows = x.numel() / n;
  RmsOut o;
  o.y = at::empty_like(x);
  if (has(residual) || (d.t > 0 && need)) o.h = at::empty_like(x);
  if (need) o.rstd = fresh({rows}, x, at::kFloat);
  const OT w = f32(weight);
  o.w = or_undefined(w);
  rms_fwd(x, dense16(residual), w, some(o.h), o.y, some(o.rstd), rows, n, eps, state, d.seed, d.offset, (int)d.t);
  return o;
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const OT& residual, const OT& weight,
                               const OT& state, int64_t t, int64_t seed, int64_t offset, double eps, c10::IValue slot) {
    const DropArgs d{t, (uint64_t)seed, (uint64_t)offset};
    const Tensor x = dense16(x_);
    RmsOut o = rms_forward(x, residual, weight, state, d, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({o.h.defined() ? o.h : x, o.w, o.rstd, or_undefined(state)});
    d.save(ctx);
    ctx->saved_data["res"] = has(residual);
    ctx->saved_data["wtype"] = has(weight) ? (int64_t)weight->scalar_type() : (int64_t)-1;
    ctx->saved_data["slot"] = std::move(slot);
    if (has(residual)) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &h = s[0], &rstd = s[2];
    const OT w = some(s[1]), state = some(s[3]);
    const DropArgs d = DropArgs::load(ctx);
    const int64_t n = h.size(-1), rows = h.numel() / n;
    const bool res = ctx->saved_data["res"].toBool();
    // (needs_input_grad counts the defined tensors)
    const bool nx = ctx->needs_input_grad(0), nr = res && ctx->needs_input_grad(1), nw = w.has_value() && ctx->needs_input_grad(1 + res);
    const Tensor dy = g[0].defined() ? dense16(g[0].detach()) : at::zeros_like(h);
    const OT dh = res && g[1].defined() ? OT(dense16(g[1].detach())) : OT();
    Tensor dx, dres, part, dw;
    const bool one = d.t == 0;  // without dropout the two gradients are one tensor
    if (nx || (nr && one)) dx = at::empty_like(h);
    if (nr && !one) dres = at::empty_like(h);
    if (nw) part = fresh({rms_bwd_blocks(rows, (int)n), n}, h, at::kFloat);
    rms_bwd(dy, h, dh, w, rstd, some(dx), some(dres), some(part), rows, n, state, d.seed, d.offset, (int)d.t);
    if (nw) {
      dw = slot_or_empty(ctx->saved_data["slot"], {n}, h);
      rows_sum(part, dw, rows ? part.size(0) : 0, n);
      const auto wt = (at::ScalarType)ctx->saved_data["wtype"].toInt();
      if (wt != at::kFloat) dw = dw.to(wt);
    }
    variable_list out = no_second({nx ? dx : Tensor(), nr ? (one ? dx : dres) : Tensor(), dw});
    return {out[0], out[1], out[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// [y] or [y, h]
std::vector<Tensor> op_rms_norm(const Tensor& x, const OT& residual, const OT& weight, const OT& state, uint64_t seed,
                                uint64_t offset, int64_t t, double eps, py::object slot) {
  no_tangent("rms_norm", {x, or_undefined(residual), or_undefined(weight)});
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || wants(residual) || wants(weight))) {
    RmsOut o = rms_forward(dense16(x), residual, weight, state, {t, seed, offset}, eps, false);
    if (has(residual)) return {o.y, o.h};
    return {o.y};
  }
  return RmsNormNode::apply(x, residual, weight, state, t, (int64_t)seed, (int64_t)offset, eps, slot_value(slot));
}

// (q, scale, h or None)
std::tuple<Tensor, Tensor, OT> op_rms_norm_fp8(const Tensor& x_, const OT& residual, const OT& weight, double eps) {
  const at::NoGradGuard no_grad;
  const Tensor x = dense16(x_);
  const int64_t n = x.size(-1), rows = x.numel() / n;
  Blocks b = empty_blocks(rows, n, 1, x);
  OT h;
  if (has(residual)) h = at::empty_like(x);
  rms_fwd_fp8(x, dense16(residual), f32(weight), h, b.q, b.sc, rows, n, eps);
  return {b.q, b.sc, h};
}

std::tuple<Tensor, Tensor> op_quantize_rows(const Tensor& x_) {
  const Tensor x = dense16(x_.detach());
  Blocks b = empty_blocks(x.size(0), x.size(1), 1, x);
  quant_rows(x, b.q, b.sc, x.size(0), x.size(1));
  return {b.q, b.sc};
}

std::tuple<Tensor, Tensor> op_quantize_tiles(const Tensor& w_) {
  const Tensor w = dense16(w_.detach());
  Blocks b = empty_blocks(w.size(0), w.size(1), 128, w);
  quant_tiles(w, b.q, b.sc);
  return {b.q, b.sc};
}

Tensor op_matmul(const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, const OT& bias, int64_t n, int64_t k,
                 int64_t btile, int64_t act, at::ScalarType out) {
  Tensor c = fresh({a.size(0), n}, a, out);
  fp8_gemm(aligned(a, 16), aligned(as, 4), aligned(b, 16), aligned(bs, 4), c, f32(bias), k, btile, (int)act);
  return c;
}

// dw[n][k] = sum over the m rows of dy[row][n] x[row][k]; dy, x: bf16, widths n, k rounded up to 8
void rows_grad(const bf16_t* dy, const Tensor& x, const Tensor& dw, int64_t m, int64_t n, int64_t k, int force) {
  const c10::DeviceGuard guard(dw.device());
  const int64_t ldy = (n + 7) / 8 * 8, ldx = (k + 7) / 8 * 8;
  typed(x, dw, at::kBFloat16, m * ldx, "x");
  TORCH_CHECK(dw.scalar_type() == at::kFloat && dw.is_contiguous() && dw.numel() == n * k && ((uintptr_t)dw.data_ptr() & 15) == 0,
              "linear_fp8: weight gradient must be contiguous float32");
  int tile = 0;
  const int splits = rows_grad_plan((int)m, (int)n, (int)k, (int)std::max(ldy, ldx), force, &tile);
  TORCH_CHECK(splits > 0, "linear_fp8: rows too wide for the weight gradient");
  Tensor slabs;
  if (splits > 1) slabs = fresh({splits * n * k}, dw, at::kFloat);
  ok(rows_grad_launch(dy, (const bf16_t*)x.data_ptr(), dw.data_ptr<float>(), splits > 1 ? slabs.data_ptr<float>() : nullptr,
                      (int)m, (int)n, (int)k, (int)ldy, (int)ldx, tile, splits, stream_of(dw)),
     "linear_fp8 weight gradient");
}

// y = act(q(x) q(w)^T + b).  Backward: dx = q(dy) q(w) in 8 bits (the weights' transpose was written beside them; 128 x
// 128 tiles keep their scale), db in float32, and dw = dy^T x on bf16 operands: weight gradients are summed into float32
// masters over many steps, and the 8-bit matrix instructions cut their products (fp8_gemm.hip) where the bf16 ones keep
// float32.
// The quantised operands of a call live in one buffer (an allocation costs a small call as much as a launch does).
struct Layout {
  int64_t size = 0;
  int64_t add(int64_t bytes) {
    const int64_t at = size;
    size += (bytes + 255) / 256 * 256;
    return at;
  }
};
int64_t blocks_of(int64_t cols) { return (cols + 127) / 128; }
int64_t scales_of(int64_t cols) { return (blocks_of(cols) + 3) / 4 * 4; }

struct LinearOut {
  Tensor y, xb, wt;  // wt: q(w)^T and, behind it, its scales
};
LinearOut linear_forward(const Tensor& x, const Tensor& weight, const OT& bias, int64_t act, bool need_x, bool need_w) {
  const c10::DeviceGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) == k && weight.device() == x.device(), "linear_fp8: weight shape");
  TORCH_CHECK(m < (1LL << 30) && n >= 1 && n < (1LL << 23) - 128 && k >= 1 && k < (1LL << 23) - 128, "linear_fp8: size");
  int tile = 0;  // (a width whose weight gradient no launch takes is refused here, not after the forward pass)
  TORCH_CHECK(!need_w || rows_grad_plan((int)m, (int)n, (int)k, (int)((std::max(n, k) + 7) / 8 * 8), rows_grad_forced(), &tile) > 0,
              "linear_fp8: rows too wide for the weight gradient");
  const int tx = type_code(x, "x"), tw = type_code(weight, "weight");
  const OT b = f32(bias);
  typed(b, x, at::kFloat, n, "bias");
  const Tensor w = dense16(weight);
  dense(x, x, "x"); dense(w, x, "weight");
  const hipStream_t st = stream_of(x);
  const int64_t kp = blocks_of(k) * 128, ks = scales_of(k), np = blocks_of(n) * 128, ns = scales_of(n);
  LinearOut o;
  o.xb = x;
  bf16_t* copy = nullptr;
  if (need_w && (tx != 0 || k % 8)) {
    o.xb = fresh({m, (k + 7) / 8 * 8}, x, at::kBFloat16);
    copy = (bf16_t*)o.xb.data_ptr();
  }
  Layout l;
  const int64_t aq = l.add(m * kp), as = l.add(m * ks), bq = l.add(n * kp), bs = l.add(blocks_of(n) * ks);
  const Tensor work = fresh({l.size}, x, at::kByte);
  uint8_t* p = work.data_ptr<uint8_t>();
  ok(quant_rows_launch(x.data_ptr(), nullptr, p + aq, p + as, copy, nullptr, m, (int)k, quant_rows_chunk(m, (int)k), kp, (int)ks,
                       (int)((k + 7) / 8 * 8), tx, st),
     "linear_fp8");
  uint8_t *t = nullptr, *ts = nullptr;
  if (need_x) {
    Layout lt;
    const int64_t q = lt.add(k * np), sc = lt.add(blocks_of(k) * ns);
    o.wt = fresh({lt.size}, x, at::kByte);
    t = o.wt.data_ptr<uint8_t>() + q;
    ts = o.wt.data_ptr<uint8_t>() + sc;
  }
  ok(quant_tiles_launch(w.data_ptr(), p + bq, p + bs, t, ts, (int)n, (int)k, kp, (int)ks, np, (int)ns, tw, st), "linear_fp8");
  o.y = fresh({m, n}, x, x.scalar_type());
  ok(fp8_gemm_launch(p + aq, p + as, p + bq, p + bs, o.y.data_ptr(), (const float*)raw(b), (int)m, (int)n, (int)blocks_of(k), 0,
                     kp, kp, (int)ks, (int)ks, 7, n, (int)act, tx, st),
     "linear_fp8");
  return o;
}

struct LinearFp8Node : torch::autograd::Function<LinearFp8Node> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& weight, const OT& bias, int64_t act,
                        bool need_x, bool need_w, c10::IValue wslot, c10::IValue bslot) {
    const Tensor x = dense16(x_);
    LinearOut o = linear_forward(x, weight, bias, act, need_x, need_w);
    ctx->save_for_backward({need_w ? o.xb : Tensor(), o.wt, act ? o.y : Tensor()});
    ctx->saved_data["m"] = x.size(0);
    ctx->saved_data["n"] = weight.size(0);
    ctx->saved_data["k"] = x.size(1);
    ctx->saved_data["wtype"] = (int64_t)weight.scalar_type();
    ctx->saved_data["bias"] = has(bias);
    ctx->saved_data["btype"] = has(bias) ? (int64_t)bias->scalar_type() : (int64_t)at::kFloat;
    ctx->saved_data["tile"] = (int64_t)rows_grad_forced();
    ctx->saved_data["wslot"] = std::move(wslot);
    ctx->saved_data["bslot"] = std::move(bslot);
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &xb = s[0], &wt = s[1], &y = s[2];
    const int64_t m = ctx->saved_data["m"].toInt(), n = ctx->saved_data["n"].toInt(), k = ctx->saved_data["k"].toInt();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    const bool nb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    const Tensor dy = dense16(g[0].detach());
    const c10::DeviceGuard guard(dy.device());
    const int type = type_code(dy, "dy");
    TORCH_CHECK(dy.dim() == 2 && dy.size(0) == m && dy.size(1) == n, "linear_fp8: dy shape");
    if (y.defined()) like(OT(y), dy, "y");
    const hipStream_t st = stream_of(dy);
    const int64_t np = blocks_of(n) * 128, ns = scales_of(n), n8 = (n + 7) / 8 * 8;
    const int chunk = quant_rows_chunk(m, (int)n);
    const int64_t groups = (m + chunk - 1) / chunk;
    // dy once: 8-bit blocks, a (masked) bf16 copy where dw needs one, partial column sums for db
    const bool copied = nw && (type != 0 || n % 8 || y.defined());
    Layout l;
    const int64_t q = l.add(nx ? m * np : 0), sc = l.add(nx ? m * ns : 0), part = l.add(nb ? groups * n * 4 : 0);
    const int64_t copy = l.add(copied ? m * n8 * 2 : 0);
    const Tensor work = fresh({l.size}, dy, at::kByte);
    uint8_t* p = work.data_ptr<uint8_t>();
    if (nx || copied || nb)
      ok(quant_rows_launch(dy.data_ptr(), y.defined() ? y.data_ptr() : nullptr, nx ? p + q : nullptr, nx ? p + sc : nullptr,
                           copied ? (bf16_t*)(p + copy) : nullptr, nb ? (float*)(p + part) : nullptr, m, (int)n, chunk, np,
                           (int)ns, (int)n8, type, st),
         "linear_fp8 backward");
    Tensor dx, dw, db;
    if (nx) {
      dx = fresh({m, k}, dy, dy.scalar_type());
      Layout lt;
      const int64_t t = lt.add(k * np), ts = lt.add(blocks_of(k) * ns);
      uint8_t* w = wt.data_ptr<uint8_t>();
      ok(fp8_gemm_launch(p + q, p + sc, w + t, w + ts, dx.data_ptr(), nullptr, (int)m, (int)k, (int)blocks_of(n), 0, np, np,
                         (int)ns, (int)ns, 7, k, 0, type, st),
         "linear_fp8 backward");
    }
    if (nw) {
      dw = slot_or_empty(ctx->saved_data["wslot"], {n, k}, dy);
      rows_grad(copied ? (const bf16_t*)(p + copy) : (const bf16_t*)dy.data_ptr(), xb, dw, m, n, k,
                (int)ctx->saved_data["tile"].toInt());
      const auto t = (at::ScalarType)ctx->saved_data["wtype"].toInt();
      if (t != at::kFloat) dw = dw.to(t);
    }
    if (nb) {
      db = slot_or_empty(ctx->saved_data["bslot"], {n}, dy);
      TORCH_CHECK(db.scalar_type() == at::kFloat && db.is_contiguous() && db.numel() == n, "linear_fp8: bias gradient");
      ok(rows_sum_launch((const float*)(p + part), db.data_ptr<float>(), (int)groups, (int)n, st), "linear_fp8 backward");
      const auto t = (at::ScalarType)ctx->saved_data["btype"].toInt();
      if (t != at::kFloat) db = db.to(t);
    }
    variable_list out = no_second({dx, dw, db});
    return {out[0], out[1], out[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor op_linear_fp8(const Tensor& x, const Tensor& weight, const OT& bias, int64_t act, py::object wslot,
                     py::object bslot) {
  no_tangent("linear_fp8", {x, weight, or_undefined(bias)});
  const bool grad = at::GradMode::is_enabled(), nx = grad && x.requires_grad(), nw = grad && weight.requires_grad();
  if (!(nx || nw || (grad && wants(bias)))) return linear_forward(dense16(x.detach()), weight, bias, act, false, false).y;
  return LinearFp8Node::apply(x, weight, bias, act, nx, nw, slot_value(wslot), slot_value(bslot));
}

}  // namespace

void register_block_ops(pybind11::module& m) {
  m.def("dropout_counter", &op_dropout_counter);
  m.def("rms_norm", &op_rms_norm);
  m.def("rms_norm_fp8", &op_rms_norm_fp8);
  m.def("quantize_fp8_rows", &op_quantize_rows);
  m.def("quantize_fp8_tiles", &op_quantize_tiles);
  m.def("dequantize_fp8", &fp8_dequant);
  m.def("matmul_fp8", [](const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, const OT& bias, int64_t n,
                         int64_t k, int64_t btile, int64_t act, py::object dtype) {
    return op_matmul(a, as, b, bs, bias, n, k, btile, act, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("linear_fp8", &op_linear_fp8);
  // which kernel runs: forced for the calling thread (tests), and the choice for given sizes
  m.def("fp8_gemm_force", &fp8_gemm_force);
  m.def("fp8_gemm_plan", [](int m, int n, int k, int btile) { return fp8_gemm_plan(m, n, (int)blocks_of(k), btile == 128 ? 7 : 0); });
  m.def("rows_grad_force", &rows_grad_force);
  m.def("rows_grad_plan", [](int m, int n, int k) {
    int tile = 0;
    const int splits = rows_grad_plan(m, n, k, std::max((n + 7) / 8, (k + 7) / 8) * 8, rows_grad_forced(), &tile);
    return std::make_tuple(tile, splits);
  });
}
