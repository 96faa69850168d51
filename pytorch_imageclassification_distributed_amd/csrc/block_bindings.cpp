// Bindings of the pre-norm 8-bit linear block (block_ops.hip, fp8_gemm.hip): every argument a kernel's indexing relies
// on is checked here, the launch goes to the current stream of the tensors' own device, and nothing is allocated.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

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
int fp8_gemm_launch(const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, const float*, int, int, int,
                    long, long, int, int, int, long, int, int, hipStream_t);

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

void quant_rows(Tensor x, OT mask, OT q, OT sc, OT copy, OT part, int64_t M, int64_t N) {
  const c10::DeviceGuard guard(x.device());
  const int code = type_code(x, "x");
  dense(x, x, "x");
  TORCH_CHECK(M >= 0 && N >= 1 && N < (1LL << 30) && x.numel() == M * N, "quantize_fp8: shape");
  like(mask, x, "mask");
  const int chunk = quant_rows_chunk(M, (int)N);
  int64_t ldq = 0, ldsc = 0, ldb = 0;
  if (raw(q)) {
    TORCH_CHECK(raw(sc), "quantize_fp8: q without scale");
    blocks(*q, *sc, x, M, N, 1);
    ldq = q->size(1); ldsc = sc->size(1);
  }
  if (raw(copy)) {
    typed(copy, x, at::kBFloat16, 0, "copy");
    TORCH_CHECK(copy->dim() == 2 && copy->size(0) == M && copy->size(1) == (N + 7) / 8 * 8, "quantize_fp8: copy shape");
    ldb = copy->size(1);
  }
  typed(part, x, at::kFloat, (M + chunk - 1) / chunk * N, "part");
  ok(quant_rows_launch(x.data_ptr(), raw(mask), (uint8_t*)raw(q), (uint8_t*)raw(sc), (bf16_t*)raw(copy),
                       (float*)raw(part), M, (int)N, chunk, ldq, (int)ldsc, (int)ldb, code, stream_of(x)),
     "quantize_fp8");
}

void quant_tiles(Tensor w, Tensor q, Tensor sc, OT qt, OT sct) {
  const c10::DeviceGuard guard(w.device());
  const int code = type_code(w, "w");
  dense(w, w, "w");
  TORCH_CHECK(w.dim() == 2 && w.size(0) < (1LL << 23) - 128 && w.size(1) >= 1 && w.size(1) < (1LL << 30),
              "quantize_fp8_weight: shape");
  const int64_t M = w.size(0), N = w.size(1);
  blocks(q, sc, w, M, N, 128);
  if (raw(qt)) {
    TORCH_CHECK(raw(sct), "quantize_fp8_weight: transpose without scale");
    blocks(*qt, *sct, w, N, M, 128);
  }
  ok(quant_tiles_launch(w.data_ptr(), (uint8_t*)q.data_ptr(), sc.data_ptr<uint8_t>(), (uint8_t*)raw(qt), (uint8_t*)raw(sct),
                        (int)M, (int)N, q.size(1), (int)sc.size(1), raw(qt) ? qt->size(1) : 0,
                        raw(qt) ? (int)sct->size(1) : 0, code, stream_of(w)),
     "quantize_fp8_weight");
}

void fp8_dequant(Tensor q, Tensor sc, Tensor y, int64_t tile) {
  const c10::DeviceGuard guard(q.device());
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
  // one block a 128 x 128 tile or smaller
  TORCH_CHECK(((M + 15) / 16) * ((N + 15) / 16) < (1LL << 31), "matmul_fp8: grid too large");
  ok(fp8_gemm_launch((const uint8_t*)a.data_ptr(), as.data_ptr<uint8_t>(), (const uint8_t*)b.data_ptr(),
                     bs.data_ptr<uint8_t>(), c.data_ptr(), (const float*)raw(bias), (int)M, (int)N, (int)(a.size(1) / 128),
                     a.size(1), b.size(1), (int)as.size(1), (int)bs.size(1), btile == 128 ? 7 : 0, N, act, code,
                     stream_of(a)),
     "matmul_fp8");
}

}  // namespace

void register_block_ops(pybind11::module& m) {
  m.def("dropout_counter", &dropout_counter);
  m.def("rms_max_cols", &rms_max_cols);
  m.def("rms_fwd", &rms_fwd);
  m.def("rms_fwd_fp8", &rms_fwd_fp8);
  m.def("rms_bwd_blocks", [](int64_t rows, int64_t N) { return rms_bwd_blocks(rows, (int)N); });
  m.def("rms_bwd", &rms_bwd);
  m.def("rows_sum", &rows_sum);
  m.def("quant_rows_groups", [](int64_t M, int64_t N) {
    const int c = quant_rows_chunk(M, (int)N);
    return (M + c - 1) / c;
  });
  m.def("quant_rows", &quant_rows);
  m.def("quant_tiles", &quant_tiles);
  m.def("fp8_dequant", &fp8_dequant);
  m.def("fp8_gemm", &fp8_gemm);
}
