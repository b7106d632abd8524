// extern "C" entry points of the operators around the scan layers (declared
// in include/mamba_lm_ops.h): argument checks, launches on the caller's
// stream, status codes and per-thread messages as in ss_capi.cu.
#include <string>

#include "../../include/mamba_lm_ops.h"
#include "ss_ops.h"

namespace {

using mss::set_error;

mss_status bad(const char* op, const char* what) {
  return set_error(MSS_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

mss_status done(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return MSS_OK;
  return set_error(MSS_INTERNAL, std::string(op) + ": " + cudaGetErrorString(e));
}

bool dtype_ok(int d) { return d == MSS_F32 || d == MSS_BF16; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t up16(int64_t k) { return (k + 15) / 16 * 16; }

// counts of CTAs, rows or blocks of 128 that the kernels keep in 32 bits
bool grid_ok(int64_t n) { return n < (1ll << 31); }

// rows up to 2^30 long: the kernels round a row's length up, and step past it, in 32 bits
bool k_ok(int32_t k) { return k <= (1 << 30); }
constexpr const char* kTooLong = "rows must be at most 2^30 long";

const char* codes_fault(const void* codes, int64_t stride, int64_t rows, int k) {
  if (!aligned(codes, 16) || stride % 16 != 0 || (rows > 1 && stride < up16(k)))
    return "codes need a 16-byte aligned base and a row stride that is a multiple of 16 and "
           "covers the row";
  return nullptr;
}

const char* scales_fault(int64_t stride, int64_t rows, int64_t k) {
  if (rows > 1 && stride < (k + 127) / 128) return "the scales' row stride must cover the row";
  return nullptr;
}

mss_status norm_checks(const char* op, int x_dtype, int residual_dtype, const void* residual,
                       int64_t rows, int dim, int64_t x_stride, int64_t residual_stride) {
  if (!dtype_ok(x_dtype) || (residual && !dtype_ok(residual_dtype)))
    return bad(op, "data types must be 0 (f32) or 1 (bf16)");
  if (rows <= 0 || !grid_ok(rows)) return bad(op, "rows must be positive and below 2^31");
  if (dim <= 0 || dim > mss::kNormMaxDim) return bad(op, "dim must be in 1..16384");
  if (rows > 1 && (x_stride < 0 || (residual && residual_stride < 0)))
    return bad(op, "row strides must not be negative");
  return MSS_OK;
}

}  // namespace

extern "C" {

mss_status mamba_ss_rms_norm_fwd(void* stream, int32_t x_dtype, int32_t residual_dtype,
                                 int64_t rows, int32_t dim, float eps, const void* x,
                                 int64_t x_stride, const void* residual, int64_t residual_stride,
                                 const float* weight, void* y, void* h) {
  const char* op = "rms_norm_fwd";
  const mss_status st = norm_checks(op, x_dtype, residual_dtype, residual, rows, dim, x_stride,
                                    residual_stride);
  if (st != MSS_OK) return st;
  if (!x || !weight || !y || (residual == nullptr) != (h == nullptr))
    return bad(op, "x, weight and y must be non-null, and h with a residual only");
  mss::NormParams p{};
  p.rows = rows; p.dim = dim; p.eps = eps;
  p.x = x; p.res = residual; p.weight = weight;
  p.x_stride = x_stride; p.res_stride = residual ? residual_stride : 0;
  p.y = y; p.h = h;
  return done(op, mss::launch_norm_fwd(p, x_dtype, residual ? residual_dtype : -1, false,
                                       static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_rms_norm_fp8(void* stream, int32_t x_dtype, int32_t residual_dtype,
                                 int64_t rows, int32_t dim, float eps, const void* x,
                                 int64_t x_stride, const void* residual, int64_t residual_stride,
                                 const float* weight, void* codes, int64_t code_stride,
                                 void* scales, int64_t scale_stride, void* h) {
  const char* op = "rms_norm_fp8";
  const mss_status st = norm_checks(op, x_dtype, residual_dtype, residual, rows, dim, x_stride,
                                    residual_stride);
  if (st != MSS_OK) return st;
  if (!x || !weight || !codes || !scales || (residual == nullptr) != (h == nullptr))
    return bad(op, "x, weight, codes and scales must be non-null, and h with a residual only");
  if (const char* f = codes_fault(codes, code_stride, rows, dim)) return bad(op, f);
  if (const char* f = scales_fault(scale_stride, rows, dim)) return bad(op, f);
  mss::NormParams p{};
  p.rows = rows; p.dim = dim; p.eps = eps;
  p.x = x; p.res = residual; p.weight = weight;
  p.x_stride = x_stride; p.res_stride = residual ? residual_stride : 0;
  p.h = h;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  p.code_stride = code_stride;
  p.scale_stride = scale_stride;
  return done(op, mss::launch_norm_fwd(p, x_dtype, residual ? residual_dtype : -1, true,
                                       static_cast<cudaStream_t>(stream)));
}

size_t mamba_ss_rms_norm_bwd_workspace_bytes(int64_t rows, int32_t dim) {
  if (rows <= 0 || dim <= 0 || dim > mss::kNormMaxDim) return 0;
  return sizeof(float) * static_cast<size_t>(mss::norm_bwd_parts(rows, dim)) * dim;
}

mss_status mamba_ss_rms_norm_bwd(void* stream, int32_t x_dtype, int32_t has_residual,
                                 int32_t residual_dtype, int64_t rows, int32_t dim, float eps,
                                 const void* h, int64_t h_stride, const void* dy,
                                 int64_t dy_stride, const void* dh, int64_t dh_stride,
                                 const float* weight, void* dx, void* dresidual, float* dweight,
                                 void* workspace, size_t workspace_bytes) {
  const char* op = "rms_norm_bwd";
  if (!has_residual) residual_dtype = x_dtype;
  const mss_status st = norm_checks(op, x_dtype, residual_dtype, h, rows, dim, h_stride,
                                    dy_stride);
  if (st != MSS_OK) return st;
  if (dh && (!has_residual || dh_stride < 0))
    return bad(op, "dh needs a residual and a row stride that is not negative");
  const bool two = has_residual && residual_dtype != x_dtype;
  if (!h || !dy || !weight || !dx || !dweight || (dresidual != nullptr) != two)
    return bad(op, "h, dy, weight, dx and dweight must be non-null, and dresidual exactly where "
                   "its type is not dx's");
  const size_t need = mamba_ss_rms_norm_bwd_workspace_bytes(rows, dim);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return bad(op, ("workspace needs " + std::to_string(need) + " bytes, 16-byte aligned").c_str());
  mss::NormBwdParams p{};
  p.rows = rows; p.dim = dim; p.eps = eps;
  p.h = h; p.dy = dy; p.dh = dh; p.weight = weight;
  p.h_stride = h_stride; p.dy_stride = dy_stride; p.dh_stride = dh ? dh_stride : 0;
  p.dx = dx; p.dres = dresidual;
  p.dw_part = static_cast<float*>(workspace);
  return done(op, mss::launch_norm_bwd(p, x_dtype, has_residual ? residual_dtype : -1, dweight,
                                       static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_quantize_fp8(void* stream, int32_t x_dtype, int32_t channel_major,
                                 int64_t batch, int64_t length, int32_t k, const void* x,
                                 int64_t x_stride, void* codes, int64_t code_stride, void* scales,
                                 int64_t scale_stride) {
  const char* op = "quantize_fp8";
  if (!dtype_ok(x_dtype)) return bad(op, "x_dtype must be 0 (f32) or 1 (bf16)");
  if (batch <= 0 || length <= 0 || k <= 0) return bad(op, "sizes must be positive");
  if (!k_ok(k)) return bad(op, kTooLong);
  const int64_t kb = (k + 127) / 128;
  if (!grid_ok(length) || batch > (1ll << 40) / length ||
      (channel_major ? batch > 65535 || kb > 65535
                     : !grid_ok(batch * length) || !grid_ok(batch * length * kb)))
    return bad(op, "sizes too large");
  if (!x || !codes || !scales) return bad(op, "x, codes and scales must be non-null");
  if (!channel_major && x_stride < 0) return bad(op, "row stride must not be negative");
  if (const char* f = codes_fault(codes, code_stride, batch * length, k)) return bad(op, f);
  if (const char* f = scales_fault(scale_stride, batch * length, k)) return bad(op, f);
  mss::QuantParams p{};
  p.batch = batch; p.length = length; p.k = k;
  p.x = x; p.x_stride = x_stride;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  p.code_stride = code_stride;
  p.scale_stride = scale_stride;
  return done(op, mss::launch_quantize(p, x_dtype, channel_major != 0,
                                       static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_quantize_fp8_both(void* stream, int32_t x_dtype, int64_t rows, int32_t k,
                                      const void* x, int64_t x_stride, void* row_codes,
                                      int64_t row_stride, void* row_scales,
                                      int64_t row_scale_stride, void* col_codes,
                                      int64_t col_stride, void* col_scales,
                                      int64_t col_scale_stride) {
  const char* op = "quantize_fp8_both";
  if (!dtype_ok(x_dtype)) return bad(op, "x_dtype must be 0 (f32) or 1 (bf16)");
  if (rows <= 0 || k <= 0) return bad(op, "sizes must be positive");
  if (!k_ok(k)) return bad(op, kTooLong);
  if (rows > (1 << 22)) return bad(op, "rows must be at most 2^22");
  if (!x || !row_codes || !row_scales || !col_codes || !col_scales)
    return bad(op, "x, codes and scales must be non-null");
  if (x_stride < 0) return bad(op, "row stride must not be negative");
  if (const char* f = codes_fault(row_codes, row_stride, rows, k)) return bad(op, f);
  if (const char* f = codes_fault(col_codes, col_stride, k, static_cast<int>(rows)))
    return bad(op, f);
  if (const char* f = scales_fault(row_scale_stride, rows, k)) return bad(op, f);
  if (const char* f = scales_fault(col_scale_stride, k, rows)) return bad(op, f);
  mss::QuantBothParams p{};
  p.rows = static_cast<int>(rows); p.k = k;
  p.x = x; p.x_stride = x_stride;
  p.row_codes = static_cast<uint8_t*>(row_codes);
  p.row_scales = static_cast<uint8_t*>(row_scales);
  p.row_stride = row_stride;
  p.col_codes = static_cast<uint8_t*>(col_codes);
  p.col_scales = static_cast<uint8_t*>(col_scales);
  p.col_stride = col_stride;
  p.row_scale_stride = row_scale_stride;
  p.col_scale_stride = col_scale_stride;
  return done(op, mss::launch_quantize_both(p, x_dtype, static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_dequantize_fp8(void* stream, int32_t out_dtype, int64_t rows, int32_t k,
                                   const void* codes, int64_t code_stride, const void* scales,
                                   int64_t scale_stride, void* out) {
  const char* op = "dequantize_fp8";
  if (!dtype_ok(out_dtype)) return bad(op, "out_dtype must be 0 (f32) or 1 (bf16)");
  if (rows <= 0 || k <= 0) return bad(op, "sizes must be positive");
  if (!k_ok(k)) return bad(op, kTooLong);
  if (!codes || !scales || !out) return bad(op, "codes, scales and out must be non-null");
  if (const char* f = codes_fault(codes, code_stride, rows, k)) return bad(op, f);
  if (const char* f = scales_fault(scale_stride, rows, k)) return bad(op, f);
  if (!aligned(out, 16)) return bad(op, "out must be 16-byte aligned");
  mss::DequantParams p{};
  p.rows = rows; p.k = k;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const uint8_t*>(scales);
  p.code_stride = code_stride;
  p.scale_stride = scale_stride;
  p.out = out;
  return done(op, mss::launch_dequantize(p, out_dtype, static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_fp8_matmul(void* stream, int32_t out_dtype, int32_t transposed, int32_t rows_a,
                               int32_t rows_b, int32_t batch, int32_t k, const void* a,
                               int64_t a_stride, const void* a_scales, int64_t a_scale_stride,
                               const void* b, int64_t b_stride, const void* b_scales,
                               int64_t b_scale_stride, void* c) {
  const char* op = "fp8_matmul";
  if (!dtype_ok(out_dtype)) return bad(op, "out_dtype must be 0 (f32) or 1 (bf16)");
  if (rows_a <= 0 || rows_b <= 0 || batch <= 0 || k <= 0)
    return bad(op, "sizes must be positive");
  if (!k_ok(k)) return bad(op, kTooLong);
  if (transposed && batch != 1) return bad(op, "the transposed form takes one batch");
  const int64_t tiles =
      ((static_cast<int64_t>(rows_a) + 127) / 128) * ((static_cast<int64_t>(rows_b) + 63) / 64);
  if (tiles > (1ll << 30) / batch || (transposed && rows_b > 65535 * 16))
    return bad(op, "sizes too large");
  if (!a || !a_scales || !b || !b_scales || !c) return bad(op, "pointers must be non-null");
  if (const char* f = codes_fault(a, a_stride, rows_a, k)) return bad(op, f);
  const int64_t all_b = static_cast<int64_t>(rows_b) * batch;
  if (const char* f = codes_fault(b, b_stride, all_b, k)) return bad(op, f);
  if (const char* f = scales_fault(a_scale_stride, rows_a, k)) return bad(op, f);
  if (const char* f = scales_fault(b_scale_stride, all_b, k)) return bad(op, f);
  mss::Fp8GemmParams p{};
  p.rows_a = rows_a; p.rows_b = rows_b; p.batch = batch; p.k = k;
  p.a = static_cast<const uint8_t*>(a);
  p.b = static_cast<const uint8_t*>(b);
  p.a_stride = a_stride; p.b_stride = b_stride;
  p.a_scale = static_cast<const uint8_t*>(a_scales);
  p.b_scale = static_cast<const uint8_t*>(b_scales);
  p.a_scale_stride = a_scale_stride;
  p.b_scale_stride = b_scale_stride;
  p.c = c;
  p.transposed = transposed != 0;
  p.wait_polls = mss::wait_polls();
  return done(op, mss::launch_fp8_gemm(p, out_dtype, static_cast<cudaStream_t>(stream)));
}

mss_status mamba_ss_sample_tokens(void* stream, int32_t dtype, int32_t rows, int32_t vocab,
                                  const void* logits, int64_t stride, const float* uniform,
                                  const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, float temperature_all,
                                  int32_t top_k_all, float top_p_all, float min_p_all,
                                  int64_t* tokens) {
  const char* op = "sample_tokens";
  if (!dtype_ok(dtype)) return bad(op, "dtype must be 0 (f32) or 1 (bf16)");
  if (rows <= 0 || rows >= (1 << 27)) return bad(op, "rows must be positive and below 2^27");
  if (vocab <= 0 || vocab > mss::kSampleMaxVocab) return bad(op, "vocab must be in 1..360448");
  if (stride < 0) return bad(op, "row stride must not be negative");
  if (!logits || !uniform || !tokens) return bad(op, "logits, uniform and tokens must be non-null");
  mss::SampleParams p{};
  p.rows = rows; p.vocab = vocab;
  p.logits = logits; p.stride = stride;
  p.uniform = uniform;
  p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.temperature_all = temperature_all; p.top_k_all = top_k_all;
  p.top_p_all = top_p_all; p.min_p_all = min_p_all;
  p.tokens = tokens;
  return done(op, mss::launch_sample(p, dtype, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
