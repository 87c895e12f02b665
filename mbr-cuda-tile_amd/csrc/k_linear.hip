// Entry point of the linear layer, and its kernels for f32 operands (linear.hpp).
#include "linear.hpp"

namespace mbrt {
namespace {

// K of nothing: act(bias) + residual, one thread per element.
__global__ __launch_bounds__(256) void linear_empty_kernel(LinArgs a) {
    const int64_t total = a.M * a.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / a.N;
        const int n = (int)(i - m * a.N);
        float v[1] = {0.0f};
        Bias<1> bias;
        bias.load(a, n);
        finish<true, 0, 1>(a, m, n, v, bias);
    }
}

}  // namespace

template int launch_linear<F32>(LinArgs& a, int align, hipStream_t st);
extern template int launch_linear<BF16>(LinArgs& a, int align, hipStream_t st);
extern template int launch_linear<F16>(LinArgs& a, int align, hipStream_t st);
}  // namespace mbrt

using namespace mbrt;

extern "C" {

int mbrt_linear(const void* x, int dtype, int64_t x_row_stride, const void* weight, int64_t weight_row_stride,
                const void* bias, int bias_dtype, const void* residual, int residual_dtype,
                int64_t residual_row_stride, void* out, int out_dtype, int64_t out_row_stride, int64_t rows,
                int64_t in_features, int64_t out_features, int act, mbrt_stream_t stream) {
    const char* op = "mbrt_linear";
    MBRT_REQUIRE_FLOAT_DT(dtype, op);
    MBRT_REQUIRE_FLOAT_DT(out_dtype, op);
    MBRT_REQUIRE(!bias || is_float_dt(bias_dtype), MBRT_E_UNSUPPORTED_DTYPE, "%s: bias dtype %d", op, bias_dtype);
    MBRT_REQUIRE(!residual || is_float_dt(residual_dtype), MBRT_E_UNSUPPORTED_DTYPE, "%s: residual dtype %d", op,
                 residual_dtype);
    MBRT_REQUIRE(act >= MBRT_ACT_NONE && act <= MBRT_ACT_TANH, MBRT_E_INVALID_ARG, "%s: unknown activation %d", op, act);
    MBRT_REQUIRE(rows >= 0 && in_features >= 0 && out_features >= 0, MBRT_E_SHAPE, "%s: negative size", op);
    if (rows == 0 || out_features == 0) return MBRT_OK;
    const int64_t es = dt_size(dtype), lim = int64_t(1) << 28;
    MBRT_REQUIRE(rows < (int64_t(1) << 40) && in_features < lim && out_features < lim, MBRT_E_SHAPE,
                 "%s: size beyond 2^28 features or 2^40 rows", op);
    MBRT_REQUIRE(x_row_stride >= 0 && weight_row_stride >= 0 && (!residual || residual_row_stride >= 0) &&
                     (out_row_stride >= out_features || rows == 1),
                 MBRT_E_SHAPE, "%s: negative row stride, or rows of out that overlap", op);
    MBRT_REQUIRE(out && (in_features == 0 || (x && weight)), MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(x, es) && aligned(weight, es) && aligned(out, dt_size(out_dtype)) &&
                     (!bias || aligned(bias, dt_size(bias_dtype))) &&
                     (!residual || aligned(residual, dt_size(residual_dtype))),
                 MBRT_E_ALIGN, "%s: pointer not aligned to its elements", op);
    LinArgs a{};
    a.x = static_cast<const char*>(x);
    a.w = static_cast<const char*>(weight);
    a.bias = bias;
    a.res = residual;
    a.out = out;
    a.xs = x_row_stride * es;
    a.ws = weight_row_stride * es;
    a.rs = residual_row_stride;
    a.os = out_row_stride;
    a.M = rows;
    a.N = (int)out_features;
    a.K = (int)in_features;
    a.bdt = bias_dtype;
    a.rdt = residual_dtype;
    a.odt = out_dtype;
    a.act = act;
    a.short_act = dtype != F32 && out_dtype != F32;
    hipStream_t st = as_stream(stream);
    if (in_features == 0) {
        hipLaunchKernelGGL(linear_empty_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(rows * out_features, 256), 1 << 16)),
                           dim3(256), 0, st, a);
        return check_launch(op);
    }
    auto rows_at = [&](int64_t bytes) {
        return aligned(x, bytes) && aligned(weight, bytes) && a.xs % bytes == 0 && a.ws % bytes == 0;
    };
    const int align = rows_at(16) ? 16 : rows_at(4) ? 4 : 2;
    const int status = dtype == F32    ? launch_linear<F32>(a, align, st)
                       : dtype == BF16 ? launch_linear<BF16>(a, align, st)
                                       : launch_linear<F16>(a, align, st);
    return status == MBRT_OK ? check_launch(op) : status;
}

}  // extern "C"
