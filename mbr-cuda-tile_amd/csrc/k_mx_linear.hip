// Entry point of the 4-bit linear layer, and its kernels for x in 4 bits (mx_linear.hpp).
#include "mx_linear.hpp"
#include "overlap.hpp"

namespace mbrt {
namespace {

// K of nothing: act(bias) + residual.  A wave per row and 512 columns, 8 in a row of each lane, so that blocks of 32 lie in
// lanes l, l ^ 16, l ^ 32, l ^ 48 as store_mx has them.
__global__ __launch_bounds__(64) void mx_empty_kernel(MxLinArgs a) {
    uint32_t row, part;
    fdivmod(blockIdx.x, a.groups, row, part);
    const int lane = threadIdx.x;
    const int64_t n = (int64_t)part * 512 + 32 * (lane % 16) + 8 * (lane / 16);
    const int at = (int)min(n, (int64_t)a.N + 32);
    float v[8] = {};
    Bias<8> bias;
    bias.load(a, at);
    if (a.odt != MXFP4) finish8<true, false>(a, row, at, v, bias);
    else if (a.short_act != 0) finish8<true, true>(a, row, at, v, bias);
    else finish8<false, true>(a, row, at, v, bias);
}

}  // namespace

template int launch_mx_linear<MXFP4>(MxLinArgs& a, int align, hipStream_t st);
extern template int launch_mx_linear<F32>(MxLinArgs& a, int align, hipStream_t st);
extern template int launch_mx_linear<F16>(MxLinArgs& a, int align, hipStream_t st);
extern template int launch_mx_linear<BF16>(MxLinArgs& a, int align, hipStream_t st);
}  // namespace mbrt

using namespace mbrt;

extern "C" int mbrt_mx_linear(const void* x, int dtype, int64_t x_row_stride, const void* x_scales,
                              int64_t x_scales_row_stride, const void* weight, int64_t weight_row_stride,
                              const void* weight_scales, int64_t weight_scales_row_stride, const void* bias, int bias_dtype,
                              const void* residual, int residual_dtype, int64_t residual_row_stride, void* out,
                              int out_dtype, int64_t out_row_stride, void* out_scales, int64_t out_scales_row_stride,
                              int64_t rows, int64_t in_features, int64_t out_features, int act, mbrt_stream_t stream) {
    const char* op = "mbrt_mx_linear";
    const bool xmx = dtype == MXFP4, omx = out_dtype == MXFP4;
    if (!xmx) MBRT_REQUIRE_FLOAT_DT(dtype, op);
    if (!omx) MBRT_REQUIRE_FLOAT_DT(out_dtype, op);
    MBRT_REQUIRE((!bias || is_float_dt(bias_dtype)) && (!residual || is_float_dt(residual_dtype)), MBRT_E_UNSUPPORTED_DTYPE,
                 "%s: bias dtype %d, residual dtype %d", op, bias_dtype, residual_dtype);
    MBRT_REQUIRE(act >= MBRT_ACT_NONE && act <= MBRT_ACT_TANH, MBRT_E_INVALID_ARG, "%s: unknown activation %d", op, act);
    MBRT_REQUIRE(rows >= 0 && in_features >= 0 && out_features >= 0, MBRT_E_SHAPE, "%s: negative size", op);
    if (rows == 0 || out_features == 0) return MBRT_OK;
    const int64_t lim = int64_t(1) << 28, kb = ceil_div(in_features, kMxBlock), ob = ceil_div(out_features, kMxBlock);
    MBRT_REQUIRE(rows < (int64_t(1) << 40) && in_features < lim && out_features < lim, MBRT_E_SHAPE,
                 "%s: size beyond 2^28 features or 2^40 rows", op);
    const int64_t xe = xmx ? 1 : dt_size(dtype), oe = omx ? 1 : dt_size(out_dtype), ocols = omx ? 16 * ob : out_features;
    if (rows == 1) {  // of a single row: not used
        x_row_stride = x_scales_row_stride = residual_row_stride = 0;
        out_row_stride = ocols;
        out_scales_row_stride = ob;
    }
    if (out_features == 1 || in_features == 0) weight_row_stride = weight_scales_row_stride = 0;
    if (in_features == 0) x_row_stride = x_scales_row_stride = 0;
    MBRT_REQUIRE(x_row_stride >= 0 && weight_row_stride >= 0 && weight_scales_row_stride >= 0 &&
                     (!xmx || x_scales_row_stride >= 0) && (!residual || residual_row_stride >= 0) && out_row_stride >= ocols &&
                     (!omx || out_scales_row_stride >= ob),
                 MBRT_E_SHAPE, "%s: negative row stride, or rows of out that overlap", op);
    MBRT_REQUIRE(out && (!omx || out_scales) && (in_features == 0 || (x && weight && weight_scales && (!xmx || x_scales))),
                 MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(weight, 16) && weight_row_stride % 16 == 0 && (xmx ? aligned(x, 16) && x_row_stride % 16 == 0 : aligned(x, xe)) &&
                     (omx ? aligned(out, 16) && out_row_stride % 16 == 0 : aligned(out, oe)) &&
                     (!bias || aligned(bias, dt_size(bias_dtype))) && (!residual || aligned(residual, dt_size(residual_dtype))),
                 MBRT_E_ALIGN, "%s: pointer not aligned to its elements, or rows of codes not to 16 bytes", op);
    const MemRows O{out, out_row_stride * oe, ocols * oe, rows}, OS{out_scales, out_scales_row_stride, ob, omx ? rows : 0};
    const MemRows in[6] = {{x, x_row_stride * xe, (xmx ? 16 * kb : in_features) * xe, x ? rows : 0},
                           {x_scales, x_scales_row_stride, kb, xmx ? rows : 0},
                           {weight, weight_row_stride, 16 * kb, out_features},
                           {weight_scales, weight_scales_row_stride, kb, out_features},
                           {bias, 0, bias ? out_features * dt_size(bias_dtype) : 0, 1},
                           {residual, residual_row_stride * dt_size(residual_dtype), out_features * dt_size(residual_dtype),
                            residual ? rows : 0}};
    const bool in_place = !omx && residual == out && residual_dtype == out_dtype && (rows == 1 || residual_row_stride == out_row_stride);
    bool clash = rows_meet(O, OS);
    for (int i = 0; i < 6; ++i) clash = clash || (!(i == 5 && in_place) && rows_meet(O, in[i])) || rows_meet(OS, in[i]);
    MBRT_REQUIRE(!clash, MBRT_E_INVALID_ARG,
                 "%s: out overlaps another operand (it may be the residual itself, in the same dtype and rows)", op);
    MxLinArgs a{};
    a.x = static_cast<const char*>(x);
    a.w = static_cast<const char*>(weight);
    a.bias = bias;
    a.res = residual;
    a.out = out;
    a.xs = x_row_stride * xe;
    a.ws = weight_row_stride;
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
    a.wsc = static_cast<const uint8_t*>(weight_scales);
    a.xsc = static_cast<const uint8_t*>(x_scales);
    a.osc = static_cast<uint8_t*>(out_scales);
    a.wss = weight_scales_row_stride;
    a.xss = x_scales_row_stride;
    a.oss = out_scales_row_stride;
    a.nb = (int)kb;
    hipStream_t st = as_stream(stream);
    if (in_features == 0) {
        const int64_t parts = ceil_div(32 * ob, 512);
        MBRT_REQUIRE(grid_fits(rows * parts, 64), MBRT_E_SHAPE, "%s: too many rows", op);
        a.groups = make_fastdiv((uint32_t)parts);
        hipLaunchKernelGGL(mx_empty_kernel, dim3((unsigned)(rows * parts)), dim3(64), 0, st, a);
        return check_launch(op);
    }
    auto rows_at = [&](int64_t bytes) { return aligned(x, bytes) && a.xs % bytes == 0; };
    const int align = rows_at(16) ? 16 : rows_at(4) ? 4 : 2;
    const int status = xmx               ? launch_mx_linear<MXFP4>(a, align, st)
                       : dtype == F32    ? launch_mx_linear<F32>(a, align, st)
                       : dtype == BF16   ? launch_mx_linear<BF16>(a, align, st)
                                         : launch_mx_linear<F16>(a, align, st);
    return status == MBRT_OK ? check_launch(op) : status;
}
