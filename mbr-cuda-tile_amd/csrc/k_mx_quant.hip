// Rows of f32, f16 or bf16 into microscaled 4-bit floats (mx.hpp) and back.
//
// A lane has 8 features of a row: 16 bytes of a 2-byte type, two loads of an f32.  The four lanes of a block agree on its
// scale by two DPP steps, each writes a dword of codes and the first of them the scale.  Both directions move 2.5 (or 4.5)
// bytes per feature and compute next to nothing: memory bounds them.  bf16 [48060, 1536], 187 MB each way, in us with 2, 4
// and 8 pieces under way per lane: quantise 34, 36 and 39, back 36, 37 and 37 (a copy of as many bytes: 37).  A large x is
// read past the caches: quantise 31, and there and back 62 rather than 72, since the codes are still in a cache for the
// second call.  Rows that are not whole 16-byte pieces lose alone what they win in a row of calls: bf16 [12421, 2013]
// 14.7 -> 17.5 alone, 32.6 -> 29.2 there and back.
#include "abi_common.hpp"
#include "mx.hpp"
#include "overlap.hpp"

#include <algorithm>

namespace mbrt {
namespace {

constexpr int kThreads = 256, kUnits = 2;

struct MxRows {
    char* codes;
    uint8_t* scales;
    char* x;
    int64_t cs, ss, xs;  // row strides in bytes
    int64_t rows, total; // pieces of 8 features, those that fill a row's last block included
    int K, pieces;       // features and pieces of a row
    FastDiv per_row;
};

// Pieces of this lane, in rows and places, and the 8 features of each as they stand in memory.
template <int DT>
struct Raw8 {
    u32x4 w[DT == F32 ? 2 : 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (auto& q : w) q = u32x4{0u, 0u, 0u, 0u};
    }
    template <int A, int NT>
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int q = 0; q < (DT == F32 ? 2 : 1); ++q) {
            if constexpr (A == 16) w[q] = gld<NT>(reinterpret_cast<const u32x4*>(p + 16 * q));
            else w[q] = ld_any<NT, A>(p + 16 * q);
        }
    }
    // n < 8 features, zeros behind them
    __device__ __forceinline__ void load_some(const char* p, int n) {
        clear();
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            if (i < n) {
                if constexpr (DT == F32) w[i / 4][i % 4] = reinterpret_cast<const uint32_t*>(p)[i];
                else w[0][i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
            }
        }
    }
    __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == F32) {
                f[i] = __uint_as_float(w[0][i]);
                f[4 + i] = __uint_as_float(w[1][i]);
            } else if constexpr (DT == BF16) {
                f[2 * i] = bf16_lo(w[0][i]);
                f[2 * i + 1] = bf16_hi(w[0][i]);
            } else {
                const f32x2 t = unpack_f16x2(w[0][i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
};

// A: 16 where every piece of x is aligned to 16 bytes and whole, else x's elements.  NT: x is read past the caches.
template <int DT, int A, int NT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(MxRows a) {
    constexpr int S = DT == F32 ? 4 : 2;
    Raw8<DT> v[kUnits];
    uint32_t row[kUnits], place[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t i = ((uint32_t)blockIdx.x * kUnits + u) * kThreads + threadIdx.x;
        fdivmod(min(i, (uint32_t)a.total - 1), a.per_row, row[u], place[u]);
        const char* p = a.x + row[u] * a.xs + (int64_t)place[u] * (8 * S);
        const int left = a.K - 8 * (int)place[u];
        if (left >= 8) v[u].template load<A, NT>(p);
        else if (A == 16) v[u].clear();
        else v[u].load_some(p, left);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        float f[8];
        v[u].values(f);
        uint32_t size = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) size = max(size, mx_size(f[i]));
        const uint32_t code = mx_scale_code(mx_group_size<4>(size));
        const uint32_t w = mx_pack8(f, mx_scale_operand(code));
        const uint32_t i = ((uint32_t)blockIdx.x * kUnits + u) * kThreads + threadIdx.x;
        if (i < (uint32_t)a.total) {
            *reinterpret_cast<uint32_t*>(a.codes + row[u] * a.cs + (int64_t)place[u] * 4) = w;
            if (place[u] % 4 == 0) a.scales[row[u] * a.ss + place[u] / 4] = (uint8_t)code;
        }
    }
}

template <int DT, int A>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(MxRows a) {
    constexpr int S = DT == F32 ? 4 : 2;
    uint32_t w[kUnits], code[kUnits], row[kUnits], place[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t i = ((uint32_t)blockIdx.x * kUnits + u) * kThreads + threadIdx.x;
        fdivmod(min(i, (uint32_t)a.total - 1), a.per_row, row[u], place[u]);
        w[u] = *reinterpret_cast<const uint32_t*>(a.codes + row[u] * a.cs + (int64_t)place[u] * 4);
        code[u] = a.scales[row[u] * a.ss + place[u] / 4];
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t i = ((uint32_t)blockIdx.x * kUnits + u) * kThreads + threadIdx.x;
        if (i >= (uint32_t)a.total) break;
        float f[8];
        mx_unpack8(w[u], mx_scale_operand(code[u]), f);
        char* p = a.x + row[u] * a.xs + (int64_t)place[u] * (8 * S);
        const int left = a.K - 8 * (int)place[u];
        if (left >= 8) {
#pragma unroll
            for (int q = 0; q < (DT == F32 ? 2 : 1); ++q) {
                u32x4 t;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    t[j] = DT == F32    ? __float_as_uint(f[4 * q + j])
                           : DT == BF16 ? pack_bf16x2(f[2 * j], f[2 * j + 1])
                                        : pack_f16x2(f[2 * j], f[2 * j + 1]);
                if constexpr (A == 16) *reinterpret_cast<u32x4*>(p + 16 * q) = t;
                else st_any<0, A>(p + 16 * q, t);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (j < left) st1<DT>(p, j, f[j]);
        }
    }
}

// Calls of more pieces than a launch counts in 32 bits go in several launches of whole rows.
template <class F>
void for_row_ranges(MxRows a, F launch) {
    const int64_t step = std::max<int64_t>(1, (int64_t(1) << 31) / a.pieces);
    for (int64_t r0 = 0, n = a.rows; r0 < n; r0 += step) {
        a.rows = std::min(step, n - r0);
        a.total = a.rows * a.pieces;
        launch(a, dim3((unsigned)ceil_div(a.total, kThreads * kUnits)));
        a.codes += a.rows * a.cs;
        a.scales += a.rows * a.ss;
        a.x += a.rows * a.xs;
    }
}

int mx_convert(const char* op, bool to_codes, char* x, int dt, int64_t xs, char* codes, int64_t cs, uint8_t* scales,
               int64_t ss, int64_t rows, int64_t K, hipStream_t st) {
    MBRT_REQUIRE_FLOAT_DT(dt, op);
    MBRT_REQUIRE(rows >= 0 && K >= 0 && K < (int64_t(1) << 28) && rows < (int64_t(1) << 40), MBRT_E_SHAPE,
                 "%s: negative size, or beyond 2^28 features or 2^40 rows", op);
    if (rows == 0 || K == 0) return MBRT_OK;
    const int64_t es = dt_size(dt), blocks = ceil_div(K, kMxBlock);
    if (rows == 1) xs = K, cs = 16 * blocks, ss = blocks;
    MBRT_REQUIRE(to_codes ? xs >= 0 && cs >= 16 * blocks && ss >= blocks : xs >= K && cs >= 0 && ss >= 0, MBRT_E_SHAPE,
                 "%s: negative row stride, or output rows that overlap", op);
    MBRT_REQUIRE(x && codes && scales, MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(x, es) && aligned(codes, 16) && cs % 16 == 0, MBRT_E_ALIGN,
                 "%s: pointer not aligned to its elements, or rows of codes not to 16 bytes", op);
    const MemRows xr{x, xs * es, K * es, rows}, cr{codes, cs, 16 * blocks, rows}, sr{scales, ss, blocks, rows};
    MBRT_REQUIRE(!rows_meet(xr, cr) && !rows_meet(xr, sr) && !(to_codes && rows_meet(cr, sr)), MBRT_E_INVALID_ARG,
                 "%s: an output overlaps another operand", op);
    MxRows a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.xs = xs * es;
    a.cs = cs;
    a.ss = ss;
    a.rows = rows;
    a.K = (int)K;
    a.pieces = (int)(4 * blocks);
    a.per_row = make_fastdiv((uint32_t)a.pieces);
    const bool al = aligned(x, 16) && a.xs % 16 == 0 && K % 8 == 0;
    const bool cold = cold_input(rows * K * es) != 0;
    with_dt(dt, [&](auto t) {
        constexpr int DT = decltype(t)::value, S = DT == F32 ? 4 : 2;
        for_row_ranges(a, [&](const MxRows& r, dim3 grid) {
            if (to_codes) {
                if (al && cold) hipLaunchKernelGGL((mx_quantize_kernel<DT, 16, 1>), grid, dim3(kThreads), 0, st, r);
                else if (al) hipLaunchKernelGGL((mx_quantize_kernel<DT, 16, 0>), grid, dim3(kThreads), 0, st, r);
                else if (cold) hipLaunchKernelGGL((mx_quantize_kernel<DT, S, 1>), grid, dim3(kThreads), 0, st, r);
                else hipLaunchKernelGGL((mx_quantize_kernel<DT, S, 0>), grid, dim3(kThreads), 0, st, r);
            } else {
                if (al) hipLaunchKernelGGL((mx_dequantize_kernel<DT, 16>), grid, dim3(kThreads), 0, st, r);
                else hipLaunchKernelGGL((mx_dequantize_kernel<DT, S>), grid, dim3(kThreads), 0, st, r);
            }
        });
    });
    return check_launch(op);
}

}  // namespace
}  // namespace mbrt

using namespace mbrt;

extern "C" {

int mbrt_mx_quantize(const void* x, int dtype, int64_t x_row_stride, void* codes, int64_t codes_row_stride, void* scales,
                     int64_t scales_row_stride, int64_t rows, int64_t features, mbrt_stream_t stream) {
    return mx_convert("mbrt_mx_quantize", true, static_cast<char*>(const_cast<void*>(x)), dtype, x_row_stride,
                      static_cast<char*>(codes), codes_row_stride, static_cast<uint8_t*>(scales), scales_row_stride, rows,
                      features, as_stream(stream));
}

int mbrt_mx_dequantize(const void* codes, int64_t codes_row_stride, const void* scales, int64_t scales_row_stride,
                       void* out, int dtype, int64_t out_row_stride, int64_t rows, int64_t features,
                       mbrt_stream_t stream) {
    return mx_convert("mbrt_mx_dequantize", false, static_cast<char*>(out), dtype, out_row_stride,
                      static_cast<char*>(const_cast<void*>(codes)), codes_row_stride,
                      static_cast<uint8_t*>(const_cast<void*>(scales)), scales_row_stride, rows, features,
                      as_stream(stream));
}

}  // extern "C"
