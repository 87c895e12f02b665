// Linear layer of weights in microscaled 4-bit floats (mx.hpp): out[r, n] = act(sum_k x[r, k] w[n, k] + bias[n]) +
// residual[r, n], for x in the same format or in f32, f16 or bf16, and out in any of the four.
//
// x in 4 bits: v_mfma_scale_f32_16x16x128 takes 32 codes of a row per lane (16 bytes, lane l = (g = l / 16, c = l % 16) block
// g of row c) and the scale of that block, so that a block is one piece of 16 bytes on its whole way.  Products are exact,
// sums f32.  Blocks behind a row's last one are whatever the row's last block holds, with scales of 2^-127 on both sides:
// 2^-254 times 36 at most, which leaves an f32 as it is.
//
// x in 16 or 32 bits: a weight below 2^128 (all but the largest under scale bytes 253 and 254, which become infinities) has two
// significant bits and a power of two, so it is exactly a bf16, and x is exactly the sum of
// one (bf16), two (f16) or three (f32) bf16 values, each the leading bits of what the ones before leave.  All of them go
// through the bf16 matrix instructions: nothing is rounded but the f32 sums.
#pragma once

#include "linear.hpp"
#include "mx.hpp"

namespace mbrt {

struct MxLinArgs : LinArgs {  // w, and x and out where they are in 4 bits: codes, rows in bytes
    const uint8_t* wsc;
    const uint8_t* xsc;
    uint8_t* osc;
    int64_t wss, xss, oss;    // row strides of the scales
    int nb;                   // blocks of a row of w
};

// x of dtype XT (MXFP4, F32, F16, BF16).  Instantiated in a source file per dtype.
template <int XT>
int launch_mx_linear(MxLinArgs& a, int align, hipStream_t st);

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mx_mma(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, f32x4 c) {
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

constexpr int mx_parts(int xt) { return xt == F32 ? 3 : xt == F16 ? 2 : 1; }

// The leading 8 significant bits of x as f32, and what they leave (nothing of an infinity; all of a NaN).
__device__ __forceinline__ float split_top(float& x) {
    const float top = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    x = __builtin_fabsf(x) == __builtin_inff() ? 0.0f : x - top;
    return top;
}

// Eight values as bf16, in parts: f[p] holds part p of all of them.
template <int XT>
__device__ __forceinline__ void to_parts(const u32x4 (&raw)[XT == F32 ? 2 : 1], u32x4 (&f)[mx_parts(XT)]) {
    if constexpr (XT == BF16) {
        f[0] = raw[0];
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (XT == F32) {
                v[i] = __uint_as_float(raw[0][i]);
                v[4 + i] = __uint_as_float(raw[1][i]);
            } else {
                const f32x2 t = unpack_f16x2(raw[0][i]);
                v[2 * i] = t.x;
                v[2 * i + 1] = t.y;
            }
        }
#pragma unroll
        for (int p = 0; p < mx_parts(XT); ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = __float_as_uint(split_top(v[2 * i])), hi = __float_as_uint(split_top(v[2 * i + 1]));
                f[p][i] = lo >> 16 | hi;
            }
    }
}

// x Phi(s x) = max(x, 0) - t Phi(-s t), t = |x|, for results in 4 bits.  With r = 1 / (1 + c t), Phi(-s t) is r P(r) 2^(-k t^2): P, of
// degree 7, comes within 2.3e-8 of the scaled function up to s t = 13.2, where Phi leaves f32's normal numbers (and the product is 0
// from there).  In f32 a value is off by at most 2^-23 (0.75 (s x)^2 + 16) of itself, as f32 rounds the argument of an erfc, so a
// block that lies wholly in the tail has the codes that the formula gives it.  12 operations and two transcendental ones ([48060, 384]
// -> 1536 and back 122 us).  A polynomial for log2 Phi alone, 9 and one (117 us), is off by 1.1e-7 at most, but by 2^-12 of the value at
// s x = -5 and by a third of it at -11: of values around -5, 2 in 10^4 then have other codes, and around -11 one in ten.
struct GeluTail {
    float c, k;
};
__device__ __forceinline__ GeluTail gelu_tail_of(int act) {  // s: sqrt 2 in the reference's form, 1 in the other
    return act == MBRT_ACT_GELU_REF ? GeluTail{0.42426407f, 1.44269504f} : GeluTail{0.3f, 0.72134752f};
}
__device__ __forceinline__ float gelu_tail(float x, GeluTail f) {
    const float t = __builtin_fabsf(x);
    const float r = fast_rcp(fmaf(f.c, t, 1.0f));
    float p = fmaf(0.0366180278f, r, -0.161052659f);
    p = fmaf(p, r, 0.212840408f);
    p = fmaf(p, r, -0.0595139973f);
    p = fmaf(p, r, 0.131569877f);
    p = fmaf(p, r, 0.0990252048f);
    p = fmaf(p, r, 0.120892622f);
    p = fmaf(p, r, 0.119620487f);
    const float e = __builtin_amdgcn_exp2f(-(t * f.k) * t);
    return fmaf(-(t * r * p), e, __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff()));  // fmaxf would quiet x first
}

// What a kernel applies to its sums: nothing, GELU in a form for short results, or any function.  What stands behind the sums of a
// tile runs once in a workgroup's life, so that code costs as much to fetch as to run: one that holds every function for all of a lane's
// values takes [17916, 1536] -> 384 from 12.8 to 28.6 us with GELU.
enum MxAct { kActNone = 0, kActGelu = 1, kActAny = 2 };

// OMX: for results in 4 bits.  SHORT: the short forms of the others.
template <int KIND, bool OMX, bool SHORT, int NV>
__device__ __forceinline__ void activate_mx(const MxLinArgs& a, float (&v)[NV]) {
    if constexpr (KIND == kActGelu) {
        if constexpr (OMX) {
            const GeluTail f = gelu_tail_of(a.act);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = gelu_tail(v[i], f);
        } else {
            const float s = a.act == MBRT_ACT_GELU_REF ? 1.0f : 0.70710678118654752440f;
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = gelu_short(v[i], s);
        }
    } else if constexpr (KIND == kActAny) {
        if (OMX && SHORT && (a.act == MBRT_ACT_GELU_REF || a.act == MBRT_ACT_GELU_STD)) activate_mx<kActGelu, true, true>(a, v);
        else activate<NV>(v, a.act, SHORT || a.short_act != 0);
    }
}

// bias, activation and residual of NV consecutive columns n .. of row m, for results that leave in 4 bits: zeros past N.
template <bool SHORT, int NV>
__device__ __forceinline__ void finish_values(const MxLinArgs& a, int64_t m, int n, float (&v)[NV], const Bias<NV>& bias) {
    bias.add_to(a, v);
    activate_mx<kActAny, true, SHORT>(a, v);
    if (a.res != nullptr) {
        const int64_t e = min(m, a.M - 1) * a.rs + n;
        if (n + NV <= a.N) {
            float r[NV];
            load_run<NV>(a.res, a.rdt, e, r);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += r[i];
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (n + i < a.N) v[i] += load1(a.res, a.rdt, e + i);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = n + i < a.N ? v[i] : 0.0f;
}

// Columns n .. n + 7 of row m into 4 bits, n a multiple of 8; the lanes l, l ^ 16, l ^ 32 and l ^ 48 hold a block.  All lanes of
// the wave call this.
__device__ __forceinline__ void store_mx(const MxLinArgs& a, int64_t m, int n, const float (&v)[8]) {
    uint32_t size = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) size = max(size, mx_size(v[i]));
    const uint32_t code = mx_scale_code(mx_rows_size(size));
    if (m < a.M && n < 32 * ((a.N + 31) / 32)) {
        char* out = static_cast<char*>(a.out) + m * a.os;
        *reinterpret_cast<uint32_t*>(out + n / 2) = mx_pack8(v, mx_scale_operand(code));
        if (n % 32 == 0) a.osc[m * a.oss + n / 32] = (uint8_t)code;
    }
}

template <bool SHORT, bool OMX>
__device__ __forceinline__ void finish8(const MxLinArgs& a, int64_t m, int n, float (&v)[8], const Bias<8>& bias) {
    if constexpr (OMX) {
        finish_values<SHORT, 8>(a, m, n, v, bias);
        store_mx(a, m, n, v);
    } else {
        finish<true, 0, 8>(a, m, n, v, bias);
    }
}

// ---- tiles -------------------------------------------------------------------------------------
// WM x WN waves of MI x NI blocks of 16 x 16, w the A operand: lane (g, c) ends with four columns of row c of each block.
// Which columns a block has is free: where results go out in 4 bits (OMX, NI = 8), block ni deals column 32 q + 4 ni + j to its
// row 4 q + j, so that lane (g, c) ends with the 32 columns 32 g .. of its row, a whole block of the format; else 32 (ni / 2) +
// 8 q + 4 (ni % 2) + j, 8 columns in a row for every two blocks.
template <bool OMX>
__device__ __forceinline__ constexpr int tile_col(int ni, int i) {
    return OMX ? 32 * (i >> 2) + 4 * ni + (i & 3) : 32 * (ni / 2) + 8 * (i >> 2) + 4 * (ni % 2) + (i & 3);
}

// LDS rows of SB bytes: piece j of a row stands at j ^ key(row), so that eight neighbouring lanes, which read the same piece of
// eight rows, find them in different banks.  key_c: the key of the row that lane c reads, of x or w.
template <int SB>
__device__ __forceinline__ int tile_key_x(int r) { return SB >= 128 ? r & 7 : (r >> 1) & 3; }
template <int SB, bool OMX>
__device__ __forceinline__ int tile_key_w(int r) {
    const int hi = OMX ? (r >> 5) & 1 : (r >> 3) & 1;
    return SB >= 128 ? (r & 3) | hi << 2 : ((r >> 1) & 1) | hi << 1;
}
template <int SB>
__device__ __forceinline__ int tile_key_c(int c) { return SB >= 128 ? c & 7 : (c >> 1) & 3; }

// The bias is where the sums begin: four columns in one load where all columns of the tile are there (a load for each column
// took [48060, 384] -> 1536 from 40 to 53 us).
template <int MI, int NI, bool OMX>
__device__ __forceinline__ void tile_begin(const MxLinArgs& a, int n0, int g, f32x4 (&acc)[MI][NI]) {
    f32x4 b[NI];
    if (a.bias == nullptr) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) b[ni] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (n0 + NI * 16 <= a.N && a.bdt == F32) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
            b[ni] = __builtin_bit_cast(f32x4, ld_any<0, 4>(static_cast<const float*>(a.bias) + n0 + tile_col<OMX>(ni, 4 * g)));
    } else {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
            for (int j = 0; j < 4; ++j) b[ni][j] = load1(a.bias, a.bdt, min(n0 + tile_col<OMX>(ni, 4 * g) + j, a.N - 1));
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) acc[mi][ni] = b[ni];
}

// Results in 4 bits of a wave's tile at row m, column n.
template <int MI, int KIND, bool SHORT, int NI>
__device__ __forceinline__ void tile_finish_mx(const MxLinArgs& a, int64_t m0, int n0, int g, int c, f32x4 (&acc)[MI][NI]) {
    static_assert(NI == 8, "a lane has a whole block");
    const int n = n0 + 32 * g;
    const bool whole = n0 + 128 <= a.N;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int64_t m = m0 + mi * 16 + c;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = acc[mi][i / 4][i % 4];
        activate_mx<KIND, true, SHORT>(a, v);
        if (a.res != nullptr && n < a.N) {
            const int64_t e = min(m, a.M - 1) * a.rs + n;
            if (n + 32 <= a.N) {
                float r[32];
                load_run<32>(a.res, a.rdt, e, r);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += r[i];
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (n + i < a.N) v[i] += load1(a.res, a.rdt, e + i);
            }
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = n + i < a.N ? v[i] : 0.0f;
        }
        // the largest of them, or NaN if one is: an operation for two values
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i += 2)
            top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, __builtin_fabsf(v[i])), __builtin_fabsf(v[i + 1]));
        const uint32_t code = mx_scale_code(__float_as_uint(__builtin_fabsf(top)));
        if (m < a.M && n < a.N) {
            u32x4 q;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float t[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
                q[i] = mx_pack8(t, mx_scale_operand(code));
            }
            *reinterpret_cast<u32x4*>(static_cast<char*>(a.out) + m * a.os + n / 2) = q;
            a.osc[m * a.oss + n / 32] = (uint8_t)code;
        }
    }
}

// Other results: 16 rows at a time through the wave's own part of LDS (stage: 1 KB per block of 16 columns), from where a
// row's columns go out side by side, whole 128-byte lines at once.  Units of four columns are dealt to even and odd
// halves of an LDS row, and then by its key, which parts neighbouring units; rows eight apart on the way in, and two neighbours on the
// way out, still share their banks (1.15e6 of 7.4e6 LDS cycles of [48060, 384] -> 1536 are conflicts).
template <int MI, int NI, int KIND, int NT>
__device__ __forceinline__ void tile_finish(const MxLinArgs& a, int64_t m0, int n0, int lane, char* stage, f32x4 (&acc)[MI][NI]) {
    constexpr int RB = NI * 64;  // bytes of a staged row
    constexpr int kTurns = KIND == kActNone ? 16 : 1;  // one copy of an activation for all rows of a block
    static_assert(NI == 2 || NI == 4 || NI == 8, "whole rows per access");
    const int g = lane / 16, c = lane % 16;
    auto place = [&](int row, int unit) { return stage + row * RB + 16 * (((unit >> 1) + 2 * NI * (unit & 1)) ^ (row & (2 * NI - 1) & 7)); };
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        asm volatile("" ::: "memory");  // a wave's LDS accesses keep their order, as long as the compiler does
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) *reinterpret_cast<f32x4*>(place(c, tile_col<false>(ni, 4 * g) / 4)) = acc[mi][ni];
        asm volatile("" ::: "memory");
        if (KIND != kActGelu && a.odt == F32) {
            constexpr int LPR = NI * 4, RPI = 64 / LPR;
#pragma unroll kTurns
            for (int k = 0; k < 16 / RPI; ++k) {
                const int r = k * RPI + lane / LPR, u = lane % LPR;
                const f32x4 t = *reinterpret_cast<const f32x4*>(place(r, u));
                float v[4] = {t[0], t[1], t[2], t[3]};
                activate_mx<KIND, false, false>(a, v);
                finish<false, NT, 4>(a, m0 + mi * 16 + r, n0 + 4 * u, v, Bias<4>());
            }
        } else {
            constexpr int LPR = NI * 2, RPI = 64 / LPR;
#pragma unroll kTurns
            for (int k = 0; k < (16 + RPI - 1) / RPI; ++k) {
                const int r = k * RPI + lane / LPR, u = lane % LPR;
                const f32x4 t = *reinterpret_cast<const f32x4*>(place(r, 2 * u)), s = *reinterpret_cast<const f32x4*>(place(r, 2 * u + 1));
                float v[8] = {t[0], t[1], t[2], t[3], s[0], s[1], s[2], s[3]};
                activate_mx<KIND, false, false>(a, v);
                finish<false, NT, 8>(a, m0 + mi * 16 + r, n0 + 8 * u, v, Bias<8>());
            }
        }
    }
}

// x in 4 bits: K in steps of SB bytes (4 or 8 blocks of each row, for one matrix instruction or two) through two LDS buffers filled
// straight from global memory.  Scales come 16 blocks at a time, 16 bytes per row, through registers, and are written to LDS by
// the thread that has the row, in front of the barrier that the step has anyway: of rows that lie 128 bytes apart every load
// fetches a line, and 4 or 8 bytes of it at a time cost as much as the codes ([4096, 4096] -> 4096 64 us).
template <int WM, int WN, int MI, int NI, int SB, int OCC, int NT, int KIND, bool OMX>
__global__ __launch_bounds__(WM * WN * 64, OCC) void mx_tile_kernel(MxLinArgs a) {
    constexpr int NW = WM * WN, BM = WM * MI * 16, BN = WN * NI * 16, NTH = NW * 64, R = BM + BN;
    constexpr int PB = SB / 16, RPL = 1024 / SB, KI = SB / 64;  // pieces of a row, rows of a load, instructions of a step
    constexpr int LX = BM / RPL / NW, LW = BN / RPL / NW, SL = (R + NTH - 1) / NTH;
    static_assert(BM % (RPL * NW) == 0 && BN % (RPL * NW) == 0 && NI % 2 == 0, "whole loads per wave, blocks in pairs");
    static_assert(SB == 64 || SB == 128, "a group of scales is four or two steps");
    constexpr int kBuf = R * SB;
    static_assert(OMX || NW * NI * 1024 <= kBuf, "room for the rows on their way out");
    __shared__ __attribute__((aligned(16))) char s0[kBuf];
    __shared__ __attribute__((aligned(16))) char s1[kBuf];
    // [instruction of a group of four][row], the next group's in the other half; four words between 32 rows and the next, so that
    // lanes that read rows 32 apart do not meet
    constexpr int RS = R + R / 8;
    __shared__ uint32_t sc[2][4 * RS];
    auto scale_at = [](int r) { return r + 4 * (r >> 5); };
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = w / WN, wn = w % WN;
    // column tiles of one row tile are neighbours, on one XCD
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    uint32_t mt, nt;
    fdivmod(tile, a.groups, mt, nt);
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN;
    const char* xb = a.x + m0 * a.xs;
    const char* wb = a.w + (int64_t)n0 * a.ws;
    const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
    const int steps = (a.nb + PB - 1) / PB;

    // lane i of load u covers LDS row RPL (LX w + u) + i / PB, place i % PB; rows past the end repeat the last one, pieces
    // behind a row's end its last one
    uint32_t xo[LX], wo[LW];
    int xp[LX], wp[LW];
#pragma unroll
    for (int u = 0; u < LX; ++u) {
        const int r = RPL * (LX * w + u) + lane / PB;
        xp[u] = (lane % PB) ^ tile_key_x<SB>(r);
        xo[u] = (uint32_t)min(r, mrows - 1) * (uint32_t)a.xs;
    }
#pragma unroll
    for (int u = 0; u < LW; ++u) {
        const int r = RPL * (LW * w + u) + lane / PB;
        wp[u] = (lane % PB) ^ tile_key_w<SB, OMX>(r);
        wo[u] = (uint32_t)min(r, nrows - 1) * (uint32_t)a.ws;
    }
    const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc((void*)xb, (short)0, -1, kBufferDword3);
    const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc((void*)wb, (short)0, -1, kBufferDword3);
    auto load = [&](int kt, char* d) {
        const int last = a.nb - 1 - PB * kt;
#pragma unroll
        for (int u = 0; u < LX; ++u) load_to_lds(xres, d + 1024 * (LX * w + u), xo[u] + 16u * min(xp[u], last), kt * SB);
#pragma unroll
        for (int u = 0; u < LW; ++u) load_to_lds(wres, d + BM * SB + 1024 * (LW * w + u), wo[u] + 16u * min(wp[u], last), kt * SB);
    };
    const uint8_t* sp[SL];
#pragma unroll
    for (int u = 0; u < SL; ++u) {
        const int r = min(tid + u * NTH, R - 1);
        sp[u] = r < BM ? a.xsc + (m0 + min(r, mrows - 1)) * a.xss : a.wsc + (int64_t)(n0 + min(r - BM, nrows - 1)) * a.wss;
    }
    typedef uint32_t any4 __attribute__((aligned(1)));
    typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));
    u32x4 sv[SL];
    auto load_scales = [&](int b0) {  // of 16 blocks, zeros behind a row's end
#pragma unroll
        for (int u = 0; u < SL; ++u) {
            if (b0 + 16 <= a.nb) {
                sv[u] = *reinterpret_cast<const any16*>(sp[u] + b0);
                continue;
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int b = b0 + 4 * s;
                sv[u][s] = 0;
                if (b + 4 <= a.nb) {
                    sv[u][s] = *reinterpret_cast<const any4*>(sp[u] + b);
                } else {
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (b + j < a.nb) sv[u][s] |= (uint32_t)sp[u][b + j] << (8 * j);
                }
            }
        }
    };
    auto put_scales = [&](uint32_t* d) {
#pragma unroll
        for (int u = 0; u < SL; ++u)
            if (tid + u * NTH < R) {
#pragma unroll
                for (int s = 0; s < 4; ++s) d[s * RS + scale_at(tid + u * NTH)] = sv[u][s];
            }
    };

    load(0, s0);
    load_scales(0);
    f32x4 acc[MI][NI];
    tile_begin<MI, NI, OMX>(a, n0 + wn * NI * 16, g, acc);
    const int xrow = wm * MI * 16 + c, wrow = BM + wn * NI * 16;
    auto compute = [&](const char* d, const uint32_t* ds) {
        const uint8_t* scale = reinterpret_cast<const uint8_t*>(ds) + g;
#pragma unroll
        for (int s = 0; s < KI; ++s) {
            if (s > 0) __builtin_amdgcn_sched_barrier(0);  // the second instruction's operands not beside the first's
            u32x4 xf[MI], wf[NI];
            uint32_t xs[MI], ws[NI];
            const int piece = 16 * ((4 * s + g) ^ tile_key_c<SB>(c));
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                const int r = xrow + mi * 16;
                xf[mi] = *reinterpret_cast<const u32x4*>(d + r * SB + piece);
                xs[mi] = scale[(s * RS + scale_at(r)) * 4];
            }
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int r = wrow + tile_col<OMX>(ni, c);
                wf[ni] = *reinterpret_cast<const u32x4*>(d + r * SB + piece);
                ws[ni] = scale[(s * RS + scale_at(r)) * 4];
            }
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mx_mma(wf[ni], ws[ni], xf[mi], xs[mi], acc[mi][ni]);
        }
    };
    // Step kt sits in d, the next one goes to dn, which held the one before; separate objects, and the loop unrolled, so that
    // the compiler sees that loads in flight into one do not touch the other.  I: the step's place in its group of scales, whose
    // first step puts them there and sends for the next ones.
    constexpr int GS = 4 / KI;  // steps of a group
    auto step = [&](int kt, auto place, char* d, char* dn) {
        constexpr int I = decltype(place)::value;
        uint32_t* const ds = sc[(kt / GS) & 1];
        if constexpr (I == 0) {
            put_scales(ds);  // waits for them; this half was last read a group ago
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        wait_loads();
        lds_barrier();  // every wave's loads and scales are there, and none still reads dn
        if (kt + 1 < steps) load(kt + 1, dn);
        if (I == 0 && kt + GS < steps) load_scales((kt + GS) * PB);
        compute(d, ds + I * KI * RS);
    };
    for (int kt = 0; kt < steps; kt += GS) {
        step(kt, std::integral_constant<int, 0>(), s0, s1);
        if (kt + 1 < steps) step(kt + 1, std::integral_constant<int, 1>(), s1, s0);
        if constexpr (GS == 4) {
            if (kt + 2 < steps) step(kt + 2, std::integral_constant<int, 2>(), s0, s1);
            if (kt + 3 < steps) step(kt + 3, std::integral_constant<int, 3>(), s1, s0);
        }
    }

    const int64_t m = m0 + wm * MI * 16;
    const int n = n0 + wn * NI * 16;
    if constexpr (OMX) {
        tile_finish_mx<MI, KIND, true>(a, m, n, g, c, acc);
    } else {
        // the buffer that the last step did not use: no wave reads it any more
        MxLinArgs rest = a;
        rest.bias = nullptr;
        tile_finish<MI, NI, KIND, NT>(rest, m, n, lane, ((steps & 1) != 0 ? s1 : s0) + w * NI * 1024, acc);
    }
}

// x in 16 or 32 bits: steps of FS features; w becomes bf16 and x its parts on their way through registers into LDS, one plane of
// rows per part.  Every load costs the same whatever its width, so a thread takes whole blocks of w, 16 bytes and a scale. Loads of
// three steps are under way while one is computed.  KG groups of waves each take a part of the steps, with buffers of their own, and
// are added in order at the end.  The parts of x meet the same weights.  LDS rows of x: piece j (8 features) at
// j ^ key(row).  Of w: piece 4 b + q of block b at (b + FS / 32 q) ^ key(row), so that the lanes that hold a row's blocks
// write side by side, and rows that are read together, or written, differ in their keys.
template <int FS, bool OMX>
__device__ __forceinline__ int wide_key_w(int r) {
    const int hi = OMX ? (r >> 5) & 1 : (r >> 3) & 1;
    return FS == 128 ? (r & 1) << 2 | hi << 1 | ((r >> 1) & 1) : ((r >> 1) & 1) << 2 | (r & 1) << 1 | hi;
}
template <int FS>
__device__ __forceinline__ int wide_key_c(int c) {  // of the row of w that lane c reads
    return FS == 128 ? (c & 1) << 2 | ((c >> 2) & 1) << 1 | ((c >> 1) & 1) : ((c >> 1) & 1) << 2 | (c & 1) << 1 | ((c >> 2) & 1);
}

template <int XT, int WM, int WN, int MI, int NI, int FS, int KG, int NT, int KIND, bool OMX>
__global__ __launch_bounds__(KG * WM * WN * 64) void mx_wide_tile_kernel(MxLinArgs a) {
    constexpr int NW = WM * WN, NTH = NW * 64, BM = WM * MI * 16, BN = WN * NI * 16, P = mx_parts(XT), Q = XT == F32 ? 2 : 1;
    constexpr int S = XT == F32 ? 4 : 2, PR = FS / 8, BR = FS / 32;     // pieces and blocks of a row's step
    constexpr int LX = BM * PR / NTH, WB = BN * BR, LW = (WB + NTH - 1) / NTH;  // pieces of x and blocks of w for a thread
    static_assert(FS == 64 || FS == 128, "one or two banks' round of a row");
    static_assert(BM * PR % NTH == 0 && NI % 2 == 0, "as much of x for every thread, blocks in pairs");
    constexpr int SB = 2 * FS, kBuf = (BM * P + BN) * SB;
    static_assert(OMX || NW * NI * 1024 <= kBuf, "room for the rows on their way out");
    static_assert(KG == 1 || MI * NI * NW * 1024 <= kBuf, "room for a group's sums");
    __shared__ __attribute__((aligned(16))) char all_lds[KG][2][kBuf];
    const int tid = threadIdx.x % NTH, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NTH);
    auto& lds = all_lds[kg];
    const int wm = w / WN, wn = w % WN;
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    uint32_t mt, nt;
    fdivmod(tile, a.groups, mt, nt);
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN;
    const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
    // a group's whole steps are first .. whole - 1; a step that the rows' end cuts is the last group's
    const int all_whole = a.K / FS, share = (all_whole + KG - 1) / KG, first = min(kg * share, all_whole), whole = min(first + share, all_whole);
    const bool cut = a.K % FS != 0;
    const char* xp[LX];
    const char* wp[LW];
    const uint8_t* sp[LW];
#pragma unroll
    for (int u = 0; u < LX; ++u) xp[u] = a.x + (m0 + min((tid + u * NTH) / PR, mrows - 1)) * a.xs;
#pragma unroll
    for (int u = 0; u < LW; ++u) {
        const int64_t r = n0 + min(min(tid + u * NTH, WB - 1) / BR, nrows - 1);
        wp[u] = a.w + r * a.ws;
        sp[u] = a.wsc + r * a.wss;
    }
    // three steps are on their way at once, each in registers of its own
    struct Regs {
        u32x4 x[LX][Q], w[LW];
        uint32_t scale[LW];
    };
    Regs r0, r1, r2;
    auto load = [&](int kt, Regs& d, auto cut) __attribute__((always_inline)) {
        const int64_t kb = ((int64_t)kt * FS + 8 * (tid % PR)) * S;
#pragma unroll
        for (int u = 0; u < LX; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) d.x[u][q] = cut ? row_piece<XT>(xp[u], kb + 16 * q, a.K) : ld_any<0, S>(xp[u] + kb + 16 * q);
        const int b = kt * BR + tid % BR, at = cut ? min(b, a.nb - 1) : b;  // past the last block, where x is zeros: its codes again
#pragma unroll
        for (int u = 0; u < LW; ++u) {
            d.w[u] = *reinterpret_cast<const u32x4*>(wp[u] + 16 * (int64_t)at);
            d.scale[u] = cut && b >= a.nb ? 0u : sp[u][at];
        }
    };
    auto put = [&](Regs& from, char* d) __attribute__((always_inline)) {
        // nothing is computed from these registers, and so waits for their loads, before this place
#pragma unroll
        for (int u = 0; u < LX; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) asm volatile("" : "+v"(from.x[u][q]));
#pragma unroll
        for (int u = 0; u < LW; ++u) asm volatile("" : "+v"(from.w[u]), "+v"(from.scale[u]));
#pragma unroll
        for (int u = 0; u < LX; ++u) {
            const int r = (tid + u * NTH) / PR;
            u32x4 f[P];
            to_parts<XT>(from.x[u], f);
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<u32x4*>(d + (p * BM + r) * SB + 16 * ((tid % PR) ^ (r & 7))) = f[p];
        }
#pragma unroll
        for (int u = 0; u < LW; ++u) {
            const int r = (tid + u * NTH) / BR, b = tid % BR;
            if (WB % NTH != 0 && r >= BN) break;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<u32x4*>(d + (P * BM + r) * SB + 16 * ((b + BR * q) ^ wide_key_w<FS, OMX>(r))) =
                    mx_unpack8_bf16(from.w[u][q], mx_scale_operand(from.scale[u]));
        }
    };
    auto ready = [&]() {  // the step is in LDS, and none still reads the other buffer; loads may be under way
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        lds_barrier();
    };
    typedef std::integral_constant<bool, false> No;
    typedef std::integral_constant<bool, true> Yes;
    if (first < whole) load(first, r0, No());
    if (first + 1 < whole) load(first + 1, r1, No());
    if (first + 2 < whole) load(first + 2, r2, No());
    f32x4 acc[MI][NI];
    tile_begin<MI, NI, OMX>(a, n0 + wn * NI * 16, g, acc);
    if (KG > 1 && kg > 0) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int xrow = wm * MI * 16 + c, wrow = P * BM + wn * NI * 16;
    auto compute = [&](const char* d) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < FS / 32; ++s) {
            u32x4 wf[NI];
#pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                wf[ni] = *reinterpret_cast<const u32x4*>(d + (wrow + tile_col<OMX>(ni, c)) * SB + 16 * ((s + BR * g) ^ wide_key_c<FS>(c)));
#pragma unroll
            for (int p = P - 1; p >= 0; --p) {
                u32x4 xf[MI];
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
                    xf[mi] = *reinterpret_cast<const u32x4*>(d + (p * BM + xrow + mi * 16) * SB + 16 * ((4 * s + g) ^ (c & 7)));
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma<BF16>(wf[ni], xf[mi], acc[mi][ni]);
            }
        }
    };
    // Step kt, whose registers `mine` are free for step kt + 3; the next one's are `next`.  No condition stands between the loads
    // (the last ones load the last whole step again), so that each wait is for the oldest of them alone.
    auto step = [&](int kt, Regs& mine, Regs& next, auto on) __attribute__((always_inline)) {
        ready();
        if (on) load(min(kt + 3, whole - 1), mine, No());
        compute(lds[(kt - first) & 1]);
        put(next, lds[(kt - first + 1) & 1]);
    };
    if (first < whole) put(r0, lds[0]);
    int kt = first;
    for (; kt + 3 <= whole; kt += 3) {
        step(kt, r0, r1, Yes());
        step(kt + 1, r1, r2, Yes());
        step(kt + 2, r2, r0, Yes());
    }
    if (kt < whole) step(kt, r0, r1, No());
    if (kt + 1 < whole) step(kt + 1, r1, r2, No());
    if (cut && kg == KG - 1) {
        load(whole, r0, Yes());
        ready();  // (what the last step put there in vain is read by none)
        put(r0, lds[(whole - first) & 1]);
        ready();
        compute(lds[(whole - first) & 1]);
    }

    char* stage = lds[(whole - first + (cut ? 1 : 0)) & 1];  // the last step's other buffer: nothing reads it or, behind a cut step, writes it
    if constexpr (KG > 1) {
        // as many barriers for every group; then the other groups' sums, in their order
        for (int i = whole - first + (cut && kg == KG - 1 ? 2 : 0); i < share + (cut ? 2 : 0); ++i) ready();
        ready();
        f32x4* const sums = reinterpret_cast<f32x4*>(all_lds[kg][0]) + w * 64 + lane;
        if (kg > 0) {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) sums[(mi * NI + ni) * NW * 64] = acc[mi][ni];
        }
        ready();
        if (kg > 0) return;
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) acc[mi][ni] += sums[k * (2 * kBuf / 16) + (mi * NI + ni) * NW * 64];
        stage = all_lds[0][0];
    }
    const int64_t m = m0 + wm * MI * 16;
    const int n = n0 + wn * NI * 16;
    if constexpr (OMX) {
        tile_finish_mx<MI, KIND, XT != F32>(a, m, n, g, c, acc);
    } else {
        MxLinArgs rest = a;
        rest.bias = nullptr;
        if constexpr (KG == 1) ready();
        tile_finish<MI, NI, KIND, NT>(rest, m, n, lane, stage + w * NI * 1024, acc);  // a wave's own part
    }
}

// ---- strips ------------------------------------------------------------------------------------
// A wave takes 16 PW columns of out against 16 R rows of x, straight from global memory; `split` waves of a block share the
// blocks of K, four at a time in turn, and are added through LDS in wave order.  PW = 2 deals the columns so that a lane ends
// with 8 in a row, as results in 4 bits need; else 4 in a row.
template <int XT>
struct StripX {  // a lane's block of a row of x
    u32x4 v[XT == MXFP4 ? 1 : XT == F32 ? 8 : 4];
    uint32_t scale;
};

template <int XT, int PW, int R, int A, bool OMX>
__global__ __launch_bounds__(1024) void mx_strip_kernel(MxLinArgs a) {
    constexpr int S = XT == F32 ? 4 : 2, NX = XT == MXFP4 ? 1 : XT == F32 ? 8 : 4;
    extern __shared__ f32x4 part[];  // [strips of the block][split][PW R][64]
    const int lane = threadIdx.x % 64, g = lane / 16, c = lane % 16;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    uint32_t piece, kw, sb, group;
    fdivmod((uint32_t)wv, a.splits, piece, kw);
    const int ks = (int)kw;
    fdivmod(blockIdx.x, a.groups, sb, group);  // the strips of a block are neighbours
    const int64_t p0 = ((int64_t)sb * a.per_block + piece) * 16 * PW, q0 = (int64_t)group * 16 * R;
    const char* wb[PW];
    const uint8_t* ws[PW];
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int64_t col = PW == 2 ? p0 + 8 * (c >> 2) + 4 * p + (c & 3) : p0 + c;
        const int64_t r = min(col, (int64_t)a.N - 1);
        wb[p] = a.w + r * a.ws;
        ws[p] = a.wsc + r * a.wss;
    }
    const char* xb[R];
    const uint8_t* xs[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = min(q0 + 16 * r + c, a.M - 1);
        xb[r] = a.x + row * a.xs;
        xs[r] = XT == MXFP4 ? a.xsc + row * a.xss : nullptr;
    }
    f32x4 acc[PW][R];
#pragma unroll
    for (int p = 0; p < PW; ++p)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[p][r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // U times four blocks, all loads before the first product; CUT: of the last four, some lie behind the row's end or are cut
    // by it
    auto blocks = [&](auto count, auto cut, int t0) {
        constexpr int U = decltype(count)::value;
        constexpr bool CUT = decltype(cut)::value;
        u32x4 wf[U][PW];
        uint32_t wc[U][PW];
        StripX<XT> xf[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = 4 * (t0 + u * a.split) + g, at = CUT ? min(b, a.nb - 1) : b;
            const bool in = !CUT || b < a.nb;
#pragma unroll
            for (int p = 0; p < PW; ++p) {
                wf[u][p] = *reinterpret_cast<const u32x4*>(wb[p] + 16 * (int64_t)at);
                wc[u][p] = in ? ws[p][at] : 0u;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if constexpr (XT == MXFP4) {
                    xf[u][r].v[0] = *reinterpret_cast<const u32x4*>(xb[r] + 16 * (int64_t)at);
                    xf[u][r].scale = in ? xs[r][at] : 0u;
                } else {
#pragma unroll
                    for (int q = 0; q < NX; ++q)
                        xf[u][r].v[q] = CUT ? row_piece<XT>(xb[r], (int64_t)b * 32 * S + 16 * q, a.K)
                                            : load_row<A>(xb[r] + (int64_t)b * 32 * S + 16 * q);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (XT == MXFP4) {
#pragma unroll
                for (int p = 0; p < PW; ++p)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[p][r] = mx_mma(wf[u][p], wc[u][p], xf[u][r].v[0], xf[u][r].scale, acc[p][r]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // 8 of the lane's 32 features
                    u32x4 wbf[PW];
#pragma unroll
                    for (int p = 0; p < PW; ++p) wbf[p] = mx_unpack8_bf16(wf[u][p][q], mx_scale_operand(wc[u][p]));
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        u32x4 raw[XT == F32 ? 2 : 1], f[mx_parts(XT)];
#pragma unroll
                        for (int i = 0; i < (XT == F32 ? 2 : 1); ++i) raw[i] = xf[u][r].v[(XT == F32 ? 2 : 1) * q + i];
                        to_parts<XT>(raw, f);
#pragma unroll
                        for (int i = mx_parts(XT) - 1; i >= 0; --i)
#pragma unroll
                            for (int p = 0; p < PW; ++p) acc[p][r] = mma<BF16>(wbf[p], f[i], acc[p][r]);
                    }
                }
            }
        }
    };
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<bool, false> Whole;
    const int whole = (XT == MXFP4 ? a.nb : a.K / 32) / 4, all = (a.nb + 3) / 4;
    constexpr int U = XT == MXFP4 ? (R * PW >= 4 ? 2 : 4) : R * PW >= 4 || XT == F32 ? 1 : 2;
    int t = ks;
    for (; t + (U - 1) * a.split < whole; t += U * a.split) blocks(std::integral_constant<int, U>(), Whole(), t);
    for (; t < whole; t += a.split) blocks(One(), Whole(), t);
    if (t < all) blocks(One(), std::integral_constant<bool, true>(), t);

    auto finish_all = [&](int r, const f32x4 (&s)[PW]) {
        const int64_t m = q0 + 16 * r + c;
        if constexpr (PW == 2) {
            const int n = (int)min<int64_t>(p0 + 8 * g, (int64_t)a.N + 32);
            Bias<8> bias;
            bias.load(a, n);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = s[i / 4][i % 4];
            finish8<XT != F32, OMX>(a, m, n, v, bias);
        } else {
            const int n = (int)min<int64_t>(p0 + 4 * g, a.N);
            Bias<4> bias;
            bias.load(a, n);
            float v[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
            finish<true, 0, 4>(a, m, n, v, bias);
        }
    };
    if (a.split == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f32x4 s[PW];
#pragma unroll
            for (int p = 0; p < PW; ++p) s[p] = acc[p][r];
            finish_all(r, s);
        }
        return;
    }
    f32x4* mine = part + (int64_t)piece * a.split * PW * R * 64 + lane;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int p = 0; p < PW; ++p) mine[((ks * R + r) * PW + p) * 64] = acc[p][r];
    __syncthreads();
    for (int r = ks; r < R; r += a.split) {
        f32x4 s[PW];
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            s[p] = mine[(r * PW + p) * 64];
            for (int k = 1; k < a.split; ++k) s[p] += mine[((k * R + r) * PW + p) * 64];
        }
        finish_all(r, s);
    }
}

// ---- few rows against many weights -----------------------------------------------------------------
// At most 16 rows of x: what takes time is reading w.  A wave takes 32 columns, dealt so that a lane ends with 8 in a row;
// `split` waves share the K of one such strip, 16 blocks at a time in turn, the scales of a row's 16 in one load.  x stands in
// LDS, as bf16 parts or as its codes, zeros up to whole turns, so that w alone waits for memory: 8 KB a wave, and the next
// turn's as many while one is computed.  Every workgroup has an x of its own, so that a large one leaves a CU room for fewer waves.  Past the caches w comes no faster ([1, 4096] bf16 -> 16384: 10.6 us either way).
template <int XT>
struct TokenX {  // bytes of a row of x in LDS, for a number of blocks
    static constexpr int kBlock = XT == MXFP4 ? 16 : 64;  // a block's codes, or one part of its values
    static __host__ __device__ int64_t row(int64_t blocks) {
        return XT == MXFP4 ? 17 * blocks + 16 - blocks % 16 : 64 * blocks * mx_parts(XT) + 16;
    }
};

template <int XT, bool OMX>
__global__ __launch_bounds__(1024) void mx_token_kernel(MxLinArgs a) {
    constexpr int P = mx_parts(XT), Q = XT == F32 ? 2 : 1, S = XT == F32 ? 4 : 2, PW = 2;
    extern __shared__ __attribute__((aligned(16))) char xl[];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int ks = __builtin_amdgcn_readfirstlane(tid / 64);
    const int turns = (a.nb + 15) / 16, padded = 16 * turns, M = (int)a.M;
    const int rb = (int)TokenX<XT>::row(padded);
    const int64_t p0 = (int64_t)blockIdx.x * 32;
    const char* wb[PW];
    const uint8_t* ws[PW];
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int64_t r = min(p0 + tile_col<false>(p, c), (int64_t)a.N - 1);
        wb[p] = a.w + r * a.ws;
        ws[p] = a.wsc + r * a.wss;
    }
    typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));
    struct Turn {
        u32x4 w[PW][4];
        u32x4 scales[PW];  // byte g of each
    };
    auto load = [&](int t, Turn& d) {  // blocks behind a row's end: its last one, scale 0 (x is zeros there)
#pragma unroll
        for (int p = 0; p < PW; ++p) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                d.w[p][s] = *reinterpret_cast<const u32x4*>(wb[p] + 16 * (int64_t)min(16 * t + 4 * s + g, a.nb - 1));
            if (16 * t + 16 <= a.nb) {
                d.scales[p] = *reinterpret_cast<const any16*>(ws[p] + 16 * t);
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int b = 16 * t + 4 * s + g;
                    d.scales[p][s] = b < a.nb ? (uint32_t)ws[p][b] << (8 * g) : 0u;
                }
            }
        }
    };
    Turn one, two;
    if (ks < turns) load(ks, one);

    if constexpr (XT == MXFP4) {
        for (int i = tid; i < M * padded; i += blockDim.x) {
            const int m = i / padded, b = i - m * padded;
            u32x4 v = {0u, 0u, 0u, 0u};
            uint32_t sc = 0;
            if (b < a.nb) {
                v = *reinterpret_cast<const u32x4*>(a.x + m * a.xs + 16 * (int64_t)b);
                sc = a.xsc[m * a.xss + b];
            }
            *reinterpret_cast<u32x4*>(xl + m * rb + 16 * b) = v;
            xl[m * rb + 16 * padded + b] = (char)sc;
        }
    } else {
        for (int i = tid; i < M * padded * 4; i += blockDim.x) {  // 8 features each
            const int m = i / (4 * padded), e = i - m * 4 * padded;
            const char* row = a.x + m * a.xs;
            u32x4 raw[Q], f[P];
#pragma unroll
            for (int q = 0; q < Q; ++q) raw[q] = row_piece<XT>(row, (int64_t)e * 8 * S + 16 * q, a.K);
            to_parts<XT>(raw, f);
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<u32x4*>(xl + m * rb + p * 64 * padded + 16 * e) = f[p];
        }
    }
    __syncthreads();

    f32x4 acc[PW];
#pragma unroll
    for (int p = 0; p < PW; ++p) acc[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const char* xr = xl + min(c, M - 1) * rb;
    auto compute = [&](int t, const Turn& d) {
        const int b = 16 * t + g;
        if constexpr (XT == MXFP4) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const u32x4 xf = *reinterpret_cast<const u32x4*>(xr + 16 * (b + 4 * s));
                const uint32_t xsc = *reinterpret_cast<const uint8_t*>(xr + 16 * padded + b + 4 * s);
#pragma unroll
                for (int p = 0; p < PW; ++p) acc[p] = mx_mma(d.w[p][s], d.scales[p][s] >> (8 * g), xf, xsc, acc[p]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    u32x4 wf[PW];
#pragma unroll
                    for (int p = 0; p < PW; ++p) wf[p] = mx_unpack8_bf16(d.w[p][s][q], mx_scale_operand(d.scales[p][s] >> (8 * g) & 255u));
#pragma unroll
                    for (int i = P - 1; i >= 0; --i) {
                        const u32x4 xf = *reinterpret_cast<const u32x4*>(xr + i * 64 * padded + 64 * (b + 4 * s) + 16 * q);
#pragma unroll
                        for (int p = 0; p < PW; ++p) acc[p] = mma<BF16>(wf[p], xf, acc[p]);
                    }
                }
        }
    };
    for (int t = ks; t < turns; t += 2 * a.split) {
        if (t + a.split < turns) load(t + a.split, two);
        compute(t, one);
        if (t + a.split < turns) {
            if (t + 2 * a.split < turns) load(t + 2 * a.split, one);
            compute(t + a.split, two);
        }
    }

    f32x4* part = reinterpret_cast<f32x4*>(xl) + lane;
    if (a.split > 1) {
        __syncthreads();  // x is not read any more
#pragma unroll
        for (int p = 0; p < PW; ++p) part[(ks * PW + p) * 64] = acc[p];
        __syncthreads();
        if (ks > 0) return;
#pragma unroll
        for (int p = 0; p < PW; ++p)
            for (int k = 1; k < a.split; ++k) acc[p] += part[(k * PW + p) * 64];
    }
    const int n = (int)min<int64_t>(p0 + 8 * g, (int64_t)a.N + 32);
    Bias<8> bias;
    bias.load(a, n);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = acc[i / 4][i % 4];
    finish8<XT != F32, OMX>(a, c, n, v, bias);
}

template <int XT, int PW, int R, bool OMX>
void launch_mx_strip(const MxLinArgs& a, int align, unsigned blocks, unsigned threads, size_t lds, hipStream_t st) {
    if constexpr (XT == MXFP4) {
        hipLaunchKernelGGL((mx_strip_kernel<XT, PW, R, 16, OMX>), dim3(blocks), dim3(threads), lds, st, a);
    } else if (align == 16) {
        hipLaunchKernelGGL((mx_strip_kernel<XT, PW, R, 16, OMX>), dim3(blocks), dim3(threads), lds, st, a);
    } else if (XT == F32 || align == 4) {
        hipLaunchKernelGGL((mx_strip_kernel<XT, PW, R, 4, OMX>), dim3(blocks), dim3(threads), lds, st, a);
    } else if constexpr (XT != F32) {
        hipLaunchKernelGGL((mx_strip_kernel<XT, PW, R, 2, OMX>), dim3(blocks), dim3(threads), lds, st, a);
    }
}

// SB, OCC: of x in 4 bits (else SB is the features of a step, OCC the groups of waves that share the steps)
template <int XT, int WM, int WN, int MI, int NI, int SB, int OCC, int NT, bool OMX>
int launch_mx_tile(MxLinArgs& a, hipStream_t st) {
    constexpr int BM = WM * MI * 16, BN = WN * NI * 16;
    a.ntiles = (uint32_t)ceil_div(a.N, BN);
    a.groups = make_fastdiv(a.ntiles);
    const int64_t tiles = ceil_div(a.M, BM) * a.ntiles;
    if (!grid_fits(tiles, WM * WN * 64)) return set_error(MBRT_E_SHAPE, "mbrt_mx_linear: too many tiles");
    const dim3 grid((unsigned)tiles), block((XT == MXFP4 ? 1 : OCC) * WM * WN * 64);
    auto launch = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        if constexpr (XT == MXFP4)
            hipLaunchKernelGGL((mx_tile_kernel<WM, WN, MI, NI, SB, OCC, NT, KIND, OMX>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((mx_wide_tile_kernel<XT, WM, WN, MI, NI, SB, OCC, NT, KIND, OMX>), grid, block, 0, st, a);
    };
    const bool gelu = a.act == MBRT_ACT_GELU_REF || a.act == MBRT_ACT_GELU_STD;
    if (a.act == MBRT_ACT_NONE) launch(std::integral_constant<int, kActNone>());
    else if (XT != F32 && gelu && a.short_act != 0) launch(std::integral_constant<int, XT != F32 ? kActGelu : kActAny>());
    else launch(std::integral_constant<int, kActAny>());
    return MBRT_OK;
}

template <int XT, bool OMX>
int launch_mx_shapes(MxLinArgs& a, int align, hipStream_t st) {
    const int64_t cus = cu_count();
    const int64_t cols = ceil_div(a.N, 16), M = a.M, N = a.N;
    // A few rows of x and a strip of 32 columns or more for every CU: x through LDS.  us of this and of strips, 16 waves a CU (8: up to
    // 1.6 more), K -> N: bf16 [1, 4096] -> 16384 10.6 and 13.9, [1, 1536] -> 8192 5.1 and 4.9, [4, 1536] -> 8192 6.3 and 5.3, [4, 4096]
    // -> 16384 12.6 and 16.3; f32 [1, 1536] -> 8192 6.2 and 8.2, [4, 1024] -> 32768 10.5 and 15.9, [8, 1024] -> 32768 19.3 and 16.4;
    // 4 bits [1, 1536] -> 8192 4.4 and 4.9, [16, 4096] -> 16384 10.6 and 17.3.  Where strips are many, a workgroup is one wave, and LDS has
    // room for only four with an x of 33 KB: bf16 [2, 8192] -> 131072 180 and 189, [4, 4096] -> 131072 113 and 108, 4 bits [16, 4096] ->
    // 131072 99 and 118.  With half as many strips as CUs it loses: bf16 and 4 bits [1, 4096] -> 4096 7.2 and 6.2, 6.0 and 5.7.
    const int64_t strips32 = ceil_div(N, 32), turns16 = ceil_div(a.nb, 16), x_row = TokenX<XT>::row(16 * turns16);
    if (M <= (XT == MXFP4 ? 16 : 4) && strips32 >= cus * (XT == BF16 ? std::min<int64_t>(M, 2) : 1) && M * x_row <= (int64_t(1) << 16)) {
        const int64_t room = std::max<int64_t>(1, std::min<int64_t>(16, 16 * cus / strips32));
        a.split = (int)ceil_div(turns16, ceil_div(turns16, room));
        const size_t lds = (size_t)std::max<int64_t>(M * x_row, a.split > 1 ? a.split * 2048 : 0);
        hipLaunchKernelGGL((mx_token_kernel<XT, OMX>), dim3((unsigned)strips32), dim3(64 * a.split), lds, st, a);
        return MBRT_OK;
    }
    // Strips for what gives the CUs no work as tiles, and for 16 rows (a tile has four times as many).  us of strips and of 64 x 64
    // tiles for bf16 and for 4 bits: [256, 1536] -> 384 6.3 and 10.6, 4.5 and 4.8; [32, 4096] -> 4096 13.1 and 21.9, 9.3 and 10.7;
    // [256, 384] -> 1536 6.0 and 5.2, 4.0 and 3.8; [512, 384] -> 1536 7.9 and 5.5, 5.1 and 3.9; [1, 8192] -> 8192 13.8 and 40, 12.7
    // and 18.1.  Two blocks of rows to a wave where that leaves a wave for every CU ([64, 1536] -> 1536 7.0 and 6.6, 5.5 and 5.1;
    // [24, 384] -> 1536 3.0 and 3.3, 2.9 and 3.0); not f32, whose parts fill the registers (10.1 and 12.5).
    const bool far = XT == MXFP4 && (a.xs >= (int64_t(1) << 22) || a.ws >= (int64_t(1) << 22));  // 32-bit offsets in a tile
    if (far || M <= 16 || ceil_div(std::max(M, N), 16) * ceil_div(std::min(M, N), 64) <= cus) {
        constexpr int PW = OMX ? 2 : 1;
        const int64_t strips = ceil_div(cols, PW);
        const int R = XT != F32 && strips * ceil_div(M, 16) > cus && M > 16 ? 2 : 1;
        const int64_t groups = ceil_div(M, 16 * R), turns = ceil_div(a.nb, 4);
        const int64_t room = std::max<int64_t>(1, std::min<int64_t>({16, 64 / (R * PW), 8 * cus / (strips * groups)}));
        a.split = (int)std::max<int64_t>(1, ceil_div(turns, ceil_div(turns, room)));
        a.splits = make_fastdiv((uint32_t)a.split);
        a.per_block = std::max(1, 4 / a.split);
        const int64_t blocks = ceil_div(strips, a.per_block) * groups;
        a.groups = make_fastdiv((uint32_t)groups);
        const unsigned threads = a.per_block * a.split * 64;
        const size_t lds = a.split == 1 ? 0 : (size_t)a.per_block * a.split * R * PW * 1024;
        if (!grid_fits(blocks, threads) || groups >= (int64_t(1) << 31)) return set_error(MBRT_E_SHAPE, "mbrt_mx_linear: too many rows");
        if (R == 1) launch_mx_strip<XT, PW, 1, OMX>(a, align, (unsigned)blocks, threads, lds, st);
        else if constexpr (XT != F32) launch_mx_strip<XT, PW, 2, OMX>(a, align, (unsigned)blocks, threads, lds, st);
        return MBRT_OK;
    }
    // Tiles of 64 x 64 (4-bit results: 64 x 128) or 128 x 128.  us of both: 16- and 32-bit x, where two small ones fill a CU's LDS, bf16
    // [2048, 1536] -> 1536, 192 large tiles, 24.7 and 20.7, [4096, 1536] -> 384, 96, 15.9 and 19.4; 4-bit x [2048, 1536] -> 1536 8.7
    // and 10.9, [4096, 384] -> 1536, 384 tiles, 9.8 and 7.8; both in 4 bits [4096, 384] -> 1536 8.0 and 9.6, [4096, 1536] -> 1536, 384,
    // 14.6 and 14.4, [6144, 1536] -> 1536, 576, 22.9 and 19.7.
    const int64_t tiles = ceil_div(M, 128) * ceil_div(N, 128);
    const bool big = XT != F32 && std::min(M, N) > 64 && (XT != MXFP4 ? 2 * tiles >= cus : OMX ? tiles >= 2 * cus : tiles >= cus);
    const bool nt = !OMX && aligned(a.out, 64) && a.os * dt_size(a.odt) % 64 == 0;
    if constexpr (XT != MXFP4) {
        constexpr int FS = XT == BF16 ? 128 : 64;
        if constexpr (OMX) {
            if (!big) return launch_mx_tile<XT, 4, 1, 1, 8, FS, 1, 0, true>(a, st);
            if constexpr (XT != F32) return launch_mx_tile<XT, 4, 1, 2, 8, 64, 1, 0, true>(a, st);
        } else {
            // At most a tile for every CU, and steps to share: two groups of waves.  us, one and two groups: bf16, f16 and f32 [700, 4096]
            // -> 1024 22.4 and 20.0, 41.9 and 33.1, 58.6 and 45.0; [512, 1536] -> 1536 11.5 and 11.3, 18.7 and 16.2, 25.0 and 20.8; [512,
            // 384] -> 1536, 3 steps of bf16 and 6 of the others, 5.5 and 5.7, 7.4 and 7.2, 9.4 and 8.9.
            if (!big && a.K >= 6 * FS && ceil_div(M, 64) * ceil_div(N, 64) <= cus) return launch_mx_tile<XT, 2, 2, 2, 2, FS, 2, 0, false>(a, st);
            if (!big) return launch_mx_tile<XT, 2, 2, 2, 2, FS, 1, 0, false>(a, st);
            if constexpr (XT != F32)
                return nt ? launch_mx_tile<XT, 2, 2, 4, 4, 64, 1, 2, false>(a, st) : launch_mx_tile<XT, 2, 2, 4, 4, 64, 1, 0, false>(a, st);
        }
        return MBRT_OK;
    } else if constexpr (OMX) {
        // steps of 64 bytes leave room for three workgroups to a CU, of 128 for two ([24000, 1536] -> 1536 55 and 57 us)
        return big ? launch_mx_tile<XT, 4, 1, 2, 8, 64, 3, 0, true>(a, st) : launch_mx_tile<XT, 4, 1, 1, 8, 64, 3, 0, true>(a, st);
    } else {
        if (!big) return launch_mx_tile<XT, 2, 2, 2, 2, 128, 4, 0, false>(a, st);
        // Long K: 256 x 256, which asks L2 and LDS for half as much per product, if four fifths of what the CUs then compute is wanted.  us
        // of 128 x 128 and of these: [4096, 4096] -> 4096, all of it wanted, 62 and 42; [24000, 1536] -> 1152, 83 %, 41 and 37, -> 1536,
        // 73 %, 48 and 55; [48060, 1536] -> 1536, 87 %, 92 and 93, -> 384, 55 %, 29 and 36; [48060, 384] -> 1536 41 and 54.
        const int64_t tiles256 = ceil_div(M, 256) * ceil_div(N, 256);
        if (a.nb >= 48 && 5.0 * (double)M * (double)N >= 4.0 * 65536.0 * (double)(ceil_div(tiles256, cus) * cus))
            return nt ? launch_mx_tile<XT, 2, 4, 8, 4, 128, 2, 2, false>(a, st) : launch_mx_tile<XT, 2, 4, 8, 4, 128, 2, 0, false>(a, st);
        // (steps of 128 bytes: [48060, 384] -> 1536 53 for 41, [24000, 4096] -> 1536 105 for 114)
        return nt ? launch_mx_tile<XT, 2, 2, 4, 4, 64, 3, 2, false>(a, st) : launch_mx_tile<XT, 2, 2, 4, 4, 64, 3, 0, false>(a, st);
    }
}

}  // namespace

template <int XT>
int launch_mx_linear(MxLinArgs& a, int align, hipStream_t st) {
    return a.odt == MXFP4 ? launch_mx_shapes<XT, true>(a, align, st) : launch_mx_shapes<XT, false>(a, align, st);
}

}  // namespace mbrt
