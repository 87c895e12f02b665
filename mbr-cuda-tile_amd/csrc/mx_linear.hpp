// Linear layer of weights in microscaled 4-bit floats (mx.hpp): out[r, n] = act(sum_k x[r, k] w[n, k] + bias[n]) +
// residual[r, n], for x in the same format or in f32, f16 or bf16, and out in any of the four.
//
// x in 4 bits: v_mfma_scale_f32_16x16x128 takes 32 codes of a row per lane (16 bytes, lane l = (g = l / 16, c = l % 16) block
// g of row c) and the scale of that block, so that a block is one piece of 16 bytes on its whole way.  Products are exact,
// sums f32.  Blocks behind a row's last one are whatever the row's last block holds, with scales of 2^-127 on both sides:
// 2^-254 times 36 at most, which leaves an f32 as it is.
//
// x in 16 or 32 bits: a weight has two significant bits and a power of two, so it is exactly a bf16, and x is exactly the sum of
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
    int rows_outer;           // strips: groups of x rows are the slower index
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

// bias, activation and residual of NV consecutive columns n .. of row m, for results that leave in 4 bits: zeros past N.
template <bool ACT, int NV>
__device__ __forceinline__ void finish_values(const MxLinArgs& a, int64_t m, int n, float (&v)[NV], const Bias<NV>& bias) {
    bias.add_to(a, v);
    if constexpr (ACT) activate<NV>(v, a.act, a.short_act != 0);
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

template <bool ACT, bool OMX, int NT>
__device__ __forceinline__ void finish8(const MxLinArgs& a, int64_t m, int n, float (&v)[8], const Bias<8>& bias) {
    if constexpr (OMX) {
        finish_values<ACT, 8>(a, m, n, v, bias);
        store_mx(a, m, n, v);
    } else {
        finish<ACT, NT, 8>(a, m, n, v, bias);
    }
}

// ---- tiles, x in 4 bits ------------------------------------------------------------------------
// As linear_tile_kernel: WM x WN waves of MI x NI blocks of 16 x 16, K in steps of 128 bytes (8 blocks, two matrix
// instructions) of every row through two LDS buffers filled straight from global memory, LDS rows of 8 pieces at j ^ key(row),
// w the A operand with columns dealt so that a lane ends with 8 in a row.  The scales of a step, 8 bytes per row, come
// through registers and are written to LDS by the thread that has the row, in front of the barrier that the step has anyway.
template <int WM, int WN, int MI, int NI, int NT, bool ACT, bool OMX>
__global__ __launch_bounds__(WM * WN * 64) void mx_tile_kernel(MxLinArgs a) {
    constexpr int NW = WM * WN, BM = WM * MI * 16, BN = WN * NI * 16, NTH = NW * 64;
    constexpr int LX = BM / 8 / NW, LW = BN / 8 / NW, SL = (BM + BN + NTH - 1) / NTH;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NI % 2 == 0, "whole loads per wave, blocks in pairs");
    constexpr int SB = kStepBytes, kBuf = (BM + BN) * SB;
    __shared__ __attribute__((aligned(16))) char s0[kBuf];
    __shared__ __attribute__((aligned(16))) char s1[kBuf];
    __shared__ __attribute__((aligned(8))) uint8_t c0[(BM + BN) * 8];
    __shared__ __attribute__((aligned(8))) uint8_t c1[(BM + BN) * 8];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = w / WN, wn = w % WN;
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    uint32_t mt, nt;
    fdivmod(tile, a.groups, mt, nt);
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN;
    const char* xb = a.x + m0 * a.xs;
    const char* wb = a.w + (int64_t)n0 * a.ws;
    const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
    const int steps = (a.nb + 7) / 8;

    int xr[LX], wr[LW];
#pragma unroll
    for (int u = 0; u < LX; ++u) xr[u] = min(8 * (LX * w + u) + lane / 8, mrows - 1);
#pragma unroll
    for (int u = 0; u < LW; ++u) wr[u] = min(8 * (LW * w + u) + lane / 8, nrows - 1);
    const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc((void*)xb, (short)0, -1, kBufferDword3);
    const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc((void*)wb, (short)0, -1, kBufferDword3);
    // pieces behind a row's end: its last one
    auto load = [&](int kt, char* d) {
        const int last = a.nb - 1 - 8 * kt;
#pragma unroll
        for (int u = 0; u < LX; ++u)
            load_to_lds(xres, d + 1024 * (LX * w + u),
                        (uint32_t)xr[u] * (uint32_t)a.xs + 16u * min((lane % 8) ^ key_x(8 * (LX * w + u) + lane / 8), last), kt * SB);
#pragma unroll
        for (int u = 0; u < LW; ++u)
            load_to_lds(wres, d + BM * SB + 1024 * (LW * w + u),
                        (uint32_t)wr[u] * (uint32_t)a.ws + 16u * min((lane % 8) ^ key_w(8 * (LW * w + u) + lane / 8), last), kt * SB);
    };
    const uint8_t* sp[SL];
#pragma unroll
    for (int u = 0; u < SL; ++u) {
        const int r = min(tid + u * NTH, BM + BN - 1);
        sp[u] = r < BM ? a.xsc + (m0 + min(r, mrows - 1)) * a.xss : a.wsc + (int64_t)(n0 + min(r - BM, nrows - 1)) * a.wss;
    }
    typedef uint32_t any8 __attribute__((ext_vector_type(2), aligned(1)));
    u32x2 sv[SL];
    auto load_scales = [&](int kt) {
        const int left = a.nb - 8 * kt;
#pragma unroll
        for (int u = 0; u < SL; ++u) {
            if (left >= 8) {
                sv[u] = *reinterpret_cast<const any8*>(sp[u] + 8 * kt);
            } else {
                sv[u] = u32x2{0u, 0u};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (j < left) sv[u][j / 4] |= (uint32_t)sp[u][8 * kt + j] << (8 * (j % 4));
            }
        }
    };
    auto put_scales = [&](uint8_t* d) {
#pragma unroll
        for (int u = 0; u < SL; ++u)
            if (tid + u * NTH < BM + BN) *reinterpret_cast<u32x2*>(d + 8 * (tid + u * NTH)) = sv[u];
    };

    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int xrow = wm * MI * 16 + c, wrow = BM + wn * NI * 16 + 8 * (c >> 2) + (c & 3);
    auto compute = [&](const char* d, const uint8_t* ds) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int piece = 16 * ((4 * s + g) ^ (c & 7));
            u32x4 xf[MI], wf[NI];
            uint32_t xs[MI], ws[NI];
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                xf[mi] = *reinterpret_cast<const u32x4*>(d + (xrow + mi * 16) * SB + piece);
                xs[mi] = ds[(xrow + mi * 16) * 8 + 4 * s + g];
            }
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                wf[ni] = *reinterpret_cast<const u32x4*>(d + (wrow + 32 * (ni / 2) + 4 * (ni % 2)) * SB + piece);
                ws[ni] = ds[(wrow + 32 * (ni / 2) + 4 * (ni % 2)) * 8 + 4 * s + g];
            }
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mx_mma(wf[ni], ws[ni], xf[mi], xs[mi], acc[mi][ni]);
        }
    };
    auto step = [&](int kt, char* d, uint8_t* ds, char* dn) {
        put_scales(ds);  // waits for them; the buffer was last read two steps ago
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_loads();
        lds_barrier();   // every wave's loads and scales are there, and none still reads dn
        if (kt + 1 < steps) {
            load(kt + 1, dn);
            load_scales(kt + 1);
        }
        compute(d, ds);
    };
    load(0, s0);
    load_scales(0);
    for (int kt = 0; kt < steps; kt += 2) {
        step(kt, s0, c0, s1);
        if (kt + 1 < steps) step(kt + 1, s1, c1, s0);
    }

    const int n = n0 + wn * NI * 16 + 8 * g;
    Bias<8> bias[NI / 2];
#pragma unroll
    for (int p = 0; p < NI / 2; ++p) bias[p].load(a, n + 32 * p);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int p = 0; p < NI / 2; ++p) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[mi][2 * p + i / 4][i % 4];
            finish8<ACT, OMX, NT>(a, m0 + wm * MI * 16 + mi * 16 + c, n + 32 * p, v, bias[p]);
        }
}

// ---- tiles, x in 16 or 32 bits -------------------------------------------------------------------
// Steps of 64 features: w becomes bf16 and x its parts on their way through registers into LDS, one plane of 128-byte rows
// per part.  The next step's loads are under way while one is computed.  The parts of x meet the same weights.
template <int XT, int WM, int WN, int MI, int NI, int NT, bool ACT, bool OMX>
__global__ __launch_bounds__(WM * WN * 64) void mx_wide_tile_kernel(MxLinArgs a) {
    constexpr int NW = WM * WN, BM = WM * MI * 16, BN = WN * NI * 16, P = mx_parts(XT), Q = XT == F32 ? 2 : 1;
    constexpr int LX = BM / 8 / NW, LW = BN / 8 / NW, S = XT == F32 ? 4 : 2;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NI % 2 == 0, "whole loads per wave, blocks in pairs");
    constexpr int SB = 128, kBuf = (BM * P + BN) * SB;
    __shared__ __attribute__((aligned(16))) char lds[2][kBuf];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = w / WN, wn = w % WN;
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    uint32_t mt, nt;
    fdivmod(tile, a.groups, mt, nt);
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN;
    const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
    const int steps = (a.K + 63) / 64;
    const char* xp[LX];
    const char* wp[LW];
    const uint8_t* sp[LW];
#pragma unroll
    for (int u = 0; u < LX; ++u) xp[u] = a.x + (m0 + min(8 * (LX * w + u) + lane / 8, mrows - 1)) * a.xs;
#pragma unroll
    for (int u = 0; u < LW; ++u) {
        const int64_t r = n0 + min(8 * (LW * w + u) + lane / 8, nrows - 1);
        wp[u] = a.w + r * a.ws;
        sp[u] = a.wsc + r * a.wss;
    }
    u32x4 px[LX][Q];
    uint32_t pw[LW], ps[LW];
    const int64_t kbytes = (int64_t)a.K * S;
    auto load = [&](int kt) {
        // lane's piece: features 64 kt + 8 j of its row, j = lane % 8 (placed at j ^ key in LDS)
        const int j = lane % 8;
        const int64_t kb = ((int64_t)kt * 64 + 8 * j) * S;
        const bool whole = ((int64_t)kt + 1) * 64 * S <= kbytes;
#pragma unroll
        for (int u = 0; u < LX; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) px[u][q] = whole ? ld_any<0, S>(xp[u] + kb + 16 * q) : row_piece<XT>(xp[u], kb + 16 * q, a.K);
        const int b = min(2 * kt + j / 4, a.nb - 1);  // past the last block, where x is zeros: its codes again
#pragma unroll
        for (int u = 0; u < LW; ++u) {
            pw[u] = *reinterpret_cast<const uint32_t*>(wp[u] + 16 * (int64_t)b + 4 * (j % 4));
            ps[u] = 2 * kt + j / 4 < a.nb ? sp[u][b] : 0u;
        }
    };
    auto put = [&](char* d) {
#pragma unroll
        for (int u = 0; u < LX; ++u) {
            const int r = 8 * (LX * w + u) + lane / 8;
            u32x4 f[P];
            to_parts<XT>(px[u], f);
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<u32x4*>(d + (p * BM + r) * SB + 16 * ((lane % 8) ^ key_x(r))) = f[p];
        }
#pragma unroll
        for (int u = 0; u < LW; ++u) {
            const int r = 8 * (LW * w + u) + lane / 8;
            *reinterpret_cast<u32x4*>(d + (P * BM + r) * SB + 16 * ((lane % 8) ^ key_w(r))) =
                mx_unpack8_bf16(pw[u], mx_scale_operand(ps[u]));
        }
    };
    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int xrow = wm * MI * 16 + c, wrow = P * BM + wn * NI * 16 + 8 * (c >> 2) + (c & 3);
    auto compute = [&](const char* d) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int piece = 16 * ((4 * s + g) ^ (c & 7));
            u32x4 wf[NI];
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) wf[ni] = *reinterpret_cast<const u32x4*>(d + (wrow + 32 * (ni / 2) + 4 * (ni % 2)) * SB + piece);
#pragma unroll
            for (int p = P - 1; p >= 0; --p) {
                u32x4 xf[MI];
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) xf[mi] = *reinterpret_cast<const u32x4*>(d + (p * BM + xrow + mi * 16) * SB + piece);
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma<BF16>(wf[ni], xf[mi], acc[mi][ni]);
            }
        }
    };
    load(0);
    put(lds[0]);
    for (int kt = 0; kt < steps; ++kt) {
        __syncthreads();  // the step is in LDS, and none still reads the other buffer
        if (kt + 1 < steps) load(kt + 1);
        compute(lds[kt & 1]);
        if (kt + 1 < steps) put(lds[(kt + 1) & 1]);
    }

    const int n = n0 + wn * NI * 16 + 8 * g;
    Bias<8> bias[NI / 2];
#pragma unroll
    for (int p = 0; p < NI / 2; ++p) bias[p].load(a, n + 32 * p);
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int p = 0; p < NI / 2; ++p) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[mi][2 * p + i / 4][i % 4];
            finish8<ACT, OMX, NT>(a, m0 + wm * MI * 16 + mi * 16 + c, n + 32 * p, v, bias[p]);
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
    // strips (of columns) of a block are neighbours; a.groups counts the faster index
    if (a.rows_outer) {
        uint32_t s;
        fdivmod(blockIdx.x, a.groups, group, s);
        sb = s;
    } else {
        fdivmod(blockIdx.x, a.groups, sb, group);
    }
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
            finish8<true, OMX, 0>(a, m, n, v, bias);
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

template <int XT, int WM, int WN, int MI, int NI, int NT, bool OMX>
int launch_mx_tile(MxLinArgs& a, hipStream_t st) {
    constexpr int BM = WM * MI * 16, BN = WN * NI * 16;
    a.ntiles = (uint32_t)ceil_div(a.N, BN);
    a.groups = make_fastdiv(a.ntiles);
    const int64_t tiles = ceil_div(a.M, BM) * a.ntiles;
    if (!grid_fits(tiles, WM * WN * 64)) return set_error(MBRT_E_SHAPE, "mbrt_mx_linear: too many tiles");
    const dim3 grid((unsigned)tiles), block(WM * WN * 64);
    auto launch = [&](auto act) {
        constexpr bool ACT = decltype(act)::value;
        if constexpr (XT == MXFP4)
            hipLaunchKernelGGL((mx_tile_kernel<WM, WN, MI, NI, NT, ACT, OMX>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((mx_wide_tile_kernel<XT, WM, WN, MI, NI, NT, ACT, OMX>), grid, block, 0, st, a);
    };
    if (a.act != MBRT_ACT_NONE) launch(std::integral_constant<bool, true>());
    else launch(std::integral_constant<bool, false>());
    return MBRT_OK;
}

template <int XT, bool OMX>
int launch_mx_shapes(MxLinArgs& a, int align, hipStream_t st) {
    const int64_t cus = cu_count();
    const int64_t cols = ceil_div(a.N, 16), rows = ceil_div(a.M, 16);
    // 32-bit offsets within a tile
    const bool far = XT == MXFP4 && (a.xs >= (int64_t(1) << 22) || a.ws >= (int64_t(1) << 22));
    if (far || ceil_div(std::max(a.M, (int64_t)a.N), 16) * ceil_div(std::min(a.M, (int64_t)a.N), 64) <= cus ||
        std::min(a.M, (int64_t)a.N) <= 16) {
        constexpr int PW = OMX ? 2 : 1;
        const int64_t strips = ceil_div(cols, PW);
        int R = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
        while (R > 1 && strips * ceil_div(a.M, 8 * R) <= cus) R /= 2;
        const int64_t groups = ceil_div(a.M, 16 * R), turns = ceil_div(a.nb, 4);
        const int64_t room = std::max<int64_t>(1, std::min<int64_t>({16, 64 / (R * PW), 8 * cus / (strips * groups)}));
        a.split = (int)std::max<int64_t>(1, ceil_div(turns, ceil_div(turns, room)));
        a.splits = make_fastdiv((uint32_t)a.split);
        a.per_block = std::max(1, 4 / a.split);
        const int64_t sblocks = ceil_div(strips, a.per_block), blocks = sblocks * groups;
        a.rows_outer = a.M > a.N;
        a.groups = make_fastdiv((uint32_t)(a.rows_outer ? sblocks : groups));
        const unsigned threads = a.per_block * a.split * 64;
        const size_t lds = a.split == 1 ? 0 : (size_t)a.per_block * a.split * R * PW * 1024;
        if (!grid_fits(blocks, threads) || groups >= (int64_t(1) << 31)) return set_error(MBRT_E_SHAPE, "mbrt_mx_linear: too many rows");
        if (R == 1) launch_mx_strip<XT, PW, 1, OMX>(a, align, (unsigned)blocks, threads, lds, st);
        else if (R == 2) launch_mx_strip<XT, PW, 2, OMX>(a, align, (unsigned)blocks, threads, lds, st);
        else launch_mx_strip<XT, PW, 4, OMX>(a, align, (unsigned)blocks, threads, lds, st);
        return MBRT_OK;
    }
    const bool big = XT != F32 && std::min(a.M, (int64_t)a.N) > 64 && ceil_div(a.M, 128) * ceil_div(a.N, 128) >= cus;
    if (!big) return launch_mx_tile<XT, 2, 2, 2, 2, 0, OMX>(a, st);
    if constexpr (XT != F32) {
        const bool nt = !OMX && aligned(a.out, 64) && a.os * dt_size(a.odt) % 64 == 0;
        if constexpr (!OMX) {
            if (nt) return launch_mx_tile<XT, 2, 2, 4, 4, 2, OMX>(a, st);
        }
        return launch_mx_tile<XT, 2, 2, 4, 4, 0, OMX>(a, st);
    }
    return MBRT_OK;
}

}  // namespace

template <int XT>
int launch_mx_linear(MxLinArgs& a, int align, hipStream_t st) {
    return a.odt == MXFP4 ? launch_mx_shapes<XT, true>(a, align, st) : launch_mx_shapes<XT, false>(a, align, st);
}

}  // namespace mbrt
