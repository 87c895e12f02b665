// Linear layer with its epilogue: out[r, n] = act(sum_k x[r, k] w[n, k] + bias[n]) + residual[r, n],
// the projections of the band-split transformer (src/mbr_cuda_tile.cu:712-3790) with the epilogues they
// end in there (bias, GELU, sigmoid, tanh) and the residual add.
//
// Both operands hold their contraction index last, so a 16-byte piece of a row of either is what one
// lane feeds to a matrix instruction: lane l = (g = l / 16, c = l % 16) takes bytes 16 g .. of a 64-byte
// piece of row c.  For 2-byte types that is one v_mfma_f32_16x16x32 (k = 8 g + j); for f32 four
// v_mfma_f32_16x16x4_f32, the j-th over the j-th element of every lane's four (k = 4 g + j): any order of the
// contraction serves if both operands have the same.  Sums are f32; the epilogue works in f32 and rounds once,
// on its store.
//
// Forms, by shape (launch_linear below): tiles of 64 x 64 up to 128 x 192 through LDS, whose groups of waves share the
// steps where tiles are few, and strips of 16 rows of the longer operand against all of a short one.
//
// What bounds it (MI355X, us; a large copy runs at 4.8 TB/s, a large library product at 1382 TFLOP/s, f32 153):
//   [48060, 384] -> 1536 bf16 67 (184 MB: 41 at the copy's rate; 844 TFLOP/s).  Stores first: 8 bytes per lane and through the
//   caches 99, 16 bytes 74, out past the caches 70; 204 MB are written for 148 MB of out (counted).  The matrix units are busy for
//   28 of it, and a product's end and the next one's first loads overlap only between the two workgroups of a CU.  With bias and
//   GELU 104 to 109: the epilogue's 20 VALU operations an element have only the other workgroup to hide behind.
//   [48060, 1536] -> 384 with residual 93 (221 MB: 46): 176 MB are read in the order in which tiles ask for them, two column tiles
//   the same rows of x, and every step ends with no load under way; the loads alone take nearly as long.  The library's product
//   alone 93 and, of the former, 120.
//   f32 [4096, 4096] -> 4096 960: 143 TFLOP/s.  One row to some hundred: the launch, and the latency of one round of loads (4.1).
// Not kept, with the times of these two: steps of 64 bytes in four buffers (no gain), 192 x 192 in three buffers (110; 88 to 90,
// less than the 93, but a form of its own for long K alone), 256 x 256 (86 and 109), persistent workgroups that store while the
// next tile loads (74 to 85; 88), fragments fetched across the barrier (no gain), rows handed round through LDS for stores of whole
// lines (67 -> 79).
#pragma once

#include "abi_common.hpp"

#include <algorithm>

namespace mbrt {

struct LinArgs {
    const char* x;
    const char* w;
    const void* bias;
    const void* res;
    void* out;
    int64_t xs, ws, rs, os;  // row strides: bytes (x, w), elements (residual, out)
    int64_t M;
    int N, K;
    int bdt, rdt, odt, act;
    int short_act;           // activations by their short forms
    uint32_t ntiles;         // tiles along N
    int split;               // strips: waves that share a strip's K
    int per_block;           // strips of a block
    FastDiv groups, splits;  // ntiles and split
};

// The linear layer for operands of one dtype; align: all rows of x and w begin at multiples of it, 16, 4 or 2
// bytes.  Instantiated in a source file per dtype.
template <int DT>
int launch_linear(LinArgs& a, int align, hipStream_t st);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;            // of every row, per step of the tile form
constexpr int kBufferDword3 = 0x00020000;  // raw buffer resource: 32-bit data format, no swizzle, no stride

// 16 bytes per lane from base + off + step straight to lds + 16 lane.  Not a template: the builtin's operands must not
// depend on one, or the host pass drops the kernel that holds it.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t base, char* lds, uint32_t off, int step) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_void*)lds, 16, off, step, 0, 0);
}

// Until this wave's loads have landed and its LDS accesses are done (vmcnt and lgkmcnt 0).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0070); }

// A barrier without the fence of __syncthreads(), which would wait for every load under way: LDS accesses stay
// on their side of it, and the caller has waited for its own.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int DT>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (DT == F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], c, 0, 0, 0);
        return c;
    }
}

// 16 bytes of a row at a multiple of A bytes: 16, 4 or 2.  Loads at odd multiples of 2 are several times slower than others,
// so with A = 2 they come as the 20 bytes around them, moved down: the dwords at both ends hold an element of the 16 bytes
// each, and nothing outside these dwords is read ([48060, 385] -> 8 in strips 25.8 -> 14.4 us, [60, 385] -> 1536 7.9 -> 4.7; with A = 4
// the fifth dword costs: [20000, 500] -> 48 15.3 -> 25.7).
template <int A>
__device__ __forceinline__ u32x4 load_row(const char* p) {
    if constexpr (A == 16) {
        return *reinterpret_cast<const u32x4*>(p);
    } else if constexpr (A == 4) {
        return ld_any<0, 4>(p);
    } else {
        const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 2;
        const char* q = p - off;
        const u32x4 v = ld_any<0, 4>(q);
        const uint32_t last = *reinterpret_cast<const uint32_t*>(q + 12 + 2 * off);  // at a multiple of 4: v[3] again
        return u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 8 * off), __builtin_amdgcn_alignbit(v[2], v[1], 8 * off),
                     __builtin_amdgcn_alignbit(v[3], v[2], 8 * off), __builtin_amdgcn_alignbit(last, v[3], 8 * off)};
    }
}

// The 16 bytes of a row of K elements that start at byte kb, zeros behind its end; at any alignment.  Where the end cuts
// 2-byte elements, the 16 bytes that end there are read and moved down: one load without a branch, so that many can be
// under way ([801, 118] -> 384 4.7 -> 4.4 us; the three elements that f32 may have there come as fast one by one).
template <int DT>
__device__ __forceinline__ u32x4 row_piece(const char* row, int64_t kb, int K) {
    constexpr int S = DT == F32 ? 4 : 2, VE = 16 / S;
    const int64_t bytes = (int64_t)K * S;
    if (S == 2 && bytes >= 16) {
        const int64_t at = min(kb, bytes - 16);
        const u32x4 v = ld_any<0, S>(row + at);
        const int drop = (int)min<int64_t>(kb - at, 16);
        uint64_t lo = v[0] | (uint64_t)v[1] << 32, hi = v[2] | (uint64_t)v[3] << 32;
        if ((drop & 8) != 0) {
            lo = hi;
            hi = 0;
        }
        const int sh = 8 * (drop & 7);
        lo = drop == 16 ? 0 : lo >> sh | (hi << 1) << (63 - sh);
        hi = drop == 16 ? 0 : hi >> sh;
        return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
    if (bytes - kb >= 16) return ld_any<0, S>(row + kb);
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < VE - 1; ++j) {
        if (bytes - kb > (int64_t)j * S) {
            if constexpr (S == 4) v[j] = reinterpret_cast<const uint32_t*>(row + kb)[j];
            else v[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row + kb)[j] << (16 * (j & 1));
        }
    }
    return v;
}

// x Phi = max(x, 0) - |x| erfc(|z|) / 2, z = s x, by Abramowitz & Stegun 7.1.26 as in one_plus_erf_as (halved
// coefficients): 12 operations and two transcendental ones.
__device__ __forceinline__ float gelu_short(float x, float s) {
    const float az = fabsf(x) * s;
    const float t = fast_rcp(fmaf(0.3275911f, az, 1.0f));
    float p = fmaf(0.5307027145f, t, -0.7265760135f);
    p = fmaf(p, t, 0.7107068705f);
    p = fmaf(p, t, -0.142248368f);
    p = fmaf(p, t, 0.127414796f);
    p *= t * __builtin_amdgcn_exp2f(az * (az * -1.44269504088896341f));
    return fmaf(-fabsf(fminf(x, 64.0f)), p, fmaxf(x, 0.0f));  // p is 0 from 64 on: inf - 64 * 0, and -inf * 0 = NaN
}

// tanh x = 1 - 2 / (e^2x + 1), and the first terms of its series where that cancels (relative error 3.3e-7 at 1/4).
__device__ __forceinline__ float tanh_short(float x) {
    const float x2 = x * x;
    const float near = x * fmaf(x2, fmaf(x2, fmaf(x2, -0.0539682540f, 0.1333333333f), -0.3333333333f), 1.0f);
    const float far = fmaf(-2.0f, fast_rcp(1.0f + __builtin_amdgcn_exp2f(fabsf(x) * 2.88539008177792681f)), 1.0f);
    return fabsf(x) < 0.25f ? near : copysignf(far, x);
}

// f32 operands and f32 results take the library's erfc and tanh, 2-byte results of 2-byte operands the short forms: GELU's
// is bias_act's in the same case, tanh's this layer's own.  tanh is within 2^-19 of itself.  GELU is within 0.75e-7 |x|, a
// part of its value that grows into the negative tail: with z = x / sqrt 2 it passes half a step of bf16 (2^-8 of the value) below
// x = -6.1, where GELU is -3e-9, and of f16 (2^-11) below -4.0, where it is -1.1e-4 and 5.5e-8 off; with z = x below -4.3 and -2.9.
template <int NV>
__device__ __forceinline__ void activate(float (&v)[NV], int act, bool short_form) {
    if (act == MBRT_ACT_GELU_REF || act == MBRT_ACT_GELU_STD) {
        const bool ref = act == MBRT_ACT_GELU_REF;
        const float s = ref ? 1.0f : 0.70710678118654752440f;
        if (short_form) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = gelu_short(v[i], s);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = 0.5f * v[i] * erfcf(-v[i] * s);
        }
    } else if (act == MBRT_ACT_SIGMOID) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = sigmoidf(v[i]);
    } else if (act == MBRT_ACT_TANH) {
        if (short_form) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = tanh_short(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = tanhf(v[i]);
        }
    }
}

// NV consecutive elements at p[e], e on, as f32: 16 bytes at a time at any alignment.
template <int NV>
__device__ __forceinline__ void load_run(const void* p, int dt, int64_t e, float (&f)[NV]) {
    static_assert(NV % 4 == 0 || NV == 1, "whole pieces, or one element");
    if constexpr (NV == 1) {
        f[0] = load1(p, dt, e);
    } else if (dt == F32) {
        const char* b = reinterpret_cast<const char*>(p) + 4 * e;
#pragma unroll
        for (int q = 0; q < NV / 4; ++q) {
            const f32x4 t = __builtin_bit_cast(f32x4, ld_any<0, 4>(b + 16 * q));
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * q + i] = t[i];
        }
    } else {
        const char* b = reinterpret_cast<const char*>(p) + 2 * e;
        if constexpr (NV % 8 == 0) {
#pragma unroll
            for (int q = 0; q < NV / 8; ++q) {
                const u32x4 t = ld_any<0, 2>(b + 16 * q);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (dt == BF16) {
                        f[8 * q + 2 * i] = bf16_lo(t[i]);
                        f[8 * q + 2 * i + 1] = bf16_hi(t[i]);
                    } else {
                        const f32x2 h = unpack_f16x2(t[i]);
                        f[8 * q + 2 * i] = h.x;
                        f[8 * q + 2 * i + 1] = h.y;
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) f[i] = load1(p, dt, e + i);
        }
    }
}
template <int NT, int NV>
__device__ __forceinline__ void store_run(void* p, int dt, int64_t e, const float (&f)[NV]) {
    static_assert(NV % 4 == 0 || NV == 1, "whole pieces, or one element");
    if constexpr (NV == 1) {
        store1(p, dt, e, f[0]);
    } else if (dt == F32) {
        char* b = reinterpret_cast<char*>(p) + 4 * e;
#pragma unroll
        for (int q = 0; q < NV / 4; ++q)
            st_any<NT, 4>(b + 16 * q, u32x4{__float_as_uint(f[4 * q]), __float_as_uint(f[4 * q + 1]),
                                           __float_as_uint(f[4 * q + 2]), __float_as_uint(f[4 * q + 3])});
    } else if constexpr (NV % 8 == 0) {
        char* b = reinterpret_cast<char*>(p) + 2 * e;
#pragma unroll
        for (int q = 0; q < NV / 8; ++q) {
            u32x4 t;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                t[i] = dt == BF16 ? pack_bf16x2(f[8 * q + 2 * i], f[8 * q + 2 * i + 1])
                                  : pack_f16x2(f[8 * q + 2 * i], f[8 * q + 2 * i + 1]);
            char* d = b + 16 * q;
            if (NT != 0 || (reinterpret_cast<uintptr_t>(b) & 2) == 0) {
                st_any<NT, 4>(d, t);
            } else {  // stores at odd multiples of 2 are as slow as loads: [48060, 384] -> 385 42.5 -> 35.5 us
                *reinterpret_cast<uint16_t*>(d) = (uint16_t)t[0];
                *reinterpret_cast<uint32_t*>(d + 2) = __builtin_amdgcn_alignbit(t[1], t[0], 16);
                *reinterpret_cast<uint32_t*>(d + 6) = __builtin_amdgcn_alignbit(t[2], t[1], 16);
                *reinterpret_cast<uint32_t*>(d + 10) = __builtin_amdgcn_alignbit(t[3], t[2], 16);
                *reinterpret_cast<uint16_t*>(d + 14) = (uint16_t)(t[3] >> 16);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) store1(p, dt, e + i, f[i]);
    }
}

// The bias of NV consecutive columns n .. as it stands in memory, turned into f32 where it is used, so that nothing waits
// for it before (columns past N: the last one's; they are not stored).
template <int NV>
struct Bias {
    uint32_t w[NV];
    __device__ __forceinline__ void load(const LinArgs& a, int n) {
#pragma unroll
        for (int i = 0; i < NV; ++i) w[i] = 0;
        if (a.bias == nullptr) return;
        if (a.bdt == F32) {
#pragma unroll
            for (int i = 0; i < NV; ++i) w[i] = reinterpret_cast<const uint32_t*>(a.bias)[min(n + i, a.N - 1)];
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) w[i] = reinterpret_cast<const uint16_t*>(a.bias)[min(n + i, a.N - 1)];
        }
    }
    __device__ __forceinline__ void add_to(const LinArgs& a, float (&v)[NV]) const {
        if (a.bias == nullptr) return;
        if (a.bdt == F32) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __uint_as_float(w[i]);
        } else if (a.bdt == BF16) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += bf16_lo(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        }
    }
};

// The epilogue of NV consecutive columns n .. of row m (columns past N and rows past M are not stored).
template <bool ACT, int NT, int NV>
__device__ __forceinline__ void finish(const LinArgs& a, int64_t m, int n, float (&v)[NV], const Bias<NV>& bias) {
    if (m >= a.M || n >= a.N) return;
    bias.add_to(a, v);
    if constexpr (ACT) activate<NV>(v, a.act, a.short_act != 0);
    const bool whole = n + NV <= a.N;
    if (a.res != nullptr) {
        float r[NV];
        const int64_t e = m * a.rs + n;
        if (whole) {
            load_run<NV>(a.res, a.rdt, e, r);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += r[i];
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (n + i < a.N) v[i] += load1(a.res, a.rdt, e + i);
        }
    }
    const int64_t e = m * a.os + n;
    if (whole) {
        store_run<NT, NV>(a.out, a.odt, e, v);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (n + i < a.N) store1(a.out, a.odt, e + i, v[i]);
    }
}

// Tile form: WM x WN waves, each with MI x NI blocks of 16 x 16.  K goes by in steps of 128 bytes of every row, in
// two LDS buffers: the next step's tiles are on their way while one is computed.  An LDS row is 8 pieces of 16 bytes; piece
// j of a row stands at j ^ key(row), which makes the eight rows that neighbouring lanes read fall on different banks.  w is
// the A operand: a lane's four results of a block are four columns of one row of out, and two blocks 2 p, 2 p + 1 take
// the columns 32 p + 8 q + 4 (ni % 2) + j (q = c / 4, j = c % 4) of the wave's, so that a lane ends with 8 columns in a
// row, and a store of 16 bytes per lane fills 64 bytes in a row of out.
// KS groups of such waves take the steps in turn and are added at the end.
// DIRECT: rows are 16-byte aligned, and whole steps go from global memory straight into LDS.  NT: out is stored past the
// caches: a large one would push x and w out of them.
__device__ __forceinline__ int key_x(int r) { return r & 7; }
__device__ __forceinline__ int key_w(int r) { return (r & 3) | (((r >> 3) & 1) << 2); }

template <int DT, int WM, int WN, int MI, int NI, bool DIRECT, int NT, int KS, bool ACT>
__global__ __launch_bounds__(WM * WN * KS * 64) void linear_tile_kernel(LinArgs a) {
    constexpr int NW = WM * WN, BM = WM * MI * 16, BN = WN * NI * 16;
    constexpr int S = DT == F32 ? 4 : 2;
    constexpr int LX = BM / 8 / NW, LW = BN / 8 / NW;  // loads of 1 KB, 8 rows, per wave and step
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NI % 2 == 0, "whole loads per wave, blocks in pairs");
    constexpr int SB = kStepBytes, kBuf = (BM + BN) * SB;
    __shared__ __attribute__((aligned(16))) char s0[KS * kBuf];
    __shared__ __attribute__((aligned(16))) char s1[KS * kBuf];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int kg = KS == 1 ? 0 : wave / NW, w = KS == 1 ? wave : wave % NW;
    char* const mine0 = s0 + kg * kBuf;
    char* const mine1 = s1 + kg * kBuf;
    const int wm = w / WN, wn = w % WN;
    // column tiles of one row tile are neighbours, on one XCD: x is read once into its L2
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    uint32_t mt, nt;
    fdivmod(tile, a.groups, mt, nt);
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN;
    const char* xb = a.x + m0 * a.xs;
    const char* wb = a.w + (int64_t)n0 * a.ws;
    const int mrows = (int)min((int64_t)BM, a.M - m0), nrows = min(BN, a.N - n0);
    const int64_t kbytes = (int64_t)a.K * S;
    const int steps = (int)((kbytes + SB - 1) / SB);
    const int whole = DIRECT ? (int)(kbytes / SB) : 0;  // steps loaded straight into LDS

    // lane i of load u covers LDS row 8 (LX w + u) + i / 8, place i % 8; rows past the end repeat the last one
    int xr[LX], wr[LW];
    uint32_t xo[LX], wo[LW];  // within the step: byte offset of the lane's piece from xb, wb (DIRECT)
#pragma unroll
    for (int u = 0; u < LX; ++u) {
        const int r = 8 * (LX * w + u) + lane / 8;
        xr[u] = min(r, mrows - 1);
        xo[u] = (uint32_t)xr[u] * (uint32_t)a.xs + 16u * ((lane % 8) ^ key_x(r));
    }
#pragma unroll
    for (int u = 0; u < LW; ++u) {
        const int r = 8 * (LW * w + u) + lane / 8;
        wr[u] = min(r, nrows - 1);
        wo[u] = (uint32_t)wr[u] * (uint32_t)a.ws + 16u * ((lane % 8) ^ key_w(r));
    }
    const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc((void*)xb, (short)0, -1, kBufferDword3);
    const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc((void*)wb, (short)0, -1, kBufferDword3);
    auto load_direct = [&](int kt, char* d) {
#pragma unroll
        for (int u = 0; u < LX; ++u) load_to_lds(xres, d + 1024 * (LX * w + u), xo[u], kt * SB);
#pragma unroll
        for (int u = 0; u < LW; ++u) load_to_lds(wres, d + BM * SB + 1024 * (LW * w + u), wo[u], kt * SB);
    };
    // a step that is cut by the end of the rows, or of rows at other alignments: through registers
    u32x4 px[LX], pw[LW];
    auto load_regs = [&](int kt) {
        if (!DIRECT && (int64_t)(kt + 1) * SB <= kbytes) {  // a whole step: no checks between the loads
#pragma unroll
            for (int u = 0; u < LX; ++u)
                px[u] = ld_any<0, S>(xb + xr[u] * a.xs + (int64_t)kt * SB + 16 * ((lane % 8) ^ key_x(8 * (LX * w + u) + lane / 8)));
#pragma unroll
            for (int u = 0; u < LW; ++u)
                pw[u] = ld_any<0, S>(wb + wr[u] * a.ws + (int64_t)kt * SB + 16 * ((lane % 8) ^ key_w(8 * (LW * w + u) + lane / 8)));
            return;
        }
#pragma unroll
        for (int u = 0; u < LX; ++u)
            px[u] = row_piece<DT>(xb + xr[u] * a.xs, (int64_t)kt * SB + 16 * ((lane % 8) ^ key_x(8 * (LX * w + u) + lane / 8)), a.K);
#pragma unroll
        for (int u = 0; u < LW; ++u)
            pw[u] = row_piece<DT>(wb + wr[u] * a.ws, (int64_t)kt * SB + 16 * ((lane % 8) ^ key_w(8 * (LW * w + u) + lane / 8)), a.K);
    };
    auto put_regs = [&](char* d) {
#pragma unroll
        for (int u = 0; u < LX; ++u) *reinterpret_cast<u32x4*>(d + 1024 * (LX * w + u) + 16 * lane) = px[u];
#pragma unroll
        for (int u = 0; u < LW; ++u) *reinterpret_cast<u32x4*>(d + BM * SB + 1024 * (LW * w + u) + 16 * lane) = pw[u];
    };

    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const int xrow = (wm * MI * 16 + c) * SB;
    const int wrow = BM * SB + (wn * NI * 16 + 8 * (c >> 2) + (c & 3)) * SB;
    auto compute = [&](const char* d) {
#pragma unroll
        for (int s = 0; s < SB / 64; ++s) {
            const int piece = 16 * ((4 * s + g) ^ (c & 7));
            u32x4 xf[MI], wf[NI];
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) xf[mi] = *reinterpret_cast<const u32x4*>(d + xrow + mi * 16 * SB + piece);
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) wf[ni] = *reinterpret_cast<const u32x4*>(d + wrow + (32 * (ni / 2) + 4 * (ni % 2)) * SB + piece);
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mma<DT>(wf[ni], xf[mi], acc[mi][ni]);
        }
    };
    if constexpr (DIRECT) {
        // The column tiles of one row tile run side by side and read the same rows of x.  Where they are few, each begins at
        // another step and goes round, so that together they have more of the rows on their way from memory at
        // once (bf16 [48060, 1536] -> 384, two tiles: 97 -> 93 us); many of them run apart by themselves, and going round
        // then costs reuse ([4096, 4096] -> 4096: 127 -> 146).
        const int first = a.ntiles <= 4 ? (int)(nt * (uint32_t)whole / a.ntiles) : 0;
        auto at = [&](int kt) { return kt + first < whole ? kt + first : kt + first - whole; };
        // Step kt of this group sits in d, its next one goes to dn, which held the one before.  The buffers are separate
        // objects and the loop is unrolled by two, so that the compiler sees that loads in flight into one do not touch the
        // other.
        auto step = [&](int kt, const char* d, char* dn) {
            wait_loads();
            lds_barrier();  // every wave's loads have landed, and none still reads dn
            if (kt + KS < whole) load_direct(at(kt + KS), dn);
            if (KS == 1 || kt < whole) compute(d);
        };
        if (kg < whole) load_direct(at(kg), mine0);
        for (int kt = 0; kt < whole; kt += 2 * KS) {
            step(kt + kg, mine0, mine1);
            if (kt + KS < whole) step(kt + KS + kg, mine1, mine0);
        }
        if (steps > whole) {  // the first group takes what the rows' end cuts
            if (kg == 0) load_regs(whole);
            __syncthreads();  // none still reads s0
            if (kg == 0) put_regs(s0);
            __syncthreads();
            if (kg == 0) compute(s0);
        }
    } else {
        // through registers: the next step's loads are issued before a step is computed and written to LDS after it
        load_regs(0);
        put_regs(s0);
        for (int kt = 0; kt < steps; kt += 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (kt + i < steps) {
                    __syncthreads();  // the step is in LDS, and none still reads the other buffer
                    const bool next = kt + i + 1 < steps;
                    if (next) load_regs(kt + i + 1);
                    compute(i == 0 ? s0 : s1);
                    if (next) put_regs(i == 0 ? s1 : s0);
                }
            }
        }
    }

    if constexpr (KS > 1) {  // the groups' sums, added in their order; group mi ends with the blocks mi
        static_assert(BM * BN * 4 <= kBuf && MI <= KS, "room for the sums, a group for each");
        __syncthreads();  // none still reads s0
        f32x4* all = reinterpret_cast<f32x4*>(s0) + w * MI * NI * 64 + lane;
        constexpr int kGroup = kBuf / 16;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) all[kg * kGroup + (mi * NI + ni) * 64] = acc[mi][ni];
        __syncthreads();
        if (kg >= MI) return;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
            f32x4 sum = all[(kg * NI + ni) * 64];
#pragma unroll
            for (int k = 1; k < KS; ++k) sum += all[k * kGroup + (kg * NI + ni) * 64];
            acc[0][ni] = sum;
        }
    }

    const int n = n0 + wn * NI * 16 + 8 * g;
    Bias<8> bias[NI / 2];
#pragma unroll
    for (int p = 0; p < NI / 2; ++p) bias[p].load(a, n + 32 * p);
#pragma unroll
    for (int mi = 0; mi < (KS > 1 ? 1 : MI); ++mi)
#pragma unroll
        for (int p = 0; p < NI / 2; ++p) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[mi][2 * p + i / 4][i % 4];
            finish<ACT, NT, 8>(a, m0 + wm * MI * 16 + (KS > 1 ? kg : mi) * 16 + c, n + 32 * p, v, bias[p]);
        }
}

// Strip form: a wave takes 16 rows of one operand and 16 R of the other, straight from global memory into the matrix
// instructions; `split` waves of a block share the K of one such piece, 128 bytes of every row at a time in turn, and are
// added through LDS in wave order.  Nothing but the loads' latency, once or twice, stands between a small call's launch and
// its stores.
// WIDE: strips of w (16 columns of out) against groups of 16 R rows of x; else strips of x against groups of 16 R columns.
// The groups of one strip are neighbours.
template <int DT, int R, bool WIDE, int A>
__global__ __launch_bounds__(1024) void linear_strip_kernel(LinArgs a) {
    constexpr int S = DT == F32 ? 4 : 2;
    extern __shared__ f32x4 part[];  // [strips of the block][split][R][64]
    const int lane = threadIdx.x % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    uint32_t strip, kw, sb, group;
    fdivmod((uint32_t)w, a.splits, strip, kw);
    fdivmod(blockIdx.x, a.groups, sb, group);
    const int ks = (int)kw;
    const int64_t p0 = ((int64_t)sb * a.per_block + strip) * 16, q0 = (int64_t)group * 16 * R;
    const int64_t P = WIDE ? a.N : a.M, Q = WIDE ? a.M : a.N;
    const char* pb = (WIDE ? a.w : a.x) + min(p0 + c, P - 1) * (WIDE ? a.ws : a.xs) + 16 * g;
    const char* qb[R];
#pragma unroll
    for (int r = 0; r < R; ++r) qb[r] = (WIDE ? a.x : a.w) + min(q0 + 16 * r + c, Q - 1) * (WIDE ? a.xs : a.ws) + 16 * g;
    const int64_t kbytes = (int64_t)a.K * S;
    const int whole = (int)(kbytes / 128);
    // w is the A operand: a lane ends with four columns n .. of one row of each block; the bias of the first block that
    // this wave finishes is on its way beside the rows
    auto column = [&](int r) { return (int)min<int64_t>(WIDE ? p0 + 4 * g : q0 + 16 * r + 4 * g, a.N); };
    Bias<4> bias;
    bias.load(a, column(a.split == 1 ? 0 : min(ks, R - 1)));

    f32x4 acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // U pieces of 128 bytes, all loads before the first product (a lane's loads are whole: no checks)
    auto pieces = [&](auto count, int t0) {
        constexpr int U = decltype(count)::value;
        u32x4 pf[U][2], qf[U][2][R];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int64_t kb = (int64_t)(t0 + u * a.split) * 128 + 64 * s;
                pf[u][s] = load_row<A>(pb + kb);
#pragma unroll
                for (int r = 0; r < R; ++r) qf[u][s][r] = load_row<A>(qb[r] + kb);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    acc[r] = WIDE ? mma<DT>(pf[u][s], qf[u][s][r], acc[r]) : mma<DT>(qf[u][s][r], pf[u][s], acc[r]);
    };
    constexpr int U = R >= 4 ? (A == 2 ? 1 : 2) : R == 2 ? 3 : 6;
    int t0 = ks;
    for (; t0 + (U - 1) * a.split < whole; t0 += U * a.split) pieces(std::integral_constant<int, U>(), t0);
    for (; t0 < whole; t0 += a.split) pieces(std::integral_constant<int, 1>(), t0);
    if (t0 == whole && kbytes > (int64_t)whole * 128) {  // this wave's turn at the piece that the rows' end cuts
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t kb = (int64_t)whole * 128 + 64 * s + 16 * g;
            if (kb - 16 * g >= kbytes) break;
            const u32x4 pf = row_piece<DT>(pb - 16 * g, kb, a.K);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const u32x4 qf = row_piece<DT>(qb[r] - 16 * g, kb, a.K);
                acc[r] = WIDE ? mma<DT>(pf, qf, acc[r]) : mma<DT>(qf, pf, acc[r]);
            }
        }
    }
    auto finish_block = [&](int r, const f32x4& s) {
        float v[4] = {s[0], s[1], s[2], s[3]};
        finish<true, 0, 4>(a, WIDE ? q0 + 16 * r + c : p0 + c, column(r), v, bias);
    };
    if (a.split == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r > 0 && !WIDE) bias.load(a, column(r));
            finish_block(r, acc[r]);
        }
        return;
    }
    f32x4* all = part + (int64_t)strip * a.split * R * 64 + lane;
#pragma unroll
    for (int r = 0; r < R; ++r) all[(ks * R + r) * 64] = acc[r];
    __syncthreads();
    for (int r = ks; r < R; r += a.split) {
        f32x4 s = all[r * 64];
        for (int k = 1; k < a.split; ++k) s += all[(k * R + r) * 64];
        if (r > ks && !WIDE) bias.load(a, column(r));
        finish_block(r, s);
    }
}

template <int DT, int R>
void launch_strip(const LinArgs& a, bool wide, int align, unsigned blocks, unsigned threads, size_t lds, hipStream_t st) {
    auto launch = [&](auto bytes) {
        constexpr int A = decltype(bytes)::value;
        if (wide) hipLaunchKernelGGL((linear_strip_kernel<DT, R, true, A>), dim3(blocks), dim3(threads), lds, st, a);
        else hipLaunchKernelGGL((linear_strip_kernel<DT, R, false, A>), dim3(blocks), dim3(threads), lds, st, a);
    };
    if (align == 16) return launch(std::integral_constant<int, 16>());
    if constexpr (DT != F32) {
        if (align == 2) return launch(std::integral_constant<int, 2>());
    }
    launch(std::integral_constant<int, 4>());
}

template <int DT, int WM, int WN, int MI, int NI, bool DIRECT, int NT, int KS = 1>
int launch_tile(LinArgs& a, hipStream_t st) {
    constexpr int BM = WM * MI * 16, BN = WN * NI * 16;
    a.ntiles = (uint32_t)ceil_div(a.N, BN);
    a.groups = make_fastdiv(a.ntiles);
    const int64_t tiles = ceil_div(a.M, BM) * a.ntiles;
    if (!grid_fits(tiles, WM * WN * KS * 64)) return set_error(MBRT_E_SHAPE, "mbrt_linear: too many tiles");
    const dim3 grid((unsigned)tiles), block(WM * WN * KS * 64);
    if (a.act != MBRT_ACT_NONE)
        hipLaunchKernelGGL((linear_tile_kernel<DT, WM, WN, MI, NI, DIRECT, NT, KS, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((linear_tile_kernel<DT, WM, WN, MI, NI, DIRECT, NT, KS, false>), grid, block, 0, st, a);
    return MBRT_OK;
}

// Tiles of 96 or 128 by 192, two workgroups to a CU: the height whose rounds over the CUs take fewer rows (the larger at a
// tie, for its reuse).  bf16 us, 96 and 128 rows: [48060, 384] -> 1536, 8 and 6 rounds, 79 and 70; [48060, 1536] -> 384, 2
// and 2 rounds, 93 and 95; [48060, 512] -> 384 43 and 51; [4096, 4096] -> 4096, 2 and 2, 127 and 137.
template <int DT>
int launch_large(LinArgs& a, bool direct, hipStream_t st) {
    const int64_t cus = cu_count();
    auto rounds = [&](int64_t bm, int64_t bn) { return ceil_div(ceil_div(a.M, bm) * ceil_div(a.N, bn), 2 * cus); };
    // Past the caches where a wave's stores fill whole 64-byte pieces; cut ones need the cache to put them together: bf16
    // [20000, 393] -> 500 40 -> 32 us through it, [48060, 385] -> 384 52 -> 37 past it.
    const int64_t ob = dt_size(a.odt);
    const bool nt = aligned(a.out, 64) && a.os * ob % 64 == 0;
    if (!direct) return nt ? launch_tile<DT, 2, 2, 3, 6, false, 2>(a, st) : launch_tile<DT, 2, 2, 3, 6, false, 0>(a, st);
    if (96 * rounds(96, 192) < 128 * rounds(128, 192))
        return nt ? launch_tile<DT, 2, 2, 3, 6, true, 2>(a, st) : launch_tile<DT, 2, 2, 3, 6, true, 0>(a, st);
    return nt ? launch_tile<DT, 2, 2, 4, 6, true, 2>(a, st) : launch_tile<DT, 2, 2, 4, 6, true, 0>(a, st);
}

}  // namespace

template <int DT>
int launch_linear(LinArgs& a, int align, hipStream_t st) {
    const bool al = align == 16;
    const int64_t es = DT == F32 ? 4 : 2, cus = cu_count();
    const bool wide = a.M <= a.N;
    const int64_t shorter = wide ? a.M : a.N, longer = wide ? a.N : a.M;
    const int64_t strips = ceil_div(longer, 16);
    // Strips, where tiles would leave most CUs idle (f32, bound by its products sooner: any), of as few rows per wave as there
    // are CUs for; rows at odd alignments, which tiles take through registers step by step, go in strips up to twice as far,
    // spread eight times as wide.  us, tiles and strips: bf16 [200, 1536] -> 384 8.5 and 6.7, [124, 1536] -> 1536 6.8 and
    // 9.7, [120, 384] -> 1536 4.1 and 4.7; f32 17 at [124, 1536] -> 1536 and 26 in tiles, [200, 384] -> 1536 9.5 and 9.7,
    // [1000, 1536] -> 384 26.5 and 31.3; [801, 118] -> 384 bf16 6.2 and 4.3, f32 7.0 and 4.9.
    // A short operand of up to 16 rows goes in strips too, which multiply no 16 rows in vain where tiles multiply 64: always
    // for f32, whose products count ([48060, 384] -> 8 25 and 18; up to 32 rows while tiles are few, [5000, 1536] -> 24 31 and 18,
    // but [48060, 1536] -> 24 81 and 93), and for 2-byte types where tiles of 64 are few ([10000, 384] -> 8 4.8 and 4.3, [16000,
    // 1536] -> 8 12.4 and 12.3) or K is short.  How short goes by what a tile loses at its rows' end: whole pieces of 128 bytes
    // up to one of them ([48060, 64] -> 8 4.3 and 4.1, [48060, 128] -> 16 4.8 and 5.2, [48060, 256] -> 16 6.3 and 7.6, [48060,
    // 384] -> 8 8.0 and 8.6, -> 16 8.1 and 10.4), as rows at odd addresses ([48060, 65] -> 8 5.9 and 5.7, [48060, 193] -> 16 8.6 and 10.3,
    // [48060, 385] -> 8 12.0 and 14.6); pieces that are cut up to six, where it turns with the other sizes (-> 8 from [48060, 200]
    // 7.1 and 5.7, 386 10.6 and 9.7, 392 10.1 and 8.2, 456 11.6 and 10.5, 648 16.5 and 17.1; -> 16 376 9.7 and 9.4, 386 10.7 and
    // 11.6, 392 10.5 and 9.4, 456 12.0 and 12.3; [16, 264] -> 20000 4.9 and 4.7, 386 6.7 and 8.3, 392 5.3 and 6.1).
    const int64_t kb = a.K * es, short_k = kb % 128 != 0 && align >= 4 ? 6 * 128 : 2 * 128;
    if (strips * ceil_div(shorter, 64) <= (DT == F32 ? (al ? 1 : 2) * cus : (al ? 1 : 4) * cus / 2) ||
        (shorter <= 16 && (DT == F32 || longer < 64 * cus || kb < short_k)) ||
        (DT == F32 && shorter <= 32 && longer < 64 * cus)) {
        int R = shorter <= 16 ? 1 : shorter <= 32 ? 2 : 4;
        while (R > 1 && strips * ceil_div(shorter, 8 * R) <= (al ? 1 : 8) * cus) R /= 2;
        const int64_t groups = ceil_div(shorter, 16 * R), pairs = ceil_div(a.K * es, 128);
        // waves to a strip's K: as many as find room side by side, each with the same number of turns
        const int64_t room = std::max<int64_t>(1, std::min<int64_t>(16, 8 * cus / (strips * groups)));
        a.split = (int)ceil_div(pairs, ceil_div(pairs, room));
        a.ntiles = (uint32_t)groups;
        const int per_block = std::max(1, 4 / a.split);
        a.per_block = per_block;
        a.groups = make_fastdiv((uint32_t)groups);
        a.splits = make_fastdiv((uint32_t)a.split);
        const int64_t blocks = ceil_div(strips, per_block) * groups;
        const size_t lds = a.split == 1 ? 0 : (size_t)per_block * a.split * R * 1024;
        const unsigned threads = per_block * a.split * 64;
        if (!grid_fits(blocks, threads)) return set_error(MBRT_E_SHAPE, "mbrt_linear: too many rows");
        if (R == 1) launch_strip<DT, 1>(a, wide, align, (unsigned)blocks, threads, lds, st);
        else if (R == 2) launch_strip<DT, 2>(a, wide, align, (unsigned)blocks, threads, lds, st);
        else launch_strip<DT, 4>(a, wide, align, (unsigned)blocks, threads, lds, st);
        return MBRT_OK;
    }
    // 32-bit offsets within a tile
    const bool direct = al && a.xs < (int64_t(1) << 22) && a.ws < (int64_t(1) << 22);
    // Tiles of 64 x 64 until larger ones fill the CUs, and for a short operand that one of them holds (bf16 us, large
    // and small: [48060, 384] -> 64 11.0 and 9.5, -> 128 12.0 and 14.1, [50, 384] -> 60000 12.7 and 10.8).  For f32 always: its
    // products bound it either way, and small tiles compute fewer columns in vain ([48060, 384] -> 128 60 and 45, -> 384 119 and
    // 117; [4096, 4096] -> 4096 1050 and 990, 139 TFLOP/s).
    const bool big = DT != F32 && shorter > 64 && ceil_div(a.M, 96) * ceil_div(a.N, 192) >= cus;
    // Few tiles leave a CU with four waves, which wait for their loads and for each other step by step: 2 or 4 groups of them
    // take the steps in turn, each in buffers of its own, and are added through LDS.  us with 1, 2 and 4 groups: bf16 [444,
    // 1536] -> 1536 (168 tiles) 14.3, 11.3 and 9.9, [5000, 1536] -> 24 (79) 13.2, 9.7 and 8.3, [801, 384] -> 384 (91, six
    // steps) 4.4, 4.1 and 4.3; [3000, 1536] -> 384 (282) 13.5, 10.9 and 15.8, [3000, 384] -> 384 4.8, 5.4 and 7.4; [1517, 1536] ->
    // 1536 (576) 15.5, 20.3 and 24.8; f32 [444, 1536] -> 1536 33, 30 and 28.
    if (!big && direct) {
        const int64_t tiles = ceil_div(a.M, 64) * ceil_div(a.N, 64), steps = a.K * es / kStepBytes;
        if (tiles <= cus && steps >= 12) return launch_tile<DT, 2, 2, 2, 2, true, 0, 4>(a, st);
        if ((tiles <= cus && steps >= 4) || (2 * tiles <= 3 * cus && steps >= 24))
            return launch_tile<DT, 2, 2, 2, 2, true, 0, 2>(a, st);
    }
    if (!big) return direct ? launch_tile<DT, 2, 2, 2, 2, true, 0>(a, st) : launch_tile<DT, 2, 2, 2, 2, false, 0>(a, st);
    if constexpr (DT != F32) return launch_large<DT>(a, direct, st);
    return MBRT_OK;
}

}  // namespace mbrt
