// The norms before and after a block, with the gate and the scale of its residual, in one pass over the rows:
//
//   u = update                                                                  (no post_gamma)
//     = update * post_scale * post_gamma / sqrt(sum update^2 + eps)
//   h = residual + alpha * layer_scale * gate * u                               rounded to residual's type
//   normed = h * scale * gamma / sqrt(sum h^2 + eps)                            of h as it is rounded
//
// Every byte is read once and written once: a group of G lanes (16, 64, or the 256 of a block) holds a row in registers through
// both norms, lane l its chunks l, l + G, ... of 16 bytes (VE elements: 8 where all operands have 2 bytes, else 4, f32 ones
// 16 bytes and 2-byte ones 8).  The two sums of squares are butterflies within the group, and sums over four waves through
// LDS where a block holds the row.  The vectors over the features are put into LDS once per block, or read where they are
// needed by a block that has one row.  All loads of rows, and those into LDS, are issued before the first use: a call of few
// rows takes one round of them.
// Both results are formed in the formula's order, one f32 rounding per operation and quotients by the roots, so that they differ from
// the formula in f32 calls by the order of the two sums alone, and 4-bit values behind them seldom do.  An h of 2 bytes that lies on
// a tie of its rounding can still fall to the other side, and normed follows it as it is stored: of [48060, 384] 146 elements in bf16
// and 754 in f16, where the formula in f32 itself differs from 64 bits in 709 and 3193.  Quotients cost 0.3 us of 13.2 (f16
// [4, 4003, 512]) against products with the reciprocal root.
// A row whose last chunk is cut has it moved back to end at the row's end: its first elements are the chunk's before, left
// out of the sums and stored twice with the same values, so that odd widths take the same loads as even ones.
// normed may leave as microscaled 4-bit floats (mx.hpp): the lanes of a block of 32 stand side by side.
#include "abi_common.hpp"
#include "mx.hpp"
#include "overlap.hpp"

#include <algorithm>

namespace mbrt {
namespace {

constexpr int kThreads = 256;

struct BlockNormArgs {
    const char* res;
    const char* upd;
    const char* gate;        // NULL: 1
    const void* gamma;       // NULL: no second norm
    const void* post_gamma;  // NULL: no first norm
    const void* ls;          // layer scale, NULL: 1
    char* sum;               // NULL: not stored
    char* out;               // normed, or its codes; NULL without gamma
    uint8_t* oscales;
    int64_t rs, us, gs, ss, os, oss;  // row strides in bytes
    uint32_t rows, row0;  // of this launch; the first one's number among all
    int dim, chunks, padded; // chunks of VE of a row: those with elements, and with the zeros that fill a block of 32
    int rdt, udt, gdt, odt, gadt, pdt, ldt;
    int gate_vec, gate_logit;
    FastDiv inner, period;   // gate row = (row / inner) % period
    float alpha, scale, post_scale, eps;
};

// N elements of S bytes as they stand in memory, at any alignment of the elements.
template <int S, int N>
struct Chunk {
    static constexpr int kWords = S * N / 4;
    uint32_t w[kWords];
    template <bool AL>
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (kWords == 4) {
            const u32x4 t = AL ? *reinterpret_cast<const u32x4*>(p) : ld_any<0, S>(p);
            w[0] = t[0]; w[1] = t[1]; w[2] = t[2]; w[3] = t[3];
        } else {
            typedef uint32_t any2 __attribute__((ext_vector_type(2), aligned(2)));
            const u32x2 t = AL ? *reinterpret_cast<const u32x2*>(p) : (u32x2)*reinterpret_cast<const any2*>(p);
            w[0] = t[0]; w[1] = t[1];
        }
    }
    template <bool AL>
    __device__ __forceinline__ void store(char* p) const {
        if constexpr (kWords == 4) {
            const u32x4 t = {w[0], w[1], w[2], w[3]};
            if constexpr (AL) *reinterpret_cast<u32x4*>(p) = t;
            else st_any<0, S>(p, t);
        } else {
            typedef uint32_t any2 __attribute__((ext_vector_type(2), aligned(2)));
            const u32x2 t = {w[0], w[1]};
            if constexpr (AL) *reinterpret_cast<u32x2*>(p) = t;
            else *reinterpret_cast<any2*>(p) = t;
        }
    }
    __device__ __forceinline__ void to_f32(int dt, float (&f)[N]) const {
        if constexpr (S == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
        } else if (dt == BF16) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const f32x2 t = unpack_f16x2(w[i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
    __device__ __forceinline__ void from_f32(int dt, const float (&f)[N]) {
        if constexpr (S == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = __float_as_uint(f[i]);
        } else if (dt == BF16) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i] = pack_f16x2(f[2 * i], f[2 * i + 1]);
        }
    }
};

// A gate for a whole row: one exp and one division each.
__device__ __forceinline__ float gate_value(float g, int logit) { return logit ? 1.0f / (1.0f + expf(-g)) : g; }

// v / sqrt(ss): the device's square root and a quotient correctly rounded (but below f32's normal numbers), by one division per row.
struct Root {
    float value, inv;
};
__device__ __forceinline__ Root root_of(float ss) {
    const float r = sqrtf(ss);
    return {r == __builtin_inff() ? 0.0f : r, 1.0f / r};  // (of an infinite sum the quotients are 0: so they stay)
}
__device__ __forceinline__ float over(float v, Root r) {
    const float q = v * r.inv;
    return fmaf(fmaf(-q, r.value, v), r.inv, q);
}

// Elements p[d] of a vector of dim >= 4, d a thread's every kThreads-th (past the end: any), as they stand in memory: a dword each, for
// two bytes the element and the next, the last two at the end.  A load per type in branches of its own would wait for the one
// before, since either could still be on its way into its register.
template <int E>
struct Staged {
    uint32_t w[E];
    __device__ __forceinline__ void load(const void* p, int dt, int dim) {
        typedef uint32_t any1 __attribute__((aligned(2)));
        const int64_t size = dt == F32 ? 4 : 2;
        const int last = dt == F32 ? dim - 1 : dim - 2;
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = 0;
        if (p == nullptr) return;
#pragma unroll
        for (int e = 0; e < E; ++e)
            w[e] = *reinterpret_cast<const any1*>(static_cast<const char*>(p) + min((int)threadIdx.x + e * kThreads, last) * size);
    }
    __device__ __forceinline__ float value(int e, int dt, int dim) const {
        if (dt == F32) return __uint_as_float(w[e]);
        const uint32_t v = (int)threadIdx.x + e * kThreads > dim - 2 ? w[e] >> 16 : w[e];
        return dt == BF16 ? bf16_lo(v) : (float)__builtin_bit_cast(_Float16, (uint16_t)v);
    }
};

// N features from d on, at any place; p NULL: ones.
template <int N>
__device__ __forceinline__ void features(const void* p, int dt, int d, float (&f)[N]) {
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = 1.0f;
    } else if (dt == F32) {
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const u32x4 t = ld_any<0, 4>(reinterpret_cast<const float*>(p) + d + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * q + i] = __uint_as_float(t[i]);
        }
    } else {
        Chunk<2, N> t;
        t.template load<false>(reinterpret_cast<const char*>(p) + 2 * d);
        t.to_f32(dt, f);
    }
}

// The sum of a chunk's squares from its element `first` on (AL: of all, or with first VE of none).  Lanes add chunk by chunk: shorter chains
// of roundings than element by element, and half the operations where nothing is left out inside a chunk.
template <bool AL, int VE>
__device__ __forceinline__ float chunk_squares(const float (&v)[VE], int first) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < VE; ++i) t = AL || i >= first ? fmaf(v[i], v[i], t) : t;
    return AL && first != 0 ? 0.0f : t;
}

// The sum over a group's lanes, in each of them.  turn: another place in LDS for each sum of a row.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* turn) {
    if constexpr (G <= 64) {
        return group_sum<G>(v);
    } else {
        v = group_sum<64>(v);
        if (threadIdx.x % 64 == 0) turn[threadIdx.x / 64] = v;
        __syncthreads();
        return (turn[0] + turn[1]) + (turn[2] + turn[3]);
    }
}

// RS, US: bytes of the residual's and the update's elements; GS: of a gate with a value per feature, 0 where there is one per
// row or none.  AL: every row of every operand begins at a multiple of its chunk's bytes and is whole chunks long.
template <int VE, int RS, int US, int GS, int G, int NC, bool AL>
__global__ __launch_bounds__(kThreads) void block_norm_kernel(BlockNormArgs a) {
    constexpr bool IN_LDS = G < kThreads;
    constexpr int E = (NC * G * VE + kThreads - 1) / kThreads;  // features of a thread as it fills LDS
    extern __shared__ float lds[];
    // IN_LDS: post_scale * post_gamma, layer_scale and scale * gamma
    float* const post = lds;
    float* const by = lds + a.dim;
    float* const gam = by + a.dim;
    const int lane = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
    const bool valid = row < a.rows;
    const int64_t r = valid ? row : a.rows - 1;
    Chunk<RS, VE> rv[NC];
    Chunk<US, VE> uv[NC];
    Chunk<GS ? GS : 2, VE> gv[NC];
    int at[NC];  // first element of the chunk
    const char* gp = a.gate;
    if (a.gate != nullptr) {
        uint32_t d, m;
        fdivmod(fdiv(a.row0 + (uint32_t)r, a.inner), a.period, d, m);
        gp += m * a.gs;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int c = min(lane + G * k, a.chunks - 1);
        at[k] = AL ? c * VE : min(c * VE, a.dim - VE);
        rv[k].template load<AL>(a.res + r * a.rs + (int64_t)at[k] * RS);
        uv[k].template load<AL>(a.upd + r * a.us + (int64_t)at[k] * US);
        if constexpr (GS != 0) gv[k].template load<AL>(gp + (int64_t)at[k] * GS);
    }
    uint32_t gw = 0;
    if (GS == 0 && a.gate != nullptr)
        gw = a.gdt == F32 ? *reinterpret_cast<const uint32_t*>(gp) : *reinterpret_cast<const uint16_t*>(gp);
    if constexpr (IN_LDS) {
        Staged<E> ls, pg, ga;
        ls.load(a.ls, a.ldt, a.dim);
        pg.load(a.post_gamma, a.pdt, a.dim);
        ga.load(a.gamma, a.gadt, a.dim);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = threadIdx.x + e * kThreads;
            if (d < a.dim) {
                post[d] = pg.value(e, a.pdt, a.dim) * a.post_scale;
                by[d] = ls.value(e, a.ldt, a.dim);
                gam[d] = ga.value(e, a.gadt, a.dim) * a.scale;
            }
        }
        __syncthreads();
    }
    float g = 1.0f;
    if (GS == 0 && a.gate != nullptr)
        g = gate_value(a.gdt == F32    ? __uint_as_float(gw)
                       : a.gdt == BF16 ? bf16_lo(gw)
                                       : (float)__builtin_bit_cast(_Float16, (uint16_t)gw),
                       a.gate_logit);
    float h[NC][VE];
    Root root{};
    if (a.post_gamma != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float u[VE];
            uv[k].to_f32(a.udt, u);
            const int first = AL ? (lane + G * k < a.chunks ? 0 : VE) : (lane + G * k) * VE - at[k];  // before it: another chunk's
            ss += chunk_squares<AL>(u, first);
        }
        root = root_of(row_sum<G>(ss, lds) + a.eps);
    }
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        float u[VE], x[VE];
        uv[k].to_f32(a.udt, u);
        rv[k].to_f32(a.rdt, x);
        const int first = AL ? (lane + G * k < a.chunks ? 0 : VE) : (lane + G * k) * VE - at[k];
        float f[VE], w[VE];
        if constexpr (GS != 0) {
            gv[k].to_f32(a.gdt, w);
            if (a.gate_logit) {
#pragma unroll
                for (int i = 0; i < VE; ++i) w[i] = sigmoidf(w[i]);
            }
        }
        if (a.post_gamma != nullptr) {
            if constexpr (IN_LDS) {
#pragma unroll
                for (int i = 0; i < VE; ++i) f[i] = post[at[k] + i];
            } else {
                features<VE>(a.post_gamma, a.pdt, at[k], f);
#pragma unroll
                for (int i = 0; i < VE; ++i) f[i] *= a.post_scale;
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) u[i] = over(u[i] * f[i], root);
        }
        if (a.ls != nullptr) {
            if constexpr (IN_LDS) {
#pragma unroll
                for (int i = 0; i < VE; ++i) f[i] = by[at[k] + i];
            } else {
                features<VE>(a.ls, a.ldt, at[k], f);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) u[i] *= f[i];
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) h[k][i] = fmaf(u[i] * (GS != 0 ? w[i] : g), a.alpha, x[i]);
        Chunk<RS, VE> t;
        t.from_f32(a.rdt, h[k]);
        t.to_f32(a.rdt, h[k]);
        if (G <= 64 && a.sum != nullptr && valid && lane + G * k < a.chunks) t.template store<AL>(a.sum + r * a.ss + (int64_t)at[k] * RS);
        ss += chunk_squares<AL>(h[k], first);
    }
    root = root_of(row_sum<G>(ss, lds + 4) + a.eps);
    if (G > 64 && a.sum != nullptr) {  // not before every wave has its part of a row that it may replace, a cut chunk's first elements too
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            Chunk<RS, VE> t;
            t.from_f32(a.rdt, h[k]);
            if (lane + G * k < a.chunks) t.template store<AL>(a.sum + r * a.ss + (int64_t)at[k] * RS);
        }
    }
    if (a.gamma == nullptr) return;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        float o[VE];
        if constexpr (IN_LDS) {
#pragma unroll
            for (int i = 0; i < VE; ++i) o[i] = gam[at[k] + i];
        } else {
            features<VE>(a.gamma, a.gadt, at[k], o);
#pragma unroll
            for (int i = 0; i < VE; ++i) o[i] *= a.scale;
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = over(h[k][i] * o[i], root);
        const bool mine = valid && lane + G * k < a.chunks;
        if (a.odt == MXFP4) {
            const int c = lane + G * k;
            if constexpr (!AL) {  // a cut chunk back to its place, zeros behind it
                const int move = c * VE - at[k];
#pragma unroll
                for (int s = VE / 2; s > 0; s /= 2) {
#pragma unroll
                    for (int i = 0; i < VE; ++i) o[i] = (move & s) != 0 ? (i + s < VE ? o[i + s] : 0.0f) : o[i];
                }
            }
            uint32_t size = 0;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                if (c >= a.chunks) o[i] = 0.0f;
                size = max(size, mx_size(o[i]));
            }
            const uint32_t code = mx_scale_code(mx_group_size<32 / VE>(size));
            if (valid && c < a.padded) {
                if constexpr (VE == 8) *reinterpret_cast<uint32_t*>(a.out + r * a.os + c * 4) = mx_pack8(o, mx_scale_operand(code));
                else *reinterpret_cast<uint16_t*>(a.out + r * a.os + c * 2) = (uint16_t)mx_pack4(o, mx_scale_operand(code));
                if (c % (32 / VE) == 0) a.oscales[r * a.oss + c / (32 / VE)] = (uint8_t)code;
            }
        } else if (mine) {
            if (VE == 4 && a.odt == F32) {
                Chunk<4, 4> t;
                float f[4] = {o[0], o[1], o[2], o[3]};
                t.from_f32(F32, f);
                t.template store<AL>(a.out + r * a.os + (int64_t)at[k] * 4);
            } else {
                Chunk<2, VE> t;
                t.from_f32(a.odt, o);
                t.template store<AL>(a.out + r * a.os + (int64_t)at[k] * 2);
            }
        }
    }
}

// Rows too long for registers and too short for a chunk: a wave per row, element by element, three passes.
__global__ __launch_bounds__(kThreads) void block_norm_loop_kernel(BlockNormArgs a) {
    const int lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * (kThreads / 64) + threadIdx.x / 64;
    if (row >= a.rows) return;  // the whole wave
    const int64_t r = row;
    const char *rp = a.res + r * a.rs, *up = a.upd + r * a.us, *gp = a.gate;
    if (gp != nullptr) {
        uint32_t d, m;
        fdivmod(fdiv(a.row0 + row, a.inner), a.period, d, m);
        gp += m * a.gs;
    }
    float root = 1.0f;
    if (a.post_gamma != nullptr) {
        float ss = 0.0f;
        for (int d = lane; d < a.dim; d += 64) {
            const float u = load1(up, a.udt, d);
            ss = fmaf(u, u, ss);
        }
        root = sqrtf(group_sum<64>(ss) + a.eps);
    }
    const float row_gate = gp != nullptr && !a.gate_vec ? gate_value(load1(gp, a.gdt, 0), a.gate_logit) : 1.0f;
    auto sum_at = [&](int d) {
        float u = load1(up, a.udt, d);
        if (a.post_gamma != nullptr) u = u * (load1(a.post_gamma, a.pdt, d) * a.post_scale) / root;
        if (a.ls != nullptr) u *= load1(a.ls, a.ldt, d);
        u *= a.gate_vec ? gate_value(load1(gp, a.gdt, d), a.gate_logit) : row_gate;
        return round_through(fmaf(u, a.alpha, load1(rp, a.rdt, d)), a.rdt);
    };
    float ss = 0.0f;
    for (int d = lane; d < a.dim; d += 64) {
        const float h = sum_at(d);
        if (a.sum != nullptr) store1(a.sum + r * a.ss, a.rdt, d, h);
        ss = fmaf(h, h, ss);
    }
    if (a.gamma == nullptr) return;
    const float sum_root = sqrtf(group_sum<64>(ss) + a.eps);
    for (int d0 = 0; d0 < a.dim; d0 += 64) {
        const int d = d0 + lane;
        float o = 0.0f;
        if (d < a.dim)  // the stored sum again: it may lie in the residual's place
            o = (a.sum != nullptr ? load1(a.sum + r * a.ss, a.rdt, d) : sum_at(d)) * (load1(a.gamma, a.gadt, d) * a.scale) / sum_root;
        if (a.odt != MXFP4) {
            if (d < a.dim) store1(a.out + r * a.os, a.odt, d, o);
            continue;
        }
        uint32_t size = mx_size(o);
#pragma unroll
        for (int s = 1; s < 32; s *= 2) size = max(size, (uint32_t)__shfl_xor((int)size, s));
        const uint32_t code = mx_scale_code(size);
        const float next = __shfl_xor(o, 1);
        if (d < 32 * ((a.dim + 31) / 32) && d % 2 == 0) {
            const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, o, next, mx_scale_operand(code), 0);
            reinterpret_cast<uint8_t*>(a.out + r * a.os)[d / 2] = (uint8_t)w;
            if (d % 32 == 0) a.oscales[r * a.oss + d / 32] = (uint8_t)code;
        }
    }
}

template <int VE, int RS, int US, int GS, bool AL>
bool launch_shape(const BlockNormArgs& a, hipStream_t st) {
    auto go = [&](auto g, auto nc) {
        constexpr int G = decltype(g)::value, NC = decltype(nc)::value;
        hipLaunchKernelGGL((block_norm_kernel<VE, RS, US, GS, G, NC, AL>), dim3((unsigned)ceil_div(a.rows, kThreads / G)),
                           dim3(kThreads), (G < kThreads ? 3 * a.dim : 8) * sizeof(float), st, a);
    };
    typedef std::integral_constant<int, 16> G16;
    typedef std::integral_constant<int, 64> G64;
    typedef std::integral_constant<int, 256> G256;
    const int n = a.odt == MXFP4 ? a.padded : a.chunks;
    // A block per row from 129 chunks on, whose loads are spread over more lanes: us, a wave and a block per row, bf16 [12, 1500] 5.6
    // and 4.6, [1800, 1536] 8.7 and 8.5, [3000, 1536] 11.8 and 11.3.  But of many rows of up to 192 half a block's lanes would have
    // next to nothing: bf16 [5000, 1536] 15.5 and 15.7, [12000, 1536] 29 and 36; f32 [6000, 768] 12.0 and 14.0, [18786, 526] 27.6 and 37.
    if (n <= 32) go(G16(), std::integral_constant<int, 2>());
    else if (n <= 64) go(G16(), std::integral_constant<int, 4>());
    else if (n <= 96) go(G16(), std::integral_constant<int, 6>());
    else if (n <= 128) go(G64(), std::integral_constant<int, 2>());
    else if (n <= 192 && a.rows >= 16 * cu_count()) go(G64(), std::integral_constant<int, 3>());
    else if (n <= 256) go(G256(), std::integral_constant<int, 1>());
    else if (n <= 512) go(G256(), std::integral_constant<int, 2>());
    else if (n <= 1024) go(G256(), std::integral_constant<int, 4>());
    else if constexpr (VE == 4) {
        if (n > 2048) return false;
        go(G256(), std::integral_constant<int, 8>());
    } else {
        return false;
    }
    return true;
}

template <int VE, bool AL>
bool launch_sizes(const BlockNormArgs& a, int gate_bytes, hipStream_t st) {
    if constexpr (VE == 8) {
        return gate_bytes == 0 ? launch_shape<8, 2, 2, 0, AL>(a, st) : launch_shape<8, 2, 2, 2, AL>(a, st);
    } else {
        auto with_gate = [&](auto rs, auto us) {
            constexpr int R = decltype(rs)::value, U = decltype(us)::value;
            return gate_bytes == 0   ? launch_shape<4, R, U, 0, AL>(a, st)
                   : gate_bytes == 2 ? launch_shape<4, R, U, 2, AL>(a, st)
                                     : launch_shape<4, R, U, 4, AL>(a, st);
        };
        typedef std::integral_constant<int, 2> B2;
        typedef std::integral_constant<int, 4> B4;
        if (a.rdt == F32) return a.udt == F32 ? with_gate(B4(), B4()) : with_gate(B4(), B2());
        return a.udt == F32 ? with_gate(B2(), B4()) : with_gate(B2(), B2());
    }
}

int launch_block_norm(BlockNormArgs a, hipStream_t st, const char* op) {
    const bool wide = a.rdt == F32 || a.udt == F32 || (a.gate_vec && a.gdt == F32) || a.odt == F32;
    const int ve = wide ? 4 : 8, gate_bytes = a.gate_vec ? dt_size(a.gdt) : 0;
    a.chunks = (int)ceil_div(a.dim, ve);
    a.padded = (int)ceil_div(a.dim, 32) * (32 / ve);
    bool vec = false, al = false;
    if (a.dim >= ve && a.dim <= 8192) {
        auto even = [&](const void* p, int64_t stride, int dt) {
            const int64_t b = (int64_t)ve * dt_size(dt);
            return p == nullptr || (aligned(p, b) && stride % b == 0);
        };
        al = a.dim % ve == 0 && even(a.res, a.rs, a.rdt) && even(a.upd, a.us, a.udt) && even(a.sum, a.ss, a.rdt) &&
             (a.odt == MXFP4 || even(a.out, a.os, a.odt)) && (!a.gate_vec || even(a.gate, a.gs, a.gdt));
        vec = true;
    }
    // a launch has fewer than 2^32 threads, up to 256 of them to a row
    const int64_t rows = a.rows, step = int64_t(1) << 23;
    for (int64_t r0 = 0; r0 < rows; r0 += step) {
        BlockNormArgs p = a;
        p.row0 = (uint32_t)r0;
        p.rows = (uint32_t)std::min(step, rows - r0);
        p.res += r0 * a.rs;
        p.upd += r0 * a.us;
        if (a.sum != nullptr) p.sum += r0 * a.ss;
        if (a.out != nullptr) p.out += r0 * a.os;
        if (a.oscales != nullptr) p.oscales += r0 * a.oss;
        bool done = false;
        if (vec && wide) done = al ? launch_sizes<4, true>(p, gate_bytes, st) : launch_sizes<4, false>(p, gate_bytes, st);
        else if (vec) done = al ? launch_sizes<8, true>(p, gate_bytes, st) : launch_sizes<8, false>(p, gate_bytes, st);
        if (!done)
            hipLaunchKernelGGL(block_norm_loop_kernel, dim3((unsigned)ceil_div(p.rows, kThreads / 64)), dim3(kThreads), 0, st, p);
    }
    return check_launch(op);
}

}  // namespace
}  // namespace mbrt

using namespace mbrt;

extern "C" int mbrt_block_norm(const void* residual, int residual_dtype, int64_t residual_row_stride, const void* update,
                               int update_dtype, int64_t update_row_stride, const void* post_gamma, int post_gamma_dtype,
                               const void* gate, int gate_dtype, int64_t gate_cols, int64_t gate_row_stride,
                               int64_t gate_inner, int64_t gate_period, int gate_is_logit, const void* layer_scale,
                               int layer_scale_dtype, const void* gamma, int gamma_dtype, void* sum_out,
                               int64_t sum_row_stride, void* normed, int normed_dtype, int64_t normed_row_stride,
                               void* normed_scales, int64_t normed_scales_row_stride, int64_t rows, int64_t dim, float alpha,
                               float post_scale, float scale, float eps, mbrt_stream_t stream) {
    const char* op = "mbrt_block_norm";
    MBRT_REQUIRE_FLOAT_DT(residual_dtype, op);
    MBRT_REQUIRE_FLOAT_DT(update_dtype, op);
    const bool mx = gamma != nullptr && normed_dtype == MXFP4;
    if (gamma && !mx) MBRT_REQUIRE_FLOAT_DT(normed_dtype, op);
    MBRT_REQUIRE((!post_gamma || is_float_dt(post_gamma_dtype)) && (!gate || is_float_dt(gate_dtype)) &&
                     (!layer_scale || is_float_dt(layer_scale_dtype)) && (!gamma || is_float_dt(gamma_dtype)),
                 MBRT_E_UNSUPPORTED_DTYPE, "%s: a gamma's, the gate's or the layer scale's dtype (expected F32/F16/BF16)", op);
    MBRT_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && dim >= 1 && dim < (int64_t(1) << 28), MBRT_E_SHAPE,
                 "%s: bad shape rows=%lld dim=%lld (fewer than 2^31 rows, 1 to 2^28 - 1 features)", op, (long long)rows,
                 (long long)dim);
    MBRT_REQUIRE(!gate || ((gate_cols == 1 || gate_cols == dim) && gate_inner >= 1 && gate_period >= 1 && gate_row_stride >= 0),
                 MBRT_E_SHAPE, "%s: gate of %lld columns, inner %lld, period %lld", op, (long long)gate_cols,
                 (long long)gate_inner, (long long)gate_period);
    if (rows == 0) return MBRT_OK;
    const int64_t blocks = ceil_div(dim, kMxBlock);
    const int64_t rb = dt_size(residual_dtype), ub = dt_size(update_dtype), ob = mx ? 1 : gamma ? dt_size(normed_dtype) : 1;
    const int64_t ocols = mx ? 16 * blocks : dim;
    if (rows == 1) {  // of a single row: not used
        residual_row_stride = update_row_stride = sum_row_stride = dim;
        normed_row_stride = ocols;
        normed_scales_row_stride = blocks;
    }
    MBRT_REQUIRE(residual_row_stride >= 0 && update_row_stride >= 0 && (!sum_out || sum_row_stride >= dim) &&
                     (!gamma || normed_row_stride >= ocols) && (!mx || normed_scales_row_stride >= blocks),
                 MBRT_E_SHAPE, "%s: negative row stride, or output rows that overlap", op);
    MBRT_REQUIRE(residual && update && (gamma ? normed != nullptr : sum_out != nullptr) && (!mx || normed_scales),
                 MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(residual, rb) && aligned(update, ub) && (!sum_out || aligned(sum_out, rb)) &&
                     (!gamma || (mx ? aligned(normed, 16) && normed_row_stride % 16 == 0 : aligned(normed, ob))) &&
                     (!gate || aligned(gate, dt_size(gate_dtype))) && (!gamma || aligned(gamma, dt_size(gamma_dtype))) &&
                     (!post_gamma || aligned(post_gamma, dt_size(post_gamma_dtype))) &&
                     (!layer_scale || aligned(layer_scale, dt_size(layer_scale_dtype))),
                 MBRT_E_ALIGN, "%s: pointer not aligned to its elements, or rows of codes not to 16 bytes", op);
    const int64_t gate_rows = gate ? std::min(gate_period, ceil_div(rows, gate_inner)) : 0;
    if (gate_rows == 1) gate_row_stride = 0;
    const MemRows R{residual, residual_row_stride * rb, dim * rb, rows}, U{update, update_row_stride * ub, dim * ub, rows};
    const MemRows S{sum_out, sum_row_stride * rb, dim * rb, sum_out ? rows : 0};
    const MemRows O{normed, normed_row_stride * ob, ocols * ob, gamma ? rows : 0};
    const MemRows C{normed_scales, normed_scales_row_stride, blocks, mx ? rows : 0};
    const MemRows Ga{gate, gate_row_stride * (gate ? dt_size(gate_dtype) : 0), gate_cols * (gate ? dt_size(gate_dtype) : 0), gate_rows};
    const MemRows V[3] = {{gamma, 0, gamma ? dim * dt_size(gamma_dtype) : 0, 1},
                          {post_gamma, 0, post_gamma ? dim * dt_size(post_gamma_dtype) : 0, 1},
                          {layer_scale, 0, layer_scale ? dim * dt_size(layer_scale_dtype) : 0, 1}};
    const bool sum_in_place = sum_out == residual && (rows == 1 || sum_row_stride == residual_row_stride);
    const bool out_in_place = gamma && !mx && normed == update && normed_dtype == update_dtype &&
                              (rows == 1 || normed_row_stride == update_row_stride);
    bool clash = (!sum_in_place && rows_meet(S, R)) || rows_meet(S, U) || rows_meet(S, Ga) || rows_meet(S, O) || rows_meet(S, C) ||
                 rows_meet(O, R) || (!out_in_place && rows_meet(O, U)) || rows_meet(O, Ga) || rows_meet(O, C) || rows_meet(C, R) ||
                 rows_meet(C, U) || rows_meet(C, Ga);
    for (const MemRows& v : V) clash = clash || rows_meet(v, S) || rows_meet(v, O) || rows_meet(v, C);
    MBRT_REQUIRE(!clash, MBRT_E_INVALID_ARG,
                 "%s: an output overlaps another operand (sum_out may be the residual, normed the update, in the same dtype and rows)",
                 op);
    BlockNormArgs a{};
    a.res = static_cast<const char*>(residual);
    a.upd = static_cast<const char*>(update);
    a.gate = static_cast<const char*>(gate);
    a.gamma = gamma;
    a.post_gamma = post_gamma;
    a.ls = layer_scale;
    a.sum = static_cast<char*>(sum_out);
    a.out = static_cast<char*>(normed);
    a.oscales = static_cast<uint8_t*>(normed_scales);
    a.rs = residual_row_stride * rb;
    a.us = update_row_stride * ub;
    a.gs = gate ? gate_row_stride * dt_size(gate_dtype) : 0;
    a.ss = sum_row_stride * rb;
    a.os = normed_row_stride * ob;
    a.oss = normed_scales_row_stride;
    a.rows = (uint32_t)rows;
    a.dim = (int)dim;
    a.rdt = residual_dtype;
    a.udt = update_dtype;
    a.gdt = gate_dtype;
    a.odt = gamma ? normed_dtype : residual_dtype;
    a.gadt = gamma_dtype;
    a.pdt = post_gamma_dtype;
    a.ldt = layer_scale_dtype;
    a.gate_vec = gate && gate_cols > 1;
    a.gate_logit = gate_is_logit != 0;
    // rows / inner and the rows of a period stay below 2^31
    a.inner = make_fastdiv((uint32_t)std::min<int64_t>(gate ? gate_inner : 1, rows));
    a.period = make_fastdiv((uint32_t)std::min<int64_t>(gate ? gate_period : 1, rows));
    a.alpha = alpha;
    a.post_scale = post_scale;
    a.scale = scale;
    a.eps = eps;
    return launch_block_norm(a, as_stream(stream), op);
}
