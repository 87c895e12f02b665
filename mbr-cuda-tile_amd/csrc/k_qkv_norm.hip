// Split of a fused qkv projection with the RMS norms of each query and key head and the rotary rotation in the
// same pass (the heads of src/mbr_cuda_tile.cu:6058-6213 with norms before their rotation): for head vector x of q or k
// at token n,
//   y = x * scale * gamma / sqrt(sum x^2 + eps),   (y0, y1) -> (y0 c - y1 s, y0 s + y1 c)
// with c, s row pos0 + n of the tables; v is copied.  All in f32, rounded once, on the store.
//
// Bound by memory: each element is read and written once.  G lanes hold one head vector, 16 bytes each, and reduce
// its sum of squares with DPP adds; a token has S such groups side by side (a wave, where it has the heads), which walk
// its heads, so that a thread reads its cos, sin and gamma once for all of them.  MI355X: bf16 [60, 801] with 8 heads of
// 64, 295 MB, 54.8 us (5.4 TB/s; a large copy 4.8 to 5.2); f32 [7, 1301], 8 heads over 2 of 128, heads outside tokens, 113 MB,
// 25.7 us; a frame of 60 rows 4.1 to 4.4, the launch.
#include "abi_common.hpp"

#include <algorithm>

namespace mbrt {
namespace {

constexpr int kThreads = 256;

struct QkvArgs {
    const void* qkv;
    void* q;
    void* k;
    void* v;  // NULL: v is left where it is
    const void* qg;
    const void* kg;
    const void* cosp;
    const void* sinp;
    int idt, odt, gdt, tdt;
    int64_t in_bs, in_ns;                // qkv strides (batch, token)
    int64_t q_bs, q_hs, q_ns;            // q strides (batch, head, token)
    int64_t kv_bs, kv_hs, kv_ns;         // k and v
    int64_t tokens, N, pos0;             // tokens = B * N
    int H, KV, D, heads;                 // heads: H + 2 KV, or H + KV where v is left
    int G, S;                            // lanes per head vector, head vectors side by side (powers of 2)
    int lane_bits, head_bits;            // their logarithms
    FastDiv ndiv;                        // N
    float scale, eps;
};

__device__ __forceinline__ float lanes_sum(float v, int G) {
    if (G >= 2) v += dpp<0xB1>(v);
    if (G >= 4) v += dpp<0x4E>(v);
    if (G >= 8) v += dpp<0x141>(v);
    if (G >= 16) v += dpp<0x140>(v);
    if (G >= 32) v += swz_xor16(v);
    if (G >= 64) v = lane_f(v, 0) + lane_f(v, 32);
    return v;
}

// where head h of token (b, n) goes
__device__ __forceinline__ void* place(const QkvArgs& a, int64_t b, int64_t n, int h, int64_t& e) {
    if (h < a.H) {
        e = b * a.q_bs + h * a.q_hs + n * a.q_ns;
        return a.q;
    }
    const int kh = h < a.H + a.KV ? h - a.H : h - a.H - a.KV;
    e = b * a.kv_bs + kh * a.kv_hs + n * a.kv_ns;
    return h < a.H + a.KV ? a.k : a.v;
}

// LG: lanes per head vector, known here with f32 tables and gammas (every load of a thread is then issued before it waits
// for one: a call for one frame 4.4 -> 4.1 us), or 0: all at run time.
template <int IDT, int ODT, int LG>
__global__ __launch_bounds__(kThreads) void qkv_norm_vec_kernel(QkvArgs a) {
    constexpr int VE = (IDT == F32 || ODT == F32) ? 4 : 8;
    constexpr int U = 4;  // head vectors in flight per thread
    // tokens per block: 256 / (G S), at least 4
    const int G = LG ? LG : a.G;
    const uint32_t bits = (uint32_t)(a.lane_bits + a.head_bits);
    const int c = (int)threadIdx.x & (G - 1), slot = ((int)threadIdx.x >> a.lane_bits) & (a.S - 1);
    const uint32_t at = blockIdx.x * (kThreads >> bits) + (threadIdx.x >> bits);
    const bool live = at < (uint32_t)a.tokens && c * VE < a.D;
    const uint32_t token = min(at, (uint32_t)a.tokens - 1);
    const int d = min(c * VE, a.D - VE);
    uint32_t b32, n32;
    fdivmod(token, a.ndiv, b32, n32);
    const int64_t b = b32, n = n32;
    const int64_t src = b * a.in_bs + n * a.in_ns + d, tab = (a.pos0 + n) * (a.D / 2) + d / 2;
    Vec<IDT, VE> in[U];
    auto load_heads = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u) in[u].load(a.qkv, src + (int64_t)min(h0 + u * a.S, a.heads - 1) * a.D);
    };
    load_heads(slot);
    float cs[VE / 2], sn[VE / 2], qg[VE], kg[VE];
    if (LG || a.tdt == F32) {
        Vec<F32, VE / 2> cv, sv;
        cv.load(a.cosp, tab);
        sv.load(a.sinp, tab);
        cv.to_f32(cs);
        sv.to_f32(sn);
    } else {
        Vec<BF16, VE / 2> cv, sv;
        cv.load(a.cosp, tab);
        sv.load(a.sinp, tab);
        cv.to_f32(cs);
        sv.to_f32(sn);
    }
    vload<VE>(a.qg, LG ? (int)F32 : a.gdt, d, qg);
    vload<VE>(a.kg, LG ? (int)F32 : a.gdt, d, kg);
    for (int h0 = slot; h0 < a.heads + slot; h0 += U * a.S) {  // the same number of rounds in every lane
        if (h0 > slot) load_heads(h0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * a.S;
            float x[VE];
            in[u].to_f32(x);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; ++i) ss = fmaf(x[i], x[i], ss);
            ss = lanes_sum(c * VE < a.D ? ss : 0.0f, G);
            if (h < a.H + a.KV) {
                const float inv = a.scale / sqrtf(ss + a.eps);
                const bool isq = h < a.H;
#pragma unroll
                for (int i = 0; i < VE; ++i) x[i] = x[i] * inv * (isq ? qg[i] : kg[i]);
                rotate<VE>(x, cs, sn);
            }
            if (live && h < a.heads) {
                int64_t e;
                void* dst = place(a, b, n, h, e);
                Vec<ODT, VE> o;
                o.from_f32(x);
                o.store(dst, e + d);
            }
        }
    }
}

// Any even D, any alignment: a wave per head vector, an element per lane and access.  One unaligned pointer or stride takes
// the whole call here: the [60, 801] above with tokens 1537 elements apart 444 us, with heads of 66 497, the f32 one 50; a frame
// of 60 rows 3.8, as the other kernel.
__global__ __launch_bounds__(kThreads) void qkv_norm_any_kernel(QkvArgs a) {
    const int lane = threadIdx.x % 64;
    const int64_t vecs = a.tokens * a.heads, waves = (int64_t)gridDim.x * (kThreads / 64);
    const int half = a.D / 2;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; i < vecs; i += waves) {
        const int64_t token = i / a.heads, b = token / a.N, n = token - b * a.N;
        const int h = (int)(i - token * a.heads);
        const int64_t src = b * a.in_bs + n * a.in_ns + (int64_t)h * a.D;
        int64_t e;
        void* dst = place(a, b, n, h, e);
        if (h >= a.H + a.KV) {
            for (int d = lane; d < a.D; d += 64) store1(dst, a.odt, e + d, load1(a.qkv, a.idt, src + d));
            continue;
        }
        float ss = 0.0f;
        for (int d = lane; d < a.D; d += 64) {
            const float x = load1(a.qkv, a.idt, src + d);
            ss = fmaf(x, x, ss);
        }
        const float inv = a.scale / sqrtf(lanes_sum(ss, 64) + a.eps);
        const void* gamma = h < a.H ? a.qg : a.kg;
        for (int p = lane; p < half; p += 64) {
            const float x0 = load1(a.qkv, a.idt, src + 2 * p) * inv * load1(gamma, a.gdt, 2 * p);
            const float x1 = load1(a.qkv, a.idt, src + 2 * p + 1) * inv * load1(gamma, a.gdt, 2 * p + 1);
            const float cv = load1(a.cosp, a.tdt, (a.pos0 + n) * half + p), sv = load1(a.sinp, a.tdt, (a.pos0 + n) * half + p);
            float y0, y1;
            rotate_pair(x0, x1, cv, sv, y0, y1);
            store1(dst, a.odt, e + 2 * p, y0);
            store1(dst, a.odt, e + 2 * p + 1, y1);
        }
    }
}

}  // namespace
}  // namespace mbrt

using namespace mbrt;

extern "C" {

int mbrt_split_qkv_norm_rotary(const void* qkv, int qkv_dtype, int64_t qkv_batch_stride, int64_t qkv_token_stride,
                               const void* q_gamma, const void* k_gamma, int gamma_dtype, const void* cos_table,
                               const void* sin_table, int trig_dtype, int64_t n_pos, int64_t pos0, void* q, void* k,
                               void* v, int out_dtype, int64_t q_batch_stride, int64_t q_head_stride,
                               int64_t q_token_stride, int64_t kv_batch_stride, int64_t kv_head_stride,
                               int64_t kv_token_stride, int64_t B, int64_t N, int64_t H, int64_t H_kv, int64_t D,
                               float scale, float eps, mbrt_stream_t stream) {
    const char* op = "mbrt_split_qkv_norm_rotary";
    MBRT_REQUIRE_FLOAT_DT(qkv_dtype, op);
    MBRT_REQUIRE_FLOAT_DT(out_dtype, op);
    MBRT_REQUIRE(gamma_dtype == F32 || gamma_dtype == BF16, MBRT_E_UNSUPPORTED_DTYPE, "%s: gamma dtype %d", op,
                 gamma_dtype);
    MBRT_REQUIRE(trig_dtype == F32 || trig_dtype == BF16, MBRT_E_UNSUPPORTED_DTYPE, "%s: trig dtype %d", op,
                 trig_dtype);
    MBRT_REQUIRE(D >= 2 && D % 2 == 0 && D <= 1 << 16, MBRT_E_SHAPE, "%s: dim_head must be even, 2 to 65536", op);
    MBRT_REQUIRE(B >= 0 && N >= 0 && H >= 1 && H_kv >= 1 && H <= 1 << 16 && H_kv <= 1 << 16, MBRT_E_SHAPE,
                 "%s: bad shape", op);
    MBRT_REQUIRE(pos0 >= 0 && pos0 <= n_pos && N <= n_pos - pos0, MBRT_E_SHAPE,
                 "%s: positions %lld .. %lld of a table of %lld", op, (long long)pos0, (long long)(pos0 + N),
                 (long long)n_pos);
    int64_t st[8] = {qkv_batch_stride, qkv_token_stride, q_batch_stride, q_head_stride, q_token_stride,
                     kv_batch_stride, kv_head_stride, kv_token_stride};
    const int64_t dim[8] = {B, N, B, H, N, B, H_kv, N};
    for (int i = 0; i < 8; ++i) {
        MBRT_REQUIRE(st[i] >= 0, MBRT_E_SHAPE, "%s: negative stride", op);
        if (dim[i] <= 1) st[i] = 0;  // of a single index: not used
    }
    MBRT_REQUIRE(B < (int64_t(1) << 31) && N < (int64_t(1) << 31), MBRT_E_SHAPE, "%s: dimension beyond 2^31", op);
    for (int i = 0; i < 2; ++i) {  // q, then k and v
        const int64_t* s = st + 2 + 3 * i;
        MBRT_REQUIRE((B <= 1 || s[0] > 0) && ((i ? H_kv : H) == 1 || s[1] > 0) && (N <= 1 || s[2] > 0), MBRT_E_SHAPE,
                     "%s: heads of an output overlap", op);
    }
    if (B == 0 || N == 0) return MBRT_OK;
    MBRT_REQUIRE(qkv && q && k && q_gamma && k_gamma && cos_table && sin_table, MBRT_E_INVALID_ARG, "%s: NULL pointer",
                 op);
    const uintptr_t es = dt_size(qkv_dtype), os = dt_size(out_dtype), gs = dt_size(gamma_dtype), ts = dt_size(trig_dtype);
    MBRT_REQUIRE(aligned(qkv, es) && aligned(q, os) && aligned(k, os) && aligned(v, os) && aligned(q_gamma, gs) &&
                     aligned(k_gamma, gs) && aligned(cos_table, ts) && aligned(sin_table, ts),
                 MBRT_E_ALIGN, "%s: pointer not aligned to its elements", op);
    QkvArgs a{};
    a.qkv = qkv;
    a.q = q;
    a.k = k;
    a.v = v;
    a.qg = q_gamma;
    a.kg = k_gamma;
    a.cosp = cos_table;
    a.sinp = sin_table;
    a.idt = qkv_dtype;
    a.odt = out_dtype;
    a.gdt = gamma_dtype;
    a.tdt = trig_dtype;
    a.in_bs = st[0];
    a.in_ns = st[1];
    a.q_bs = st[2];
    a.q_hs = st[3];
    a.q_ns = st[4];
    a.kv_bs = st[5];
    a.kv_hs = st[6];
    a.kv_ns = st[7];
    a.tokens = B * N;
    a.N = N;
    a.pos0 = pos0;
    a.H = (int)H;
    a.KV = (int)H_kv;
    a.D = (int)D;
    a.heads = (int)(H + (v ? 2 : 1) * H_kv);
    a.scale = scale;
    a.eps = eps;
    hipStream_t stm = as_stream(stream);
    const int ve = (qkv_dtype == F32 || out_dtype == F32) ? 4 : 8;
    // one vector access each: ve elements of the input and of the outputs, ve / 2 of the tables, up to 16 bytes
    bool vec = D % ve == 0 && D / ve <= 64 && aligned(qkv, ve * es) && aligned(q, ve * os) && aligned(k, ve * os) &&
               aligned(v, ve * os) && aligned(q_gamma, std::min<uintptr_t>(16, ve * gs)) &&
               aligned(k_gamma, std::min<uintptr_t>(16, ve * gs)) && aligned(cos_table, ve / 2 * ts) &&
               aligned(sin_table, ve / 2 * ts);
    for (int i = 0; i < 8; ++i) vec = vec && st[i] % ve == 0;
    if (vec) {
        a.G = 1;
        while (a.G * ve < D) a.G *= 2;
        a.S = 64 / a.G;
        while (a.S > a.heads) a.S /= 2;
        for (int i = 1; i < a.G; i *= 2) ++a.lane_bits;
        for (int i = 1; i < a.S; i *= 2) ++a.head_bits;
        a.ndiv = make_fastdiv((uint32_t)N);
        const int64_t blocks = ceil_div(a.tokens * a.G * a.S, kThreads);
        vec = a.tokens < (int64_t(1) << 31) && grid_fits(blocks, kThreads);  // 32-bit token numbers
        if (vec)
            with_dt(qkv_dtype, [&](auto it) {
                with_dt(out_dtype, [&](auto ot) {
                    constexpr int I = decltype(it)::value, O = decltype(ot)::value;
                    const dim3 grid((unsigned)blocks);
                    const bool f32 = gamma_dtype == F32 && trig_dtype == F32;
                    if (f32 && a.G == 8) hipLaunchKernelGGL((qkv_norm_vec_kernel<I, O, 8>), grid, dim3(kThreads), 0, stm, a);
                    else if (f32 && a.G == 16) hipLaunchKernelGGL((qkv_norm_vec_kernel<I, O, 16>), grid, dim3(kThreads), 0, stm, a);
                    else if (f32 && a.G == 32) hipLaunchKernelGGL((qkv_norm_vec_kernel<I, O, 32>), grid, dim3(kThreads), 0, stm, a);
                    else hipLaunchKernelGGL((qkv_norm_vec_kernel<I, O, 0>), grid, dim3(kThreads), 0, stm, a);
                });
            });
    }
    if (!vec)
        hipLaunchKernelGGL(qkv_norm_any_kernel,
                           dim3((unsigned)std::min<int64_t>(ceil_div(a.tokens * a.heads, kThreads / 64), 1 << 16)),
                           dim3(kThreads), 0, stm, a);
    return check_launch(op);
}

}  // extern "C"
