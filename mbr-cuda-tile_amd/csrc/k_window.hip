// Attention through a sliding window with sinks, on MFMA, for bf16 or f16 heads of 32, 64 or 128: the fused
// attention's companion for long songs and for streaming (mbrt_attention_window's comment in mbrt.h holds the
// definition).  Key j is visible to the query at position p iff
//   j < len_b,  j <= p + right,  and  j >= p - left or j < sinks.
//
// Query rows: the H / H_kv query heads that share a key head are rows of one matrix, row r = (query r / G, head
// r % G), so that each key and value is read once for all of them.
// Keys: what the rows of a tile may see is one list, the sinks before the window and then the window's keys lo .. hi
// of all its rows: t -> j = t < s ? t : lo + t - s, with s <= lo, which loads by rows and never touches a
// key outside.  Whatever stands in keys that no row of the tile sees (NaN behind a sequence's end) is not read.
//
// Per 32 keys, with v_mfma_f32_16x16x32 (lane l = (g, c): A[c][8 g + j], B[8 g + j][c], C[4 g + i][c]):
//   S^T = K Q^T      A = K rows, B = the wave's 16 query rows: lane (g, c) holds S^T[key 16 kb + 4 g + i][row c].
//   online softmax   per row c, as in the fused attention: the exponent's reference m moves only when a score
//                    outgrows it by 2^8, each lane sums its own keys' p, the four lanes of a row are added at the end.
//   O^T += V^T P^T   B = P^T from the S^T registers: slot j of lane group g is key 4 g + j, or 16 + 4 g + j - 4 from
//                    j = 4 on; A = V^T by LDS transpose reads.  P enters as a sum of two or three values of the
//                    2-byte type (split_p), so that only the inputs' and the output's own rounding is left.
// A-row 4 q + j of block db of four is column 64 (db / 4) + 16 q + 4 (db % 4) + j, so that a lane ends with 16
// neighbouring columns of its row (of two blocks for D = 32: 8 q + 4 db + j, 8 columns).
//
// A value that a row does not see but another row of its tile does enters the product with weight 0.  Where that
// value is infinite or NaN the product is NaN; a row that ends with anything not finite is computed again from the
// keys that it sees alone (row_alone), so that the definition holds for it too.
#include "abi_common.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace mbrt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLazy = 8.0f;  // log2 units the running max may outgrow the exponent's reference
constexpr int kTile = 64;      // keys per LDS tile
constexpr int kChunk = 32;     // keys per arithmetic step

struct WinArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    void* out;
    const int32_t* lens;
    const void* gate;
    float* ws;
    int64_t q_bs, q_hs, q_ns, kv_bs, kv_hs, kv_ns, o_bs, o_hs, o_ns;  // elements
    int nq, nk, rows;        // rows = nq * G
    int H, KV;
    int left, right, sinks, start;  // left, right -1: no limit; start -1: queries at the end
    int gdt, glogit, odt;
    float sl2;               // scale * log2(e)
    uint32_t qtiles, splits;
    FastDiv gdiv, kvdiv;     // G, KV
};

// The keys that the query rows qa .. qb of a batch entry may see, as one list.
struct Span {
    int len, start;          // the entry's keys, position of its query 0
    int lo, hi, s, count;
    __device__ __forceinline__ int key(int t) const { return t < s ? t : lo + t - s; }
};

__device__ __forceinline__ Span make_span(const WinArgs& a, int b, int qa, int qb) {
    Span p;
    p.len = a.nk;
    if (a.lens != nullptr) p.len = min(max(a.lens[b], 0), a.nk);
    p.start = a.start >= 0 ? a.start : p.len - a.nq;
    p.hi = a.right < 0 ? p.len - 1 : min(p.len - 1, p.start + qb + a.right);
    p.lo = a.left < 0 ? 0 : max(0, p.start + qa - a.left);
    p.s = max(0, min(min(a.sinks, p.lo), p.hi + 1));
    p.count = p.s + max(0, p.hi - p.lo + 1);
    return p;
}

template <int DT>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two values of P as NP 2-byte values each: bf16 truncated (exact difference) and the last part rounded, f16 rounded to
// nearest each time (exact differences too; p <= 2^8, and parts below 2^-24 are lost beside a row sum of 1 or more).  Two
// parts of bf16 hold 17 bits and of f16 22; an f32 output of bf16 heads takes three, 24 bits.
template <int DT, int NP>
__device__ __forceinline__ void split_p(float p0, float p1, uint32_t (&w)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        if constexpr (DT == BF16) {
            if (i == NP - 1) {
                w[i] = pack_bf16x2(p0, p1);
            } else {
                const uint32_t b0 = __float_as_uint(p0) & 0xffff0000u, b1 = __float_as_uint(p1) & 0xffff0000u;
                w[i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
                p0 -= __uint_as_float(b0);
                p1 -= __uint_as_float(b1);
            }
        } else {
            w[i] = pack_f16x2(p0, p1);
            const f32x2 h = unpack_f16x2(w[i]);
            p0 -= h.x;
            p1 -= h.y;
        }
    }
}

template <int DT>
__device__ __forceinline__ float elem(const uint16_t* p, int64_t i) {
    if constexpr (DT == BF16) return __uint_as_float((uint32_t)p[i] << 16);
    else return (float)__builtin_bit_cast(_Float16, p[i]);
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// K and V tiles in LDS: rows of D 2-byte elements in 16-byte pieces, piece j of row r at j ^ swz(r): eight
// neighbouring rows' pieces j fall on different banks (rows of 64 bytes: two rows to a line of banks).
template <int D>
__device__ __forceinline__ int swz(int r) { return D >= 64 ? (r & 7) : ((r >> 1) & 3); }

// Transpose reads of V^T fragments for 32 keys: rows r and r + 16 (HI bytes further) at NB addresses.
template <int HI, int NB>
__device__ __forceinline__ void lds_read_vt(const uint32_t (&ad)[NB], uint32_t off, u32x4 (&va)[NB]) {
    static_assert(NB == 4 || NB == 2, "blocks per group");
    u32x2 r[2 * NB];
    if constexpr (NB == 4) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\t"
            "ds_read_b64_tr_b16 %1, %8 offset:%[hi]\n\t"
            "ds_read_b64_tr_b16 %2, %9\n\t"
            "ds_read_b64_tr_b16 %3, %9 offset:%[hi]\n\t"
            "ds_read_b64_tr_b16 %4, %10\n\t"
            "ds_read_b64_tr_b16 %5, %10 offset:%[hi]\n\t"
            "ds_read_b64_tr_b16 %6, %11\n\t"
            "ds_read_b64_tr_b16 %7, %11 offset:%[hi]\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
            : "v"(ad[0] + off), "v"(ad[1] + off), "v"(ad[2] + off), "v"(ad[3] + off), [hi] "n"(HI)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %4\n\t"
            "ds_read_b64_tr_b16 %1, %4 offset:%[hi]\n\t"
            "ds_read_b64_tr_b16 %2, %5\n\t"
            "ds_read_b64_tr_b16 %3, %5 offset:%[hi]\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
            : "v"(ad[0] + off), "v"(ad[1] + off), [hi] "n"(HI)
            : "memory");
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) va[i] = u32x4{r[2 * i].x, r[2 * i].y, r[2 * i + 1].x, r[2 * i + 1].y};
}

// 16 bytes per lane from the lane's own p straight to lds + 16 lane.  Not a template: the builtin's operands must not
// depend on one, or the host pass drops the kernel that holds it.
__device__ __forceinline__ void load_to_lds(const uint16_t* p, char* lds) {
    __builtin_amdgcn_global_load_lds((global_void*)p, (lds_void*)lds, 16, 0, 0);
}

template <int D>
struct Cols {
    static constexpr int NB = D >= 64 ? 4 : 2;      // blocks of a group: a lane holds 4 NB neighbouring columns of each
    static constexpr int NG = D / (16 * NB);        // groups of 16 NB columns
};

// Running state of a wave's 16 QS rows.
template <int D, int QS>
struct State {
    f32x4 o[QS][D / 16];
    float m[QS], l[QS];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int x = 0; x < QS; ++x) {
#pragma unroll
            for (int db = 0; db < D / 16; ++db) o[x][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m[x] = -FLT_MAX;  // finite: p of a hidden key is exp2(-inf - m) = 0 also before the first visible one
            l[x] = 0.0f;
        }
    }
};

// The rows a wave works on: each lane's row c of each sub-block x, and the wave's first and last position.
template <int QS>
struct Rows {
    int jlo[QS], jhi[QS];  // window of the lane's row
    int pa, pb;
};

template <int QS>
__device__ __forceinline__ Rows<QS> make_rows(const WinArgs& a, const Span& sp, int r0, int c) {
    Rows<QS> rw;
#pragma unroll
    for (int x = 0; x < QS; ++x) {
        const int p = sp.start + (int)fdiv((uint32_t)min(r0 + 16 * x + c, a.rows - 1), a.gdiv);
        rw.jlo[x] = a.left < 0 ? 0 : p - a.left;
        rw.jhi[x] = a.right < 0 ? sp.len - 1 : min(sp.len - 1, p + a.right);
    }
    rw.pa = sp.start + (int)fdiv((uint32_t)min(r0, a.rows - 1), a.gdiv);
    rw.pb = sp.start + (int)fdiv((uint32_t)min(r0 + 16 * QS - 1, a.rows - 1), a.gdiv);
    return rw;
}

// Whether the 32 keys from t0 on are hidden from every row of the wave.
template <int QS>
__device__ __forceinline__ bool all_hidden(const WinArgs& a, const Span& sp, const Rows<QS>& rw, int t0) {
    if (t0 >= sp.count) return true;
    const int ja = sp.key(t0), jb = sp.key(min(t0 + kChunk, sp.count) - 1);
    return (a.right >= 0 && ja > rw.pb + a.right) || (a.left >= 0 && jb < rw.pa - a.left && ja >= a.sinks);
}
// Whether any of them is hidden from any.
template <int QS>
__device__ __forceinline__ bool any_hidden(const WinArgs& a, const Span& sp, const Rows<QS>& rw, int t0) {
    if (t0 + kChunk > sp.count) return true;
    const int ja = sp.key(t0), jb = sp.key(t0 + kChunk - 1);
    return (a.right >= 0 && jb > rw.pa + a.right) || (a.left >= 0 && ja < rw.pb - a.left && jb >= a.sinks);
}

// One step over the 32 keys from t0 on.  kf[kb][s]: K[16 kb + c][32 s + 8 g ..]; vad: the lane's transpose
// addresses of the V tile's row 0, voff the byte offset of the step's first row.
template <int DT, int D, int QS, int NP>
__device__ __forceinline__ void attend(const WinArgs& a, const Span& sp, const Rows<QS>& rw, int t0,
                                       const u32x4 (&kf)[2][D / 32], const u32x4 (&qf)[QS][D / 32],
                                       const uint32_t (&vad)[Cols<D>::NG][Cols<D>::NB], uint32_t voff, int g,
                                       State<D, QS>& st) {
    f32x4 s[QS][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int x = 0; x < QS; ++x) {
            s[x][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < D / 32; ++e) s[x][kb] = mma<DT>(kf[kb][e], qf[x][e], s[x][kb]);
        }
    if (any_hidden<QS>(a, sp, rw, t0)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = sp.key(t0 + 16 * kb + 4 * g + i);
#pragma unroll
                for (int x = 0; x < QS; ++x)
                    if (j > rw.jhi[x] || (j < rw.jlo[x] && j >= a.sinks)) s[x][kb][i] = -INFINITY;
            }
    }
    u32x4 pp[QS][NP];
#pragma unroll
    for (int x = 0; x < QS; ++x) {
        float mx = s[x][0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[x][kb][i]);
        if (__builtin_amdgcn_ballot_w64(mx * a.sl2 > st.m[x] + kLazy) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.sl2;
            const float mn = mx > st.m[x] + kLazy ? mx : st.m[x];
            const float alpha = __builtin_amdgcn_exp2f(st.m[x] - mn);
            st.l[x] *= alpha;
#pragma unroll
            for (int db = 0; db < D / 16; ++db) st.o[x][db] *= alpha;
            st.m[x] = mn;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[x][kb][i], a.sl2, -st.m[x]));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[x][kb][i + 1], a.sl2, -st.m[x]));
                st.l[x] += p0 + p1;
                uint32_t parts[NP];
                split_p<DT, NP>(p0, p1, parts);
#pragma unroll
                for (int n = 0; n < NP; ++n) pp[x][n][2 * kb + i / 2] = parts[n];
            }
    }
#pragma unroll
    for (int gr = 0; gr < Cols<D>::NG; ++gr) {
        u32x4 va[Cols<D>::NB];
        lds_read_vt<32 * D, Cols<D>::NB>(vad[gr], voff, va);
#pragma unroll
        for (int i = 0; i < Cols<D>::NB; ++i)
#pragma unroll
            for (int x = 0; x < QS; ++x) {
                f32x4& o = st.o[x][gr * Cols<D>::NB + i];
#pragma unroll
                for (int n = 0; n < NP; ++n) o = mma<DT>(va[i], pp[x][n], o);
            }
    }
}

// The lane's transpose addresses of a V tile: lane (g, c) points to row 4 g + c / 4, columns 16 NB gr + 4 NB (c % 4)
// + 4 i .. + 3, and receives, for column 16 NB gr + 4 NB (c / 4) + 4 i + c % 4, the four rows 4 g ...
template <int D>
__device__ __forceinline__ void v_addresses(const void* tile, int g, int c, uint32_t (&vad)[Cols<D>::NG][Cols<D>::NB]) {
    constexpr int NB = Cols<D>::NB;
    const int row = 4 * g + (c >> 2);
    const uint32_t base = lds_addr(reinterpret_cast<const char*>(tile)) + 2 * D * row;
#pragma unroll
    for (int gr = 0; gr < Cols<D>::NG; ++gr)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int col = 16 * NB * gr + 4 * NB * (c & 3) + 4 * i;
            vad[gr][i] = base + 16 * ((col >> 3) ^ swz<D>(row)) + 2 * (col & 7);
        }
}

__device__ __forceinline__ float gate_of(const WinArgs& a, int b, int qi, int h) {
    if (a.gate == nullptr) return 1.0f;
    const float x = load1(a.gate, a.gdt, ((int64_t)b * a.nq + qi) * a.H + h);
    return a.glogit ? sigmoidf(x) : x;
}

// One row by the whole wave from the keys that it sees alone, element d = lane, lane + 64: for rows whose tile held
// something not finite.  The gate is the caller's.
template <int DT, int D>
__device__ __forceinline__ void row_alone(const WinArgs& a, int b, int kv, int r, float (&y)[2]) {
    const int lane = threadIdx.x % 64;
    const int qi = (int)fdiv((uint32_t)r, a.gdiv), h = kv * (int)a.gdiv.d + r - qi * (int)a.gdiv.d;
    const Span sp = make_span(a, b, qi, qi);
    const uint16_t* q = a.q + b * a.q_bs + h * a.q_hs + qi * a.q_ns;
    const uint16_t* k = a.k + b * a.kv_bs + kv * a.kv_hs;
    const uint16_t* v = a.v + b * a.kv_bs + kv * a.kv_hs;
    constexpr int E = D > 64 ? 2 : 1;
    float qv[E], acc[E], m = -FLT_MAX, l = 0.0f;
    const bool in = lane < D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = in ? elem<DT>(q, lane + 64 * e) : 0.0f;
        acc[e] = 0.0f;
    }
    auto score = [&](int64_t at) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += in ? qv[e] * elem<DT>(k, at + lane + 64 * e) : 0.0f;
#pragma unroll
        for (int w = 1; w < 64; w *= 2) s += __shfl_xor(s, w);
        return s * a.sl2;
    };
    for (int t = 0; t < sp.count; ++t) {
        const float s = score(sp.key(t) * a.kv_ns), mn = fmaxf(m, s);
        l = l * __builtin_amdgcn_exp2f(m - mn) + __builtin_amdgcn_exp2f(s - mn);
        m = mn;
    }
    // weights that add up to 1, so that no sum outgrows the values
    for (int t = 0; t < sp.count; ++t) {
        const int64_t at = sp.key(t) * a.kv_ns;
        const float p = __builtin_amdgcn_exp2f(score(at) - m) / l;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += in ? p * elem<DT>(v, at + lane + 64 * e) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) y[e] = e < E ? acc[e < E ? e : 0] : 0.0f;
}

template <int DT, int D>
__device__ __forceinline__ void store_row_alone(const WinArgs& a, int b, int kv, int r) {
    float y[2];
    row_alone<DT, D>(a, b, kv, r, y);
    const int lane = threadIdx.x % 64;
    const int qi = (int)fdiv((uint32_t)r, a.gdiv), h = kv * (int)a.gdiv.d + r - qi * (int)a.gdiv.d;
    const float gv = gate_of(a, b, qi, h);
    const int64_t e = b * a.o_bs + h * a.o_hs + qi * a.o_ns;
    if (lane < D) store1(a.out, a.odt, e + lane, y[0] * gv);
    if (D > 64) store1(a.out, a.odt, e + lane + 64, y[1] * gv);
}

// NV neighbouring columns at element e (a multiple of 8 elements, out 16-byte aligned).
template <int NV>
__device__ __forceinline__ void store_cols(void* out, int dt, int64_t e, const float (&f)[NV]) {
#pragma unroll
    for (int i = 0; i < NV / 8; ++i) {
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = f[8 * i + j];
        store8(out, dt, e + 8 * i, t);
    }
}

// ---- tiles of query rows -----------------------------------------------------------------------

// Four waves of 16 QS rows; tiles of 64 keys come straight into LDS, two of them in turn.
template <int DT, int D, int QS, int NP>
__global__ __launch_bounds__(256) void window_tile_kernel(WinArgs a) {
    constexpr int kRow = 2 * D, CH = D / 8;            // bytes and pieces of a key row
    constexpr int RPL = 1024 / kRow, LD = kTile / RPL / 4;  // rows per load instruction; loads per wave, tile and tensor
    constexpr int NB = Cols<D>::NB, NG = Cols<D>::NG;
    __shared__ __attribute__((aligned(16))) char k0[kTile * kRow];
    __shared__ __attribute__((aligned(16))) char v0[kTile * kRow];
    __shared__ __attribute__((aligned(16))) char k1[kTile * kRow];
    __shared__ __attribute__((aligned(16))) char v1[kTile * kRow];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    // the row tiles of one key head are neighbours on one XCD, which reads its keys into its L2 once
    const uint32_t tile = xcd_tile(blockIdx.x, gridDim.x);
    const uint32_t bkv = tile / a.qtiles;
    uint32_t b, kv;
    fdivmod(bkv, a.kvdiv, b, kv);
    const int t_r0 = (int)(tile % a.qtiles) * 64 * QS, r0 = t_r0 + w * 16 * QS;
    const int G = (int)a.gdiv.d;
    const Span sp = make_span(a, b, (int)fdiv((uint32_t)t_r0, a.gdiv),
                              (int)fdiv((uint32_t)min(t_r0 + 64 * QS, a.rows) - 1, a.gdiv));
    const Rows<QS> rw = make_rows<QS>(a, sp, r0, c);

    u32x4 qf[QS][D / 32];
#pragma unroll
    for (int x = 0; x < QS; ++x) {
        const int r = min(r0 + 16 * x + c, a.rows - 1), qi = (int)fdiv((uint32_t)r, a.gdiv);
        const uint16_t* q = a.q + b * a.q_bs + (kv * G + r - qi * G) * a.q_hs + qi * a.q_ns;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) qf[x][s] = *reinterpret_cast<const u32x4*>(q + 32 * s + 8 * g);
    }
    State<D, QS> st;
    st.reset();

    const uint16_t* kb_ = a.k + b * a.kv_bs + kv * a.kv_hs;
    const uint16_t* vb_ = a.v + b * a.kv_bs + kv * a.kv_hs;
    auto load_tile = [&](int t0, char* kd, char* vd) {
#pragma unroll
        for (int u = 0; u < LD; ++u) {
            const int r = (w * LD + u) * RPL + lane / CH;
            const int64_t at = (int64_t)sp.key(min(t0 + r, sp.count - 1)) * a.kv_ns + 8 * ((lane % CH) ^ swz<D>(r));
            load_to_lds(kb_ + at, kd + 1024 * (w * LD + u));
            load_to_lds(vb_ + at, vd + 1024 * (w * LD + u));
        }
    };
    auto step = [&](int t0, const char* ks, const char* vs, char* kn, char* vn) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile has landed
        __syncthreads();                     // every wave's has, and none still reads the other buffers
        if (t0 + kTile < sp.count) load_tile(t0 + kTile, kn, vn);
        if (r0 >= a.rows) return;
        uint32_t vad[NG][NB];
        v_addresses<D>(vs, g, c, vad);
#pragma unroll
        for (int hh = 0; hh < kTile / kChunk; ++hh) {
            const int t = t0 + hh * kChunk;
            if (all_hidden<QS>(a, sp, rw, t)) continue;
            u32x4 kf[2][D / 32];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int s = 0; s < D / 32; ++s)
                    kf[kb][s] = *reinterpret_cast<const u32x4*>(ks + (hh * kChunk + 16 * kb + c) * kRow + 16 * ((4 * s + g) ^ swz<D>(c)));
            attend<DT, D, QS, NP>(a, sp, rw, t, kf, qf, vad, hh * kChunk * kRow, g, st);
        }
    };
    if (sp.count > 0) load_tile(0, k0, v0);
    for (int t0 = 0; t0 < sp.count; t0 += 2 * kTile) {
        step(t0, k0, v0, k1, v1);
        if (t0 + kTile < sp.count) step(t0 + kTile, k1, v1, k0, v0);
    }

#pragma unroll
    for (int x = 0; x < QS; ++x) {
        float l = st.l[x];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int r = r0 + 16 * x + c, qi = (int)fdiv((uint32_t)min(r, a.rows - 1), a.gdiv);
        const int h = kv * G + min(r, a.rows - 1) - qi * G;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
        bool bad = not_finite(l);
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) bad = bad || not_finite(st.o[x][db][i]);
        uint64_t rows_bad = __builtin_amdgcn_ballot_w64(bad && r < a.rows);
        rows_bad |= rows_bad >> 32;
        rows_bad = (rows_bad | (rows_bad >> 16)) & 0xffff;
        const float gv = gate_of(a, b, qi, h);
        if (r < a.rows && ((rows_bad >> c) & 1) == 0) {
            const int64_t e = b * a.o_bs + h * a.o_hs + qi * a.o_ns;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float f[4 * NB];
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[4 * i + j] = st.o[x][gr * NB + i][j] * inv * gv;
                store_cols<4 * NB>(a.out, a.odt, e + 16 * NB * gr + 4 * NB * g, f);
            }
        }
        while (rows_bad != 0) {
            const int rc = __builtin_ctzll(rows_bad);
            rows_bad &= rows_bad - 1;
            store_row_alone<DT, D>(a, b, kv, r0 + 16 * x + rc);
        }
    }
}

// ---- few query rows against many keys -------------------------------------------------------------

// A block holds 16 rows and a share of their key list; its waves take 32 keys at a time in turn, each with its own
// V tile in LDS, and are joined through LDS.  With more than one share the block leaves its rows' (m, l, O) in the
// workspace for window_join_kernel: part[(b, kv, tile, row of 16)][split][D + 2].
template <int DT, int D, int NP>
__global__ __launch_bounds__(512) void window_split_kernel(WinArgs a) {
    constexpr int kRow = 2 * D, CH = D / 8;
    constexpr int RPL = 1024 / kRow, LD = kChunk / RPL;
    constexpr int NB = Cols<D>::NB, NG = Cols<D>::NG;
    constexpr int kPart = D + 2;
    // V tiles while the keys are read, then the waves' rows: [wave][16][D + 2] f32
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64), nw = blockDim.x / 64;
    const uint32_t split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
    const uint32_t bkv = tile / a.qtiles;
    uint32_t b, kv;
    fdivmod(bkv, a.kvdiv, b, kv);
    const int r0 = (int)(tile % a.qtiles) * 16, G = (int)a.gdiv.d;
    const Span sp = make_span(a, b, (int)fdiv((uint32_t)r0, a.gdiv), (int)fdiv((uint32_t)min(r0 + 16, a.rows) - 1, a.gdiv));
    const Rows<1> rw = make_rows<1>(a, sp, r0, c);
    // this block's share of the list, in whole steps
    const int steps = (sp.count + kChunk - 1) / kChunk;
    const int sa = (int)((int64_t)steps * split / a.splits), sb = (int)((int64_t)steps * (split + 1) / a.splits);

    u32x4 qf[1][D / 32];
    {
        const int r = min(r0 + c, a.rows - 1), qi = (int)fdiv((uint32_t)r, a.gdiv);
        const uint16_t* q = a.q + b * a.q_bs + (kv * G + r - qi * G) * a.q_hs + qi * a.q_ns;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) qf[0][s] = *reinterpret_cast<const u32x4*>(q + 32 * s + 8 * g);
    }
    State<D, 1> st;
    st.reset();
    const uint16_t* kb_ = a.k + b * a.kv_bs + kv * a.kv_hs;
    const uint16_t* vb_ = a.v + b * a.kv_bs + kv * a.kv_hs;
    char* vt = lds + w * kChunk * kRow;
    uint32_t vad[NG][NB];
    v_addresses<D>(vt, g, c, vad);
    for (int i = sa + w; i < sb; i += nw) {
        const int t0 = i * kChunk;
#pragma unroll
        for (int u = 0; u < LD; ++u) {
            const int r = u * RPL + lane / CH;
            const int64_t at = (int64_t)sp.key(min(t0 + r, sp.count - 1)) * a.kv_ns + 8 * ((lane % CH) ^ swz<D>(r));
            load_to_lds(vb_ + at, vt + 1024 * u);
        }
        u32x4 kf[2][D / 32];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const uint16_t* k = kb_ + (int64_t)sp.key(min(t0 + 16 * kb + c, sp.count - 1)) * a.kv_ns + 8 * g;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) kf[kb][s] = *reinterpret_cast<const u32x4*>(k + 32 * s);
        }
        wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        attend<DT, D, 1, NP>(a, sp, rw, t0, kf, qf, vad, 0, g, st);
    }

    // the waves' rows, joined: m, l and O of each, the four lanes of a row holding its columns
    float l = st.l[0];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the V tiles are done with
    float* mine = reinterpret_cast<float*>(lds) + (w * 16 + c) * kPart;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[16 * NB * gr + 4 * NB * g + 4 * i + j] = st.o[0][gr * NB + i][j];
    if (g == 0) {
        mine[D] = st.m[0];
        mine[D + 1] = l;
    }
    __syncthreads();
    for (int rr = w; rr < 16 && r0 + rr < a.rows; rr += nw) {
        const float* p = reinterpret_cast<const float*>(lds) + rr * kPart;
        float m = -FLT_MAX;
        for (int i = 0; i < nw; ++i) m = fmaxf(m, p[i * 16 * kPart + D]);
        float ls = 0.0f, o[2] = {0.0f, 0.0f};
        for (int i = 0; i < nw; ++i) {
            const float* q = p + i * 16 * kPart;
            const float f = __builtin_amdgcn_exp2f(q[D] - m);
            ls += q[D + 1] * f;
            if (lane < D) o[0] += q[lane] * f;
            if (D > 64) o[1] += q[lane + 64] * f;
        }
        const int r = r0 + rr;
        if (a.splits > 1) {
            float* dst = a.ws + (((int64_t)bkv * a.rows + r) * a.splits + split) * kPart;
            if (lane < D) dst[lane] = o[0];
            if (D > 64) dst[lane + 64] = o[1];
            if (lane == 0) {
                dst[D] = m;
                dst[D + 1] = ls;
            }
            continue;
        }
        if (__builtin_amdgcn_ballot_w64(not_finite(ls) || not_finite(o[0]) || not_finite(o[1])) != 0) {
            store_row_alone<DT, D>(a, b, kv, r);
            continue;
        }
        const int qi = (int)fdiv((uint32_t)r, a.gdiv), h = kv * G + r - qi * G;
        const float f = (ls == 0.0f ? 0.0f : 1.0f / ls) * gate_of(a, b, qi, h);
        const int64_t e = b * a.o_bs + h * a.o_hs + qi * a.o_ns;
        if (lane < D) store1(a.out, a.odt, e + lane, o[0] * f);
        if (D > 64) store1(a.out, a.odt, e + lane + 64, o[1] * f);
    }
}

// One block per query row: its waves take the shares in turn.
template <int DT, int D>
__global__ __launch_bounds__(512) void window_join_kernel(WinArgs a) {
    constexpr int kPart = D + 2;
    __shared__ float part[8][kPart];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64, nw = blockDim.x / 64;
    const uint32_t bkv = blockIdx.x / a.rows;
    const int r = (int)(blockIdx.x % a.rows);
    uint32_t b, kv;
    fdivmod(bkv, a.kvdiv, b, kv);
    const float* p = a.ws + (int64_t)blockIdx.x * a.splits * kPart;
    float m = -FLT_MAX;
    for (uint32_t i = lane; i < a.splits; i += 64) m = fmaxf(m, p[i * kPart + D]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x));
    float l = 0.0f, o[2] = {0.0f, 0.0f};
    for (uint32_t i = w; i < a.splits; i += nw) {
        const float* q = p + i * kPart;
        const float f = __builtin_amdgcn_exp2f(q[D] - m);
        l += q[D + 1] * f;
        if (lane < D) o[0] += q[lane] * f;
        if (D > 64) o[1] += q[lane + 64] * f;
    }
    if (lane < D) part[w][lane] = o[0];
    if (D > 64) part[w][lane + 64] = o[1];
    if (lane == 0) part[w][D] = l;
    __syncthreads();
    if (w > 0) return;
    for (int i = 1; i < nw; ++i) {
        l += part[i][D];
        if (lane < D) o[0] += part[i][lane];
        if (D > 64) o[1] += part[i][lane + 64];
    }
    if (__builtin_amdgcn_ballot_w64(not_finite(l) || not_finite(o[0]) || not_finite(o[1])) != 0) {
        store_row_alone<DT, D>(a, b, kv, r);
        return;
    }
    const int qi = (int)fdiv((uint32_t)r, a.gdiv), h = kv * (int)a.gdiv.d + r - qi * (int)a.gdiv.d;
    const float f = (l == 0.0f ? 0.0f : 1.0f / l) * gate_of(a, b, qi, h);
    const int64_t e = b * a.o_bs + h * a.o_hs + qi * a.o_ns;
    if (lane < D) store1(a.out, a.odt, e + lane, o[0] * f);
    if (D > 64) store1(a.out, a.odt, e + lane + 64, o[1] * f);
}

// ---- choice of the form ------------------------------------------------------------------------------

struct Plan {
    bool few;        // window_split_kernel
    int waves;       // its waves per block
    int64_t splits;  // its shares of the key list
};

Plan make_plan(int64_t B, int64_t H, int64_t KV, int64_t nq, int64_t nk, int64_t left, int64_t right, int64_t sinks) {
    Plan p{};
    const int64_t cus = cu_count(), rows = nq * (H / KV);
    // the most keys that a tile of rows may see
    int64_t span = nk;
    if (left >= 0 && right >= 0) span = std::min(nk, sinks + left + right + std::min<int64_t>(nq, 64));
    p.few = rows <= 16 || (rows <= 256 && B * KV * ceil_div(rows, 64) < cus && span > 1024);
    if (!p.few) return p;
    const int64_t tiles = B * KV * ceil_div(rows, 16), steps = ceil_div(span, kChunk);
    p.waves = 4;
    p.splits = std::max<int64_t>(1, std::min(ceil_div(4 * cus, tiles), steps / 8));
    return p;
}

bool sizes_ok(int64_t B, int64_t H, int64_t KV, int64_t nq, int64_t nk, int64_t D, int64_t sinks) {
    constexpr int64_t lim = int64_t(1) << 28;
    return B >= 0 && H >= 1 && KV >= 1 && H % KV == 0 && nq >= 0 && nk >= 0 && sinks >= 0 &&
           (D == 32 || D == 64 || D == 128) && nq < lim && nk < lim && H < (1 << 16) && B < lim && nq * (H / KV) < lim &&
           B * KV < lim;
}

}  // namespace
}  // namespace mbrt

using namespace mbrt;

extern "C" {

int64_t mbrt_attention_window_workspace_bytes(int64_t B, int64_t H, int64_t H_kv, int64_t n_q, int64_t n_k,
                                              int64_t head_dim, int64_t left, int64_t right, int64_t sinks) {
    if (!sizes_ok(B, H, H_kv, n_q, n_k, head_dim, sinks)) return -1;
    if (B == 0 || n_q == 0) return 0;
    const Plan p = make_plan(B, H, H_kv, n_q, n_k, left, right, std::min(sinks, n_k));
    return p.few && p.splits > 1 ? B * H * n_q * p.splits * (head_dim + 2) * 4 : 0;
}

int mbrt_attention_window(const void* q, const void* k, const void* v, int dtype, int64_t B, int64_t H, int64_t H_kv,
                          int64_t n_q, int64_t n_k, int64_t head_dim, int64_t q_batch_stride, int64_t q_head_stride,
                          int64_t q_row_stride, int64_t kv_batch_stride, int64_t kv_head_stride, int64_t kv_row_stride,
                          int64_t left, int64_t right, int64_t sinks, int64_t q_start, const int32_t* key_lens,
                          const void* gate, int gate_dtype, int gate_is_logit, void* out, int out_dtype,
                          int64_t out_batch_stride, int64_t out_head_stride, int64_t out_row_stride, float scale,
                          void* workspace, int64_t workspace_bytes, mbrt_stream_t stream) {
    const char* op = "mbrt_attention_window";
    MBRT_REQUIRE(dtype == BF16 || dtype == F16, MBRT_E_UNSUPPORTED_DTYPE, "%s: q/k/v must be BF16 or F16", op);
    MBRT_REQUIRE_FLOAT_DT(out_dtype, op);
    MBRT_REQUIRE(!gate || is_float_dt(gate_dtype), MBRT_E_UNSUPPORTED_DTYPE, "%s: gate dtype %d", op, gate_dtype);
    MBRT_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, MBRT_E_SHAPE,
                 "%s: head_dim %lld (32, 64 and 128 are built)", op, (long long)head_dim);
    MBRT_REQUIRE(H >= 1 && H_kv >= 1 && H % H_kv == 0, MBRT_E_SHAPE, "%s: %lld heads over %lld key heads", op,
                 (long long)H, (long long)H_kv);
    MBRT_REQUIRE(sizes_ok(B, H, H_kv, n_q, n_k, head_dim, sinks), MBRT_E_SHAPE,
                 "%s: negative size, or a dimension beyond 2^28 (2^16 heads)", op);
    MBRT_REQUIRE(left >= -1 && right >= -1 && q_start >= -1 && q_start < (int64_t(1) << 28), MBRT_E_INVALID_ARG,
                 "%s: left, right and q_start are -1 or more, q_start below 2^28", op);
    MBRT_REQUIRE(scale >= 0.0f && std::isfinite(scale), MBRT_E_INVALID_ARG, "%s: scale must be finite and >= 0", op);
    if (B == 0 || n_q == 0) return MBRT_OK;
    MBRT_REQUIRE(q && out && (n_k == 0 || (k && v)), MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(key_lens, 4) &&
                     (!gate || aligned(gate, dt_size(gate_dtype))),
                 MBRT_E_ALIGN, "%s: q, k, v and out must be 16-byte aligned", op);
    const int64_t st[9] = {q_batch_stride, q_head_stride, q_row_stride, kv_batch_stride, kv_head_stride,
                           kv_row_stride, out_batch_stride, out_head_stride, out_row_stride};
    for (int i = 0; i < 9; ++i)
        MBRT_REQUIRE(st[i] >= 0 && st[i] % 8 == 0, MBRT_E_ALIGN, "%s: strides must be non-negative multiples of 8", op);
    const Plan plan = make_plan(B, H, H_kv, n_q, n_k, left, right, std::min(sinks, n_k));
    const int64_t need = mbrt_attention_window_workspace_bytes(B, H, H_kv, n_q, n_k, head_dim, left, right, sinks);
    MBRT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 4)), MBRT_E_INVALID_ARG,
                 "%s: workspace of %lld bytes, %lld needed", op, (long long)(workspace ? workspace_bytes : 0),
                 (long long)need);
    const int64_t G = H / H_kv, far = int64_t(1) << 28;
    WinArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.out = out;
    a.lens = key_lens;
    a.gate = gate;
    a.ws = static_cast<float*>(workspace);
    a.q_bs = q_batch_stride;
    a.q_hs = q_head_stride;
    a.q_ns = q_row_stride;
    a.kv_bs = kv_batch_stride;
    a.kv_hs = kv_head_stride;
    a.kv_ns = kv_row_stride;
    a.o_bs = out_batch_stride;
    a.o_hs = out_head_stride;
    a.o_ns = out_row_stride;
    a.nq = (int)n_q;
    a.nk = (int)n_k;
    a.rows = (int)(n_q * G);
    a.H = (int)H;
    a.KV = (int)H_kv;
    a.left = (int)std::min(left, 2 * far);  // beyond every position: the same keys
    a.right = (int)std::min(right, 2 * far);
    a.sinks = (int)std::min(sinks, n_k);
    a.start = (int)q_start;
    a.gdt = gate_dtype;
    a.glogit = gate_is_logit ? 1 : 0;
    a.odt = out_dtype;
    a.sl2 = (scale == 0.0f ? 1.0f / std::sqrt((float)head_dim) : scale) * 1.44269504088896340736f;
    a.gdiv = make_fastdiv((uint32_t)G);
    a.kvdiv = make_fastdiv((uint32_t)H_kv);
    a.splits = (uint32_t)plan.splits;
    hipStream_t stm = as_stream(stream);
    const int64_t bkv = B * H_kv;
    a.qtiles = (uint32_t)ceil_div(a.rows, plan.few ? 16 : 64);
    const int64_t blocks = bkv * a.qtiles * (plan.few ? plan.splits : 1);
    MBRT_REQUIRE(blocks < kMaxGridX && bkv * a.rows < kMaxGridX, MBRT_E_SHAPE, "%s: too many tiles", op);
    auto launch = [&](auto dt, auto dim, auto parts) {
        constexpr int DTv = decltype(dt)::value, Dv = decltype(dim)::value, NP = decltype(parts)::value;
        if (!plan.few) {
            hipLaunchKernelGGL((window_tile_kernel<DTv, Dv, 1, NP>), dim3((unsigned)blocks), dim3(256), 0, stm, a);
            return;
        }
        const size_t lds = (size_t)plan.waves * 16 * (Dv + 2) * 4;  // the joined rows; the V tiles need less
        static_assert(kChunk * 2 * Dv <= 16 * (Dv + 2) * 4, "V tile within the rows' space");
        hipLaunchKernelGGL((window_split_kernel<DTv, Dv, NP>), dim3((unsigned)blocks), dim3(plan.waves * 64), lds, stm, a);
        if (plan.splits > 1)
            hipLaunchKernelGGL((window_join_kernel<DTv, Dv>), dim3((unsigned)(bkv * a.rows)), dim3(512), 0, stm, a);
    };
    auto by_dim = [&](auto dt, auto parts) {
        if (head_dim == 32) launch(dt, std::integral_constant<int, 32>(), parts);
        else if (head_dim == 64) launch(dt, std::integral_constant<int, 64>(), parts);
        else launch(dt, std::integral_constant<int, 128>(), parts);
    };
    const std::integral_constant<int, 2> two;
    if (dtype == F16) by_dim(std::integral_constant<int, F16>(), two);
    else if (out_dtype != F32) by_dim(std::integral_constant<int, BF16>(), two);
    else by_dim(std::integral_constant<int, BF16>(), std::integral_constant<int, 3>());
    return check_launch(op);
}

}  // extern "C"
