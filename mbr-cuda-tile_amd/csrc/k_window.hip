// Attention through a sliding window with sinks, on MFMA, for bf16 or f16 heads of 32, 64 or 128: the fused
// attention's companion for long songs and for streaming (mbrt_attention_window's comment in mbrt.h holds the
// definition).  Key j is visible to the query at position p iff
//   j < len_b,  j <= p + right,  and  j >= p - left or j < sinks.
//
// Query rows: the H / H_kv query heads that share a key head are rows of one matrix, row r = (query r / G, head
// r % G), so that each key and value is read once for all of them.
// Keys: what the rows of a tile may see is one list, the sinks before the window and then the window's keys lo .. hi
// of all its rows: t -> j = t < s ? t : lo + t - s, with s <= lo.  No key outside is read, whatever stands there (NaN
// behind a sequence's end).
//
// Per 32 keys, with v_mfma_f32_16x16x32 (lane l = (g, c): A[c][8 g + j], B[8 g + j][c], C[4 g + i][c]):
//   S^T = K Q^T      A = K rows, B = the wave's 16 query rows: lane (g, c) holds S^T[key 16 kb + 4 g + i][row c].
//   online softmax   per row c, as in the fused attention: the exponent's reference m moves only when a score
//                    outgrows it by 2^kTop, each lane sums its own keys' p, the four lanes of a row are added at the end.
//   O^T += V^T P^T   B = P^T from the S^T registers: slot j of lane group g is key 4 g + j, or 16 + 4 g + j - 4 from
//                    j = 4 on; A = V^T by LDS transpose reads.  P enters as a sum of two or three values of the
//                    2-byte type (split_p), so that little beside the inputs' and the output's own rounding is left.
// Lane (g, c) ends with columns 16 db + 4 g .. + 3 of row c.
//
// What bounds it (MI355X, us; counters by rocprofv3): bf16 [60, 801], 8 heads of 64 through 101 keys and 8 sinks, 57.5 to 60; its
// loads and stores alone take 43 (197 MB at 4.6 TB/s), the rest is the softmax's VALU work, which hides behind them only in
// part (a wave's tile of 64 keys: 24 MFMAs of 16 clocks, about 170 VALU instructions of 4 and 16 exponentials of 16, and 16 KB of
// LDS reads), a third of it for nothing: a wave's 16 rows see 124 keys, the list of its tile holds 172, and it works on 192.
// f16 [2, 16389], 8 heads over 2 of 128 through 1024 keys, 210 to 215: 134 GFLOP, half as many again for the second
// part of p (145 at a large library product's rate), on matrix units that are busy half the time, the
// VALU for about as long (9 operations and an exponential for each score), which two waves per SIMD overlap only in
// part.  One token: 60 caches of 1601 frames 20.4, 100 MB at 4.9 TB/s, as a
// copy; [1, 200003] 22.7.
// Not kept: steps of 64 keys, priorities around the MFMAs, row sums by the matrix unit (no gain), V fragments read two
// blocks ahead (1 %); skipping steps that
// are hidden from a wave, which cost as much in register copies as it saved.  Kept: transpose reads by the
// compiler's builtin, which it can place early, 71 -> 64 at 32 rows per wave; addresses of a tile from one scalar base and a
// layout without bank conflicts 290 -> 267 at f16 [2, 16389] with 16 rows per wave, 32 rows per wave 216.
//
// A value that a row does not see but another row of its tile does enters the product with weight 0.  Where that
// value is infinite or NaN the product is NaN; a row that ends with anything not finite is computed again from the
// keys that it sees alone (row_alone), so that the definition holds for it too.  That takes its time, key by key, unless the row
// turns out NaN: f16 [2, 16389] as above with one infinity in a value of one head 25 ms, in a sink's 102.
#include "abi_common.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace mbrt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The weights are p = 2^(score - m) with a reference m that moves only when a score outgrows 2^kTop, and then to where the
// score is 2^kBase: a row's largest weight lies between the two.  f16 has its smallest step at 2^-24, so its weights use the
// top of its range.  A smaller distance loses less of small weights and moves m more often: f16 [2, 16389], 8 heads over 2 of
// 128 through 1024 keys, with 2^13 220 us, 2^11 214, 2^10 210, 2^7 209 and 2^0 (to 2^8) 209.
template <int DT> constexpr float kBase = DT == F16 ? 10.0f : 0.0f;
template <int DT> constexpr float kTop = DT == F16 ? 15.0f : 8.0f;
constexpr int kBufferDword3 = 0x00020000;  // raw buffer resource: 32-bit data format, no swizzle, no stride
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
    p.s = a.left < 0 ? 0 : max(0, min(a.sinks, p.hi + 1));
    p.lo = max(p.lo, p.s);
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

// Two values of P as NP 2-byte values each, rounded to nearest each time (exact differences).  Two parts of bf16 hold p to
// 2^-17 of itself, three to 2^-24.  Two of f16 hold it to 2^-23, about what exp2 leaves of it, or to half of f16's smallest step
// where that is more: 2^-25, which is 2^-35 of the row's largest weight or less.
// bf16 heads take three parts for f32 outputs, and where few queries share out their keys (window_split_kernel), which wait for
// memory: one frame against 60 caches 22.0 us with two and with three, four against 20 caches of 1000 8.1 and 8.4.  The tiles of
// query rows take two for 2-byte outputs: a third costs [60, 801] through 109 keys 57.5 -> 62, through all 155 -> 184, and
// 2^-17 is below a hundredth of the output's own half step of 2^-8.
template <int DT, int NP>
__device__ __forceinline__ void split_p(float p0, float p1, uint32_t (&w)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        if constexpr (DT == BF16) {
            if (i == NP - 1) {
                w[i] = pack_bf16x2(p0, p1);
            } else {
                w[i] = pack_bf16x2(p0, p1);
                p0 -= bf16_lo(w[i]);
                p1 -= bf16_hi(w[i]);
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

// Whether query row r sees a key at all.  Where the weights of one that does add up to 0, every key that it sees scores
// -infinity, and its softmax is NaN; zeros are for rows that see none.
__device__ __forceinline__ bool sees_any(const WinArgs& a, int b, int r) {
    const int qi = (int)fdiv((uint32_t)r, a.gdiv);
    return make_span(a, b, qi, qi).count > 0;
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// K and V tiles in LDS: rows of D 2-byte elements in 16-byte pieces, piece j of row r at j ^ swz(r).  The banks are 256
// bytes wide; an access of 16 bytes per lane goes by lanes 0-3, 12-15, 20-23, 24-27 (and the complement) at a time, one of 8
// bytes by 32 lanes.  These keys keep both the K fragments (16 rows' pieces j, j ^ 1) and V's transpose reads (8 rows' pieces 2 i,
// 2 i + 1) on different banks: no conflicts counted.
template <int D>
__device__ __forceinline__ int swz(int r) {
    return D == 128 ? ((r & 7) << 1) : D == 64 ? (r & 7) : (-(r >> 2) & 3);
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
// A V^T fragment of 32 keys by two transpose reads: rows r and r + 16 (32 D bytes further).
template <int D>
__device__ __forceinline__ u32x4 lds_read_vt(const char* p) {
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 32 * D)));
    return u32x4{a.x, a.y, b.x, b.y};
}

// 16 bytes per lane from the lane's own p straight to lds + 16 lane.  Not a template: the builtin's operands must not
// depend on one, or the host pass drops the kernel that holds it.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t base, char* lds, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_void*)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void load_to_lds(const uint16_t* p, char* lds) {
    __builtin_amdgcn_global_load_lds((global_void*)p, (lds_void*)lds, 16, 0, 0);
}

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

// The rows a wave works on, in the list's places t: the window of the lane's row c of each sub-block x is first ..
// first + n - 1, behind the sinks; it sees sink t (< s) iff t <= jhi.  From all0 to all1 every row of the wave sees every
// key; sinks from sink1 on are seen by none.
template <int QS>
struct Rows {
    int first[QS], n[QS], jhi[QS];
    int all0, all1, sink1;
};

template <int QS>
__device__ __forceinline__ Rows<QS> make_rows(const WinArgs& a, const Span& sp, int r0, int c) {
    Rows<QS> rw;
    const int off = sp.s - sp.lo;  // t of key j behind the sinks: j + off
#pragma unroll
    for (int x = 0; x < QS; ++x) {
        const int p = sp.start + (int)fdiv((uint32_t)min(r0 + 16 * x + c, a.rows - 1), a.gdiv);
        const int jlo = a.left < 0 ? sp.lo : max(sp.lo, p - a.left);
        rw.jhi[x] = a.right < 0 ? sp.hi : min(sp.hi, p + a.right);
        rw.first[x] = jlo + off;
        rw.n[x] = max(0, rw.jhi[x] - jlo + 1);
    }
    const int pa = sp.start + (int)fdiv((uint32_t)min(r0, a.rows - 1), a.gdiv);
    const int pb = sp.start + (int)fdiv((uint32_t)min(r0 + 16 * QS - 1, a.rows - 1), a.gdiv);
    const int hia = a.right < 0 ? sp.hi : min(sp.hi, pa + a.right), hib = a.right < 0 ? sp.hi : min(sp.hi, pb + a.right);
    rw.all0 = (a.left < 0 ? sp.lo : max(sp.lo, pb - a.left)) + off;
    rw.all1 = hia + 1 + off;
    rw.sink1 = min(sp.s, hib + 1);
    return rw;
}

// One step over the 32 NC keys from t0 on.  kf(kb, s): K[16 kb + c][32 s + 8 g ..]; vad: the lane's transpose addresses
// from the step's first V row.
template <int DT, int D, int QS, int NP, int NC, class KF>
__device__ __forceinline__ void attend(const WinArgs& a, const Span& sp, const Rows<QS>& rw, int t0, KF kf,
                                       const u32x4 (&qf)[QS][D / 32], const char* vtile, const uint32_t (&vad)[D / 16],
                                       int g, State<D, QS>& st) {
    constexpr int KB = 2 * NC;
    f32x4 s[QS][KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int x = 0; x < QS; ++x) s[x][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const u32x4 k = kf(kb, e);
#pragma unroll
            for (int x = 0; x < QS; ++x) s[x][kb] = mma<DT>(k, qf[x][e], s[x][kb]);
        }
    }
    // Keys hidden from some row: before its window, behind it, or (both at once) in a step that holds sinks, which a row
    // sees up to jhi.  k = 16 kb + i is the key's place from t0 + 4 g on.
    if (t0 < rw.sink1) {
#pragma unroll
        for (int x = 0; x < QS; ++x) {
            const int lo = rw.first[x] - (t0 + 4 * g), hi = lo + rw.n[x], sink = min(sp.s, rw.jhi[x] + 1) - (t0 + 4 * g);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = 16 * kb + i;
                    s[x][kb][i] = (bool)(((int)(k >= lo) & (int)(k < hi)) | (int)(k < sink)) ? s[x][kb][i] : -INFINITY;
                }
        }
    } else {
        if (t0 < rw.all0) {
#pragma unroll
            for (int x = 0; x < QS; ++x) {
                const int lo = rw.first[x] - (t0 + 4 * g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[x][kb][i] = 16 * kb + i < lo ? -INFINITY : s[x][kb][i];
            }
        }
        if (t0 + kChunk * NC > rw.all1) {
#pragma unroll
            for (int x = 0; x < QS; ++x) {
                const int hi = rw.first[x] + rw.n[x] - (t0 + 4 * g);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[x][kb][i] = 16 * kb + i >= hi ? -INFINITY : s[x][kb][i];
            }
        }
    }
    float mx[QS];
    bool grown = false;
#pragma unroll
    for (int x = 0; x < QS; ++x) {
        mx[x] = s[x][0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[x] = fmaxf(mx[x], s[x][kb][i]);
        grown = grown || mx[x] * a.sl2 > st.m[x] + kTop<DT>;
    }
    if (__builtin_amdgcn_ballot_w64(grown) != 0) {
#pragma unroll
        for (int x = 0; x < QS; ++x) {
            float top = fmaxf(mx[x], __shfl_xor(mx[x], 16));
            top = fmaxf(top, __shfl_xor(top, 32)) * a.sl2;
            const float mn = top > st.m[x] + kTop<DT> ? top - kBase<DT> : st.m[x];
            const float alpha = __builtin_amdgcn_exp2f(st.m[x] - mn);
            st.l[x] *= alpha;
#pragma unroll
            for (int db = 0; db < D / 16; ++db) st.o[x][db] *= alpha;
            st.m[x] = mn;
        }
    }
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
        u32x4 pp[QS][NP];
#pragma unroll
        for (int x = 0; x < QS; ++x)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[x][2 * cc + kb][i], a.sl2, -st.m[x]));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[x][2 * cc + kb][i + 1], a.sl2, -st.m[x]));
                    st.l[x] += p0 + p1;
                    uint32_t parts[NP];
                    split_p<DT, NP>(p0, p1, parts);
#pragma unroll
                    for (int n = 0; n < NP; ++n) pp[x][n][2 * kb + i / 2] = parts[n];
                }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
            const u32x4 va = lds_read_vt<D>(vtile + 2 * D * kChunk * cc + vad[db]);
#pragma unroll
            for (int x = 0; x < QS; ++x)
#pragma unroll
                for (int n = 0; n < NP; ++n) st.o[x][db] = mma<DT>(va, pp[x][n], st.o[x][db]);
        }
    }
}

// The lane's transpose addresses of a V tile, from its first row: lane (g, c) points to row 4 g + c / 4, columns 16 db +
// 4 (c % 4) .. + 3, and receives column 16 db + c of the rows 4 g .. 4 g + 3.
template <int D>
__device__ __forceinline__ void v_addresses(int g, int c, uint32_t (&vad)[D / 16]) {
    const int row = 4 * g + (c >> 2);
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
        vad[db] = 2 * D * row + 16 * ((2 * db + ((c & 3) >> 1)) ^ swz<D>(row)) + 8 * (c & 1);
}

__device__ __forceinline__ float gate_of(const WinArgs& a, int b, int qi, int h) {
    if (a.gate == nullptr) return 1.0f;
    const float x = load1(a.gate, a.gdt, ((int64_t)b * a.nq + qi) * a.H + h);
    return a.glogit ? sigmoidf(x) : x;
}

// One row by the whole wave from the keys that it sees alone, element d = lane, lane + 64: for rows whose tile held
// something not finite, and rows whose weights are all 0 (1 / 0 here, and so NaN).  The gate is the caller's.
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
        if (not_finite(l)) {  // a score that is NaN or +infinite: so is every weight
            y[0] = y[1] = l;
            return;
        }
    }
    // weights that add up to 1, so that no sum outgrows the values
    for (int t = 0; t < sp.count; ++t) {
        const int64_t at = sp.key(t) * a.kv_ns;
        const float p = __builtin_amdgcn_exp2f(score(at) - m) / l;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += in ? p * elem<DT>(v, at + lane + 64 * e) : 0.0f;
        bool open = false;  // a column that more keys can still change
#pragma unroll
        for (int e = 0; e < E; ++e) open = open || (in && !isnan(acc[e]));
        if (__builtin_amdgcn_ballot_w64(open) == 0) break;
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

// A row's D columns from its four lanes: lane g holds columns 16 db + 4 g .. + 3.  f32: 16 bytes each.  2-byte types: the
// lanes of a pair (g, g ^ 1) exchange halves, so that each stores 8 columns of one of two blocks, 16 bytes; `store` is
// uniform within a pair.
template <int D>
__device__ __forceinline__ void store_row(const WinArgs& a, int64_t e, const f32x4 (&o)[D / 16], float f, int g, bool store) {
    if (a.odt == F32) {
        if (!store) return;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.out) + e + 16 * db + 4 * g) = o[db] * f;
        return;
    }
#pragma unroll
    for (int p = 0; p < D / 32; ++p) {
        u32x2 w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 v = o[2 * p + i] * f;
            w[i] = a.odt == BF16 ? u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}
                                 : u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
        }
        const bool odd = g & 1;
        const u32x2 give = odd ? w[0] : w[1];
        const u32x2 got = {(uint32_t)__shfl_xor((int)give.x, 16), (uint32_t)__shfl_xor((int)give.y, 16)};
        const u32x4 v = odd ? u32x4{got.x, got.y, w[1].x, w[1].y} : u32x4{w[0].x, w[0].y, got.x, got.y};
        if (store)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(a.out) + e + 16 * (2 * p + (g & 1)) + 8 * (g >> 1)));
    }
}

// ---- tiles of query rows -----------------------------------------------------------------------

// Four waves of 16 QS rows; tiles of 64 keys come straight into LDS, two of them in turn.
template <int DT, int D, int QS, int NP>
__global__ __launch_bounds__(256) void window_tile_kernel(WinArgs a) {
    constexpr int kRow = 2 * D, CH = D / 8;            // bytes and pieces of a key row
    constexpr int RPL = 1024 / kRow, LD = kTile / RPL / 4;  // rows per load instruction; loads per wave, tile and tensor
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
    // Lane offsets within a tile of neighbouring keys: such a tile's rows are one scalar base and these.
    uint32_t loff[LD];
#pragma unroll
    for (int u = 0; u < LD; ++u) {
        const int r = (w * LD + u) * RPL + lane / CH;
        loff[u] = 2u * ((uint32_t)r * (uint32_t)a.kv_ns + 8u * ((lane % CH) ^ swz<D>(r)));
    }
    auto load_tile = [&](int t0, char* kd, char* vd) {
        if (t0 >= sp.s && t0 + kTile <= sp.count && a.kv_ns < (1 << 24)) {  // 32-bit offsets
            const int64_t first = (int64_t)(sp.lo + t0 - sp.s) * a.kv_ns;
            const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc((void*)(kb_ + first), (short)0, -1, kBufferDword3);
            const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc((void*)(vb_ + first), (short)0, -1, kBufferDword3);
#pragma unroll
            for (int u = 0; u < LD; ++u) {
                load_to_lds(krs, kd + 1024 * (w * LD + u), loff[u]);
                load_to_lds(vrs, vd + 1024 * (w * LD + u), loff[u]);
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < LD; ++u) {
            const int r = (w * LD + u) * RPL + lane / CH;
            const int64_t at = (int64_t)sp.key(min(t0 + r, sp.count - 1)) * a.kv_ns + 8 * ((lane % CH) ^ swz<D>(r));
            load_to_lds(kb_ + at, kd + 1024 * (w * LD + u));
            load_to_lds(vb_ + at, vd + 1024 * (w * LD + u));
        }
    };
    uint32_t vad[D / 16];
    v_addresses<D>(g, c, vad);
    auto step = [&](int t0, const char* ks, const char* vs, char* kn, char* vn) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile has landed
        __syncthreads();                     // every wave's has, and none still reads the other buffers
        if (t0 + kTile < sp.count) load_tile(t0 + kTile, kn, vn);
        auto kf = [&](int kb, int s) {
            return *reinterpret_cast<const u32x4*>(ks + (16 * kb + c) * kRow + 16 * ((4 * s + g) ^ swz<D>(16 * kb + c)));
        };
        attend<DT, D, QS, NP, kTile / kChunk>(a, sp, rw, t0, kf, qf, vs, vad, g, st);
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
        bool bad = not_finite(l) || (l == 0.0f && sees_any(a, b, min(r, a.rows - 1)));
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) bad = bad || not_finite(st.o[x][db][i]);
        uint64_t rows_bad = __builtin_amdgcn_ballot_w64(bad && r < a.rows);
        rows_bad |= rows_bad >> 32;
        rows_bad = (rows_bad | (rows_bad >> 16)) & 0xffff;
        const float gv = gate_of(a, b, qi, h);
        store_row<D>(a, b * a.o_bs + h * a.o_hs + qi * a.o_ns, st.o[x], inv * gv, g, r < a.rows && ((rows_bad >> c) & 1) == 0);
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
constexpr int kSplitWaves = 8;
template <int DT, int D, int NP>
__global__ __launch_bounds__(kSplitWaves * 64) void window_split_kernel(WinArgs a) {
    constexpr int kRow = 2 * D, CH = D / 8;
    constexpr int RPL = 1024 / kRow, LD = kChunk / RPL;
    constexpr int kPart = D + 2;
    // V tiles while the keys are read, then the waves' rows: [wave][16][D + 2] f32
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / 64);
    constexpr int nw = kSplitWaves;
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
    uint32_t vad[D / 16];
    v_addresses<D>(g, c, vad);
    for (int i = sa + w; i < sb; i += nw) {
        const int t0 = i * kChunk;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's reads of the V tile are done
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
        attend<DT, D, 1, NP, 1>(a, sp, rw, t0, [&](int kb, int s) { return kf[kb][s]; }, qf, vt, vad, g, st);
    }

    // the waves' rows, joined: m, l and O of each, the four lanes of a row holding its columns
    float l = st.l[0];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the V tiles are done with
    float* mine = reinterpret_cast<float*>(lds) + (w * 16 + c) * kPart;
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[16 * db + 4 * g + j] = st.o[0][db][j];
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
        if (__builtin_amdgcn_ballot_w64(not_finite(ls) || not_finite(o[0]) || not_finite(o[1])) != 0 ||
            (ls == 0.0f && sees_any(a, b, r))) {
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

// One block per query row; each wave joins its shares (64 at most: splits <= kJoinWaves * 64), with every load on its way at
// once, and the first one joins the waves.
constexpr int kJoinWaves = 8;
template <int DT, int D>
__global__ __launch_bounds__(kJoinWaves * 64) void window_join_kernel(WinArgs a) {
    constexpr int kPart = D + 2;
    __shared__ float part[kJoinWaves][kPart];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const uint32_t bkv = blockIdx.x / a.rows;
    const int r = (int)(blockIdx.x % a.rows);
    uint32_t b, kv;
    fdivmod(bkv, a.kvdiv, b, kv);
    const int per = ((int)a.splits + kJoinWaves - 1) / kJoinWaves, mine = min(per, (int)a.splits - w * per);
    const float* p = a.ws + ((int64_t)blockIdx.x * a.splits + w * per) * kPart;
    float m = -FLT_MAX, l = 0.0f, o[2] = {0.0f, 0.0f};
    if (lane < mine) {
        m = p[lane * kPart + D];
        l = p[lane * kPart + D + 1];
    }
    float top = m;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float f = lane < mine ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    l *= f;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
    for (int i0 = 0; i0 < mine; i0 += 8) {  // a lane's weight is 0 from share `mine` on
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float fi = __shfl(f, i0 + u);
            const float* q = p + min(i0 + u, mine - 1) * kPart;
            if (lane < D) o[0] += q[lane] * fi;
            if (D > 64) o[1] += q[lane + 64] * fi;
        }
    }
    if (lane < D) part[w][lane] = o[0];
    if (D > 64) part[w][lane + 64] = o[1];
    if (lane == 0) {
        part[w][D] = top;
        part[w][D + 1] = l;
    }
    __syncthreads();
    if (w > 0) return;
    m = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < kJoinWaves; ++i) m = fmaxf(m, part[i][D]);
    l = o[0] = o[1] = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWaves; ++i) {
        const float g = __builtin_amdgcn_exp2f(part[i][D] - m);
        l += part[i][D + 1] * g;
        if (lane < D) o[0] += part[i][lane] * g;
        if (D > 64) o[1] += part[i][lane + 64] * g;
    }
    if (__builtin_amdgcn_ballot_w64(not_finite(l) || not_finite(o[0]) || not_finite(o[1])) != 0 ||
        (l == 0.0f && sees_any(a, b, r))) {
        store_row_alone<DT, D>(a, b, kv, r);
        return;
    }
    const int qi = (int)fdiv((uint32_t)r, a.gdiv), h = kv * (int)a.gdiv.d + r - qi * (int)a.gdiv.d;
    const float q = (l == 0.0f ? 0.0f : 1.0f / l) * gate_of(a, b, qi, h);
    const int64_t e = b * a.o_bs + h * a.o_hs + qi * a.o_ns;
    if (lane < D) store1(a.out, a.odt, e + lane, o[0] * q);
    if (D > 64) store1(a.out, a.odt, e + lane + 64, o[1] * q);
}

// ---- choice of the form ------------------------------------------------------------------------------

struct Plan {
    bool few;        // window_split_kernel
    int qs;          // window_tile_kernel: 16-row blocks per wave
    int64_t splits;  // window_split_kernel: shares of the key list
};

// Few rows (of one tile of 16, or of up to 256 while the tiles of 64 would leave CUs idle before long lists) go to the kernel that
// shares out the keys, 8 waves to a share.  Past 256 rows every tile of 64 walks its list alone, however few tiles there are:
// [1, 100003] keys of 2 heads of 64, 64 queries of 8 heads 67 us and 65 1374; of 8 key heads 256 queries 238 and 257 1382.  What bounds a share is what one CU can read (16 waves to it gain nothing: 805 keys
// of 64 columns 7.1 us with 8, 7.5 with 16); what a second one costs is the join's launch.  So a list is shared out from 32
// pieces on, of 32 keys and 64 columns each (8 KB of keys and values), 5 to a share, over at most a workgroup per CU, and shorter ones
// than 64 pieces only where there are 4 shares or more to it.  us, one share and shared out: 16 lists of 25 pieces 7.3 and
// 8.7, of 38 9.3 and 8.7, of 50 11.9 and 9.4, of 63 13.4 and 9.6; 80 lists of 38 9.7 and 11.0; 120 of 50 14.5
// and 14.8, of 58 17.5 and 16.8.
// One token against [1, 200003] keys of 2 heads 24.7 with a workgroup per CU; with two each, the join taking longer, 33.5.
// Of 128 columns, 32 rows per wave use each fragment read from LDS twice, which pays where lists are long and the larger
// tiles still fill the CUs: [2, 16389] f16 over 1024 keys 259 -> 216 us, [16, 801] bf16 over all 109 -> 103; over 300 keys [30, 801]
// 90 -> 92, over 100 72 -> 76.  Of 64 columns they gain nothing: [60, 801] over all keys 162 -> 160, over 101 60 -> 69.
Plan make_plan(int64_t B, int64_t H, int64_t KV, int64_t nq, int64_t nk, int64_t D, int64_t left, int64_t right,
               int64_t sinks) {
    Plan p{};
    const int64_t cus = cu_count(), rows = nq * (H / KV);
    // the most keys that a tile of rows may see
    int64_t span = nk;
    if (left >= 0 && right >= 0) span = std::min(nk, sinks + std::min(left, nk) + std::min(right, nk) + std::min<int64_t>(nq, 64));
    p.few = rows <= 16 || (rows <= 256 && B * KV * ceil_div(rows, 64) < cus && span > 1024);
    p.qs = D == 128 && span >= 512 && B * KV * ceil_div(rows, 128) >= 2 * cus ? 2 : 1;
    const int64_t tiles = B * KV * ceil_div(rows, 16), pieces = ceil_div(span, kChunk) * D / 64;
    const int64_t shares = std::min<int64_t>(std::min(cus / tiles, ceil_div(pieces, 5)), kJoinWaves * 64);
    p.splits = p.few && pieces >= (shares >= 4 ? 32 : 64) && shares > 1 ? shares : 1;
    return p;
}

int64_t workspace_bytes_of(const Plan& p, int64_t B, int64_t H, int64_t nq, int64_t D) {
    return p.splits > 1 ? B * H * nq * p.splits * (D + 2) * 4 : 0;
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
    const Plan p = make_plan(B, H, H_kv, n_q, n_k, head_dim, left, right, std::min(sinks, n_k));
    return workspace_bytes_of(p, B, H, n_q, head_dim);
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
    const float sl2 = (scale == 0.0f ? 1.0f / std::sqrt((float)head_dim) : scale) * 1.44269504088896340736f;  // of powers of 2
    MBRT_REQUIRE(scale >= 0.0f && std::isfinite(sl2), MBRT_E_INVALID_ARG,
                 "%s: scale must be finite, as scale * log2(e) must, and >= 0", op);
    if (B == 0 || n_q == 0) return MBRT_OK;
    MBRT_REQUIRE(q && out && (n_k == 0 || (k && v)), MBRT_E_INVALID_ARG, "%s: NULL pointer", op);
    MBRT_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(key_lens, 4) &&
                     (!gate || aligned(gate, dt_size(gate_dtype))),
                 MBRT_E_ALIGN, "%s: q, k, v and out must be 16-byte aligned", op);
    int64_t st[9] = {q_batch_stride, q_head_stride, q_row_stride, kv_batch_stride, kv_head_stride,
                     kv_row_stride, out_batch_stride, out_head_stride, out_row_stride};
    const int64_t dim[9] = {B, H, n_q, B, H_kv, n_k, B, H, n_q};
    for (int i = 0; i < 9; ++i) {
        if (st[i] > 0 && dim[i] <= 1) st[i] = 0;  // of a single index: not used
        MBRT_REQUIRE(st[i] >= 0 && st[i] % 8 == 0, MBRT_E_ALIGN, "%s: strides must be non-negative multiples of 8", op);
    }
    MBRT_REQUIRE((B == 1 || out_batch_stride > 0) && (H == 1 || out_head_stride > 0) && (n_q == 1 || out_row_stride > 0),
                 MBRT_E_SHAPE, "%s: rows of out overlap", op);
    const Plan plan = make_plan(B, H, H_kv, n_q, n_k, head_dim, left, right, std::min(sinks, n_k));
    const int64_t need = workspace_bytes_of(plan, B, H, n_q, head_dim);
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
    a.q_bs = st[0];
    a.q_hs = st[1];
    a.q_ns = st[2];
    a.kv_bs = st[3];
    a.kv_hs = st[4];
    a.kv_ns = st[5];
    a.o_bs = st[6];
    a.o_hs = st[7];
    a.o_ns = st[8];
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
    a.sl2 = sl2;
    a.gdiv = make_fastdiv((uint32_t)G);
    a.kvdiv = make_fastdiv((uint32_t)H_kv);
    a.splits = (uint32_t)plan.splits;
    hipStream_t stm = as_stream(stream);
    const int64_t bkv = B * H_kv;
    a.qtiles = (uint32_t)ceil_div(a.rows, plan.few ? 16 : 64 * plan.qs);
    const int64_t blocks = bkv * a.qtiles * plan.splits;
    MBRT_REQUIRE(grid_fits(blocks, plan.few ? kSplitWaves * 64 : 256), MBRT_E_SHAPE, "%s: too many tiles", op);
    auto launch = [&](auto dt, auto dim, auto parts) {
        constexpr int DTv = decltype(dt)::value, Dv = decltype(dim)::value, NP = decltype(parts)::value;
        if (!plan.few) {
            if constexpr (Dv == 128) {
                if (plan.qs == 2) {
                    hipLaunchKernelGGL((window_tile_kernel<DTv, Dv, 2, NP>), dim3((unsigned)blocks), dim3(256), 0, stm, a);
                    return;
                }
            }
            hipLaunchKernelGGL((window_tile_kernel<DTv, Dv, 1, NP>), dim3((unsigned)blocks), dim3(256), 0, stm, a);
            return;
        }
        const size_t lds = (size_t)kSplitWaves * 16 * (Dv + 2) * 4;  // the joined rows; the V tiles need less
        static_assert(kChunk * 2 * Dv <= 16 * (Dv + 2) * 4, "V tile within the rows' space");
        hipLaunchKernelGGL((window_split_kernel<DTv, Dv, DTv == BF16 ? 3 : 2>), dim3((unsigned)blocks), dim3(kSplitWaves * 64), lds, stm, a);
        if (plan.splits > 1)
            hipLaunchKernelGGL((window_join_kernel<DTv, Dv>), dim3((unsigned)(bkv * a.rows)), dim3(kJoinWaves * 64), 0, stm, a);
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
