// Operators on paged K/V caches, gfx950: store (per-head RMSNorm and rotation of new queries and keys,
// keys and values written to their slots as fp16 or q8), attention of every sequence's new tokens over
// its slots, load (slots read back).  A pool's K and V are row-major .icua matrices of 128 columns,
// rows [page][KV head][slot]: a (page, head)'s slots are contiguous, so a 16-slot tile is one run of
// 4 KiB (fp16) or 2 KiB of codes and 128 bytes of scales (q8).
#include <algorithm>
#include <type_traits>

#include "icua_device.h"
#include "icua_kernels.h"

namespace icua {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int QG = 32;       // values that share a q8 scale
constexpr int NG = HD / QG;  // scales of a row
constexpr float NEG_INF = -__builtin_inff();

// ------------------------------------------------------------------------------------------
// Rows of 128 values held by 16 lanes: lane l has values 4 l .. 4 l + 3 and 64 + 4 l .. + 3, so that
// the pairs (i, i + 64) of a whole-head rotation are in one lane and a q8 group is 8 lanes.

template <int TYPE>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i) {
    if constexpr (TYPE == TYPE_F32) return *(const f32x4*)((const float*)p + i);
    const v4h h = *(const v4h*)((const f16*)p + i);
    return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}
template <int TYPE>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
    if constexpr (TYPE == TYPE_F32)
        *(f32x4*)((float*)p + i) = v;
    else
        *(v4h*)((f16*)p + i) = v4h{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
}

// q8 code and scale of four values of a group held by 8 consecutive lanes, with the float32 steps of
// the converter's quantiser (Convert.swift:215-241), so a stored row of numbers has the bytes that
// quantising the float32 row as a matrix gives.  The maximum is taken of magnitudes as integers, in which
// NaN is the largest: a group with one gets a scale that is none (as floats the maximum passes it over, and
// its code would stand for the group's largest value).
__device__ __forceinline__ uint32_t q8_codes(f32x4 v, uint16_t& scale) {
#pragma clang fp contract(off)
    auto larger = [](float a, float b) { return as_f32(max(as_u32(a), as_u32(b))); };  // of magnitudes
    float amax = larger(larger(fabsf(v[0]), fabsf(v[1])), larger(fabsf(v[2]), fabsf(v[3])));
    amax = larger(amax, dpp<DPP_XOR1>(amax));
    amax = larger(amax, dpp<DPP_XOR2>(amax));
    amax = larger(amax, dpp<DPP_HALF_MIRROR>(amax));
    uint16_t sh = f2h(amax / 127.0f);
    if (h2f(sh) * 127.0f < amax) sh = (uint16_t)(sh + 1u);
    scale = sh;
    const float s = h2f(sh);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        word |= (uint32_t)(uint8_t)(int8_t)fmaxf(-127.0f, fminf(127.0f, roundf(v[k] * inv))) << (8 * k);
    return word;
}

// Rotation of four values x at d .. d + 3 of a head whose first `rot` values turn: pairs (i, i + rot / 2),
// or (2 i, 2 i + 1) interleaved.  o: for the first layout the four partners, normalised as x is.
__device__ __forceinline__ f32x4 rotate4(f32x4 x, f32x4 o, int d, int rot, bool interleaved, const float* cs) {
    if (d >= rot) return x;
    if (interleaved) {
        const f32x4 t = *(const f32x4*)(cs + d);  // (cos, sin) of pairs d / 2 and d / 2 + 1
        return f32x4{x[0] * t[0] - x[1] * t[1], x[1] * t[0] + x[0] * t[1], x[2] * t[2] - x[3] * t[3],
                     x[3] * t[2] + x[2] * t[3]};
    }
    const int half = rot / 2, i = d < half ? d : d - half;
    const f32x4 t0 = *(const f32x4*)(cs + 2 * i), t1 = *(const f32x4*)(cs + 2 * i + 4);
    const float c[4] = {t0[0], t0[2], t1[0], t1[2]}, s[4] = {t0[1], t0[3], t1[1], t1[3]};
    f32x4 y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = d < half ? x[k] * c[k] - o[k] * s[k] : x[k] * c[k] + o[k] * s[k];
    return y;
}

// 16 lanes a (token, head) vector, 16 vectors a workgroup.  Bound by memory: a token's row is read once
// and its queries, keys and values written once.  4096 tokens of 16 + 8 + 8 heads, fp32 in, fp16 out: 101 MB in
// 24 us, 4.2 TB/s, four fifths of what a copy reaches; eight tokens: 3.4 us, a launch.
template <int TYPE, int QTYPE, int FMT>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedStoreArgs a) {
    const int nvec = a.n_heads + 2 * a.map.n_kv;
    const int64_t v = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (v >= (int64_t)a.n_tokens * nvec) return;
    const int t = (int)(v / nvec), vec = (int)(v - (int64_t)t * nvec), l = threadIdx.x % 16;
    const bool is_q = vec < a.n_heads, is_v = vec >= a.n_heads + a.map.n_kv;
    const int pos = a.pos ? a.pos[t] : 0;
    const int64_t at = (int64_t)t * a.qkv_stride + vec * HD;
    // Loaded before the slot and position are there (a prompt of 4096 tokens: 24.8 us else).
    f32x4 x[2] = {load4<TYPE>(a.qkv, at + 4 * l), load4<TYPE>(a.qkv, at + 64 + 4 * l)};
    const bool pos_ok = !a.rot || (pos >= 0 && pos < a.rope_rows);
    const int row = is_q ? 0 : pool_slot_row(a.map, a.slots[t]);
    if (!is_q && (row < 0 || !pos_ok)) return;
    if (!is_v) {
        const float* w = is_q ? a.q_norm : a.k_norm;
        float scale = 1.0f;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) ss += x[0][k] * x[0][k] + x[1][k] * x[1][k];
            scale = 1.0f / sqrtf(sum16(ss) / (float)HD + a.eps);
        }
        auto normed = [&](f32x4 y, int d) {
            if (!w) return y;
            return y * scale * *(const f32x4*)(w + d);
        };
        f32x4 y[2] = {normed(x[0], 4 * l), normed(x[1], 64 + 4 * l)};
        if (a.rot && pos_ok) {
            const float* cs = a.rope + (int64_t)pos * a.rot;
            f32x4 o[2] = {y[1], y[0]};
            if (a.rot != HD && !a.interleaved)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 64 * h + 4 * l, p = d < a.rot / 2 ? d + a.rot / 2 : d - a.rot / 2;
                    if (d < a.rot) o[h] = normed(load4<TYPE>(a.qkv, at + p), p);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = rotate4(y[h], o[h], 64 * h + 4 * l, a.rot, a.interleaved, cs);
        } else {
            x[0] = y[0];
            x[1] = y[1];
        }
    }
    if (is_q) {
        if (!pos_ok) x[0] = x[1] = f32x4{} + __builtin_nanf("");  // a position outside the table: no query
        const int64_t o = (int64_t)t * a.q_stride + vec * HD;
        store4<QTYPE>(a.q, o + 4 * l, x[0]);
        store4<QTYPE>(a.q, o + 64 + 4 * l, x[1]);
        return;
    }
    const int64_t r = (int64_t)row + (int64_t)(vec - a.n_heads - (is_v ? a.map.n_kv : 0)) * a.map.page_slots;
    void* dst = is_v ? a.v : a.k;
    if constexpr (FMT == FMT_F16) {
        store4<TYPE_F16>(dst, r * HD + 4 * l, x[0]);
        store4<TYPE_F16>(dst, r * HD + 64 + 4 * l, x[1]);
    } else {
        uint16_t* sb = (uint16_t*)(is_v ? a.v_sb : a.k_sb);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint16_t s;
            const uint32_t codes = q8_codes(x[h], s);
            *(uint32_t*)((int8_t*)dst + r * HD + 64 * h + 4 * l) = codes;
            if (l % 8 == 0) sb[r * NG + 2 * h + l / 8] = s;
        }
    }
}

// ------------------------------------------------------------------------------------------
// Read-back: 16 lanes a (row, KV head), 8 values a lane, K and V by one lane.  Bound by memory: 16 sessions of up
// to 16384 fp16 slots in 186 us, 5.8 TB/s of reads and writes; 4096 q8 slots, 26 MB, in 7 us.
template <int TYPE, int FMT>
__global__ __launch_bounds__(256) void paged_load_kernel(PagedLoadArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (i >= (int64_t)a.n_rows * a.map.n_kv) return;
    const int t = (int)(i / a.map.n_kv), g = (int)(i - (int64_t)t * a.map.n_kv), l = threadIdx.x % 16;
    const int row = pool_slot_row(a.map, a.slots[t]);
    if (row < 0) return;
    const int64_t r = (int64_t)row + (int64_t)g * a.map.page_slots;
    const int64_t o = (int64_t)t * a.token_stride + (int64_t)g * a.head_stride + 8 * l;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const void* src = kv ? a.v : a.k;
        void* dst = kv ? a.v_out : a.k_out;
        if (!dst) continue;
        float x[8];
        if constexpr (FMT == FMT_F16) {
            const v8h h = *(const v8h*)((const f16*)src + r * HD + 8 * l);
            if constexpr (TYPE == TYPE_F16) {
                *(v8h*)((f16*)dst + o) = h;
                continue;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (float)h[k];
        } else {
            const u32x2 c = *(const u32x2*)((const int8_t*)src + r * HD + 8 * l);
            const float s = h2f(((const uint16_t*)(kv ? a.v_sb : a.k_sb))[r * NG + l / 4]);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = s * (float)(int8_t)(c[k / 4] >> (8 * (k % 4)));
        }
        store4<TYPE>(dst, o, f32x4{x[0], x[1], x[2], x[3]});
        store4<TYPE>(dst, o + 4, f32x4{x[4], x[5], x[6], x[7]});
    }
}

// ------------------------------------------------------------------------------------------
// Attention.  out = softmax(scale q . k) v over the slots that a token sees, one pass with a running
// maximum m and denominator l:  m' = max(m, s), l' = l e^(m - m') + e^(s - m'), O' likewise.
//
// A KV head's query rows are (token i, head of the group h), numbered i * group + h.  Products run
// transposed on v_mfma_f32_16x16x32_f16, 16 query rows as columns: S^T = K Q^T leaves lane (column c,
// q) with slots 4 q .. 4 q + 3 of a 16-slot tile, which is the B operand of O^T = V^T P^T when the V
// operand takes its slots in that order.  Exponentials are taken of base-2 scores, shifted by 2^9 (of
// numerator and denominator alike): fp16 probabilities down to 2^-33 of the largest keep their value,
// where unshifted ones would round to nothing below 2^-24, which adds up over long caches.  The maximum
// that is subtracted may lag 2^6 behind the true one, so accumulators are seldom rescaled.
//
// fp32 queries and probabilities are split into fp16 hi + lo parts, two products each; queries are
// first scaled by a power of two that puts the row's largest value in [2^9, 2^10), so that neither
// part leaves fp16's range.  The parts of a probability have 22 bits from 2^-12 of the row's largest on, and
// 2^-34 of the largest below that.

constexpr float P_SHIFT = 9.0f, P_SLACK = 6.0f;

// Max over the lanes l and l ^ 32.
__device__ __forceinline__ float max_x2(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
    return fmaxf(as_f32(r[0]), as_f32(r[1]));
}
// The power of two that scales a query row with this largest magnitude.
__device__ __forceinline__ int query_shift(float amax) {
    return amax > 0.f && amax < __builtin_inff() ? 10 - __builtin_amdgcn_frexp_expf(amax) : 0;
}

// The query rows of a workgroup's tile: which token and head a column stands for.
struct RowOf {
    int t;     // token of the call, -1: no such row
    int head;
    int last;  // last slot that it sees (negative: none)
};
__device__ __forceinline__ RowOf row_of(const SeqSpan& sp, int row, int group, int g) {
    const int i = row / group;
    if (i >= sp.n_q) return {-1, 0, -1};
    return {sp.t0 + i, g * group + row - i * group, sp.n_kv - sp.n_q + i};
}

// The B operands of a column's query and the factor that turns its products into base-2 scores.
template <int TYPE>
struct Query {
    v8h hi[4], lo[TYPE == TYPE_F32 ? 4 : 1];
    float c;
};
// Its values as they are in memory, and the operands made of them: what is loaded in between is under way
// meanwhile.
template <int TYPE>
struct QueryRow {
    u32x4 x[TYPE == TYPE_F32 ? 8 : 4];
};
template <int TYPE>
__device__ __forceinline__ QueryRow<TYPE> load_query(const PagedAttnArgs& a, const RowOf& r, int q) {
    QueryRow<TYPE> y;
    const int64_t at = (int64_t)r.t * a.q_stride + r.head * HD + 8 * q;
    if constexpr (TYPE == TYPE_F16) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) y.x[ks] = r.t < 0 ? u32x4{} : *(const u32x4*)((const f16*)a.q + at + 32 * ks);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) y.x[k] = r.t < 0 ? u32x4{} : *(const u32x4*)((const float*)a.q + at + 32 * (k / 2) + 4 * (k % 2));
    }
    return y;
}
template <int TYPE>
__device__ __forceinline__ Query<TYPE> query_of(const QueryRow<TYPE>& r, float scale) {
    Query<TYPE> y;
    y.c = scale * 1.4426950408889634f;
    if constexpr (TYPE == TYPE_F16) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) y.hi[ks] = __builtin_bit_cast(v8h, r.x[ks]);
    } else {
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(as_f32(r.x[k][e])));
        amax = max_x4(amax);
        const int k2 = query_shift(amax);
        y.c = ldexpf(y.c, -k2);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = ldexpf(as_f32(r.x[k][e]), k2);
                const f16 h = (f16)v;
                y.hi[k / 2][4 * (k % 2) + e] = h;
                y.lo[k / 2][4 * (k % 2) + e] = (f16)(v - (float)h);
            }
    }
    return y;
}

__device__ __forceinline__ f32x4 mfma(v8h a, v8h b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// A 16-slot tile of K or V as a lane reads it from memory (K: slot r16, dims 32 ks + 8 q .. + 7; V: slots
// 4 q .. + 3, dims 8 r16 .. + 7), with q8 scales (K: slots 4 q .. + 3, four each; V: of its 8 dims).
template <int FMT>
struct Tile {
    u32x4 k[4], v[4];
};
template <>
struct Tile<FMT_Q8> {
    u32x2 k[4], v[4];
    u32x4 ks[2];
    uint16_t vs[4];
};
// Any values: those of a tile of before need not be kept.
template <int FMT>
__device__ __forceinline__ void no_tile(Tile<FMT>* t) {
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t[j].k[i] = __builtin_nondeterministic_value(t[j].k[i]);
            t[j].v[i] = __builtin_nondeterministic_value(t[j].v[i]);
            if constexpr (FMT == FMT_Q8) t[j].vs[i] = __builtin_nondeterministic_value(t[j].vs[i]);
        }
        if constexpr (FMT == FMT_Q8)
#pragma unroll
            for (int i = 0; i < 2; ++i) t[j].ks[i] = __builtin_nondeterministic_value(t[j].ks[i]);
    }
}
template <int FMT>
__device__ __forceinline__ void load_tile(const PagedAttnArgs& a, int row, int lane, Tile<FMT>& t) {
    const int q = lane >> 4, r16 = lane & 15;
    if constexpr (FMT == FMT_F16) {
        const uint8_t* k = (const uint8_t*)a.k + (int64_t)row * (HD * 2) + r16 * (HD * 2) + q * 16;
        const uint8_t* v = (const uint8_t*)a.v + (int64_t)row * (HD * 2) + q * 4 * (HD * 2) + r16 * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) t.k[i] = *(const u32x4*)(k + 64 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.v[i] = *(const u32x4*)(v + i * HD * 2);
    } else {
        const uint8_t* k = (const uint8_t*)a.k + (int64_t)row * HD + r16 * HD + q * 8;
        const uint8_t* ks = (const uint8_t*)a.k_sb + (int64_t)row * (NG * 2) + q * 32;
        const uint8_t* v = (const uint8_t*)a.v + (int64_t)row * HD + q * 4 * HD + r16 * 8;
        const uint16_t* vs = (const uint16_t*)a.v_sb + (int64_t)row * NG + q * 4 * NG + r16 / 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) t.k[i] = *(const u32x2*)(k + 32 * i);
        t.ks[0] = *(const u32x4*)ks;
        t.ks[1] = *(const u32x4*)(ks + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.v[i] = *(const u32x2*)(v + i * HD);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.vs[i] = vs[i * NG];
    }
}

// All ones for the bits of an infinity or no number, else zero.
__device__ __forceinline__ uint32_t no_number(uint32_t x) { return (uint32_t)((int32_t)((x & 0x7F800000u) + 0x00800000u) >> 31); }

// Four int8 codes as exact fp16 values: code + 128 under the exponent of 1024 is 1152 + code.
__device__ __forceinline__ void codes_h2(uint32_t w, f16x2 y[2]) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 bias = {(f16)1152.f, (f16)1152.f};
    y[0] = as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x05010400u)) - bias;
    y[1] = as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x05030402u)) - bias;
}

// Replaces values that are no numbers by finite ones; `odd` is not zero if there were any.
__device__ __forceinline__ void keep_finite(v8h& v, uint32_t& odd) {
    const v8h top = (v8h)(f16)65504.f, fin = __builtin_elementwise_max(__builtin_elementwise_min(v, top), -top);
    const u32x4 d = __builtin_bit_cast(u32x4, v) ^ __builtin_bit_cast(u32x4, fin);
    odd |= d[0] | d[1] | d[2] | d[3];
    v = fin;
}

// Scores of a tile, products with the column's query: fp16 rows directly; q8 codes are exact in fp16
// and a 32-value group is one product's depth, so each group's sum takes its scale in fp32.
template <int TYPE, int FMT>
__device__ __forceinline__ f32x4 tile_scores(const Tile<FMT>& t, const Query<TYPE>& y) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        if constexpr (FMT == FMT_F16) {
            const v8h k = __builtin_bit_cast(v8h, t.k[ks]);
            s = mfma(k, y.hi[ks], s);
            if constexpr (TYPE == TYPE_F32) s = mfma(k, y.lo[ks], s);
        } else {
            f16x2 c[4];
            codes_h2(t.k[ks][0], c);
            codes_h2(t.k[ks][1], c + 2);
            const v8h k = {c[0].x, c[0].y, c[1].x, c[1].y, c[2].x, c[2].y, c[3].x, c[3].y};
            f32x4 p = mfma(k, y.hi[ks], f32x4{0.f, 0.f, 0.f, 0.f});
            if constexpr (TYPE == TYPE_F32) p = mfma(k, y.lo[ks], p);
            // The scale of slot 4 q + i, group ks: half 4 i + ks of t.ks.
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[i] = __builtin_fmaf(p[i], h2f((uint16_t)(t.ks[i / 2][2 * (i % 2) + ks / 2] >> (16 * (ks % 2)))), s[i]);
        }
    }
    return s;
}

// q8: the largest scale (its fp16 bits) whose products with codes are all fp16 numbers: 256.
constexpr uint16_t V_TOP = 0x5C00;
__device__ __forceinline__ bool beyond_fp16(uint16_t scale) { return (scale & 0x7FFF) > V_TOP; }

// The V^T operand dims 8 r16 + dt of two tiles over this lane's eight slots (4 q .. + 3 of each tile), hi
// and, for q8, the lo part of the exact product code x scale (scales up to V_TOP).
template <int TYPE, int FMT>
struct VOp {
    static constexpr bool LO = FMT == FMT_Q8;
    v8h hi, lo;
};
template <int TYPE, int FMT>
__device__ __forceinline__ VOp<TYPE, FMT> v_operand(const Tile<FMT>* t, int dt) {
    VOp<TYPE, FMT> o;
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // slots 2 j, 2 j + 1 of the eight
        const Tile<FMT>& x = t[j / 2];
        const int r = 2 * (j % 2);
        if constexpr (FMT == FMT_F16) {
            // The low (even dt) or high halves of a word of two rows: one byte select.
            hi[j] = __builtin_amdgcn_perm(x.v[r + 1][dt / 2], x.v[r][dt / 2], dt % 2 ? 0x07060302u : 0x05040100u);
        } else {
            // Byte dt % 4 of both rows' words (sign flipped before) under the exponent of 1024, less 1152.
            const uint32_t sel = 0x0C000C00u | (uint32_t)(dt % 4) | (uint32_t)(4 + dt % 4) << 16;
            const f16x2 bias = {(f16)1152.f, (f16)1152.f};
            const f16x2 c = as_h2(__builtin_amdgcn_perm(x.v[r + 1][dt / 4], x.v[r][dt / 4], sel) | 0x64006400u) - bias;
            const f16x2 s = as_h2((uint32_t)x.vs[r] | (uint32_t)x.vs[r + 1] << 16);
            const f16x2 h = c * s;
            hi[j] = h2_bits(h);
            if constexpr (VOp<TYPE, FMT>::LO) lo[j] = h2_bits(__builtin_elementwise_fma(c, s, -h));  // exact
        }
    }
    o.hi = __builtin_bit_cast(v8h, hi);
    if constexpr (VOp<TYPE, FMT>::LO) o.lo = __builtin_bit_cast(v8h, lo);
    return o;
}

// Value d of a row of V.
template <int FMT>
__device__ __forceinline__ float row_value(const void* v, const void* v_sb, int64_t row, int d) {
    if constexpr (FMT == FMT_F16) return (float)((const f16*)v)[row * HD + d];
    return h2f(((const uint16_t*)v_sb)[row * NG + d / QG]) * (float)((const int8_t*)v)[row * HD + d];
}

// The slots that a sequence goes through: with a window all but those between the first ones and its first row's
// window; behind a shared prefix those after it.  The prefix itself is gone through once for the rows of all the
// group's tokens (the chunk kernel's first workgroups), and a row's two parts are joined.

// Lane g: group g.  (Its loads, and those of span_of, are of places inside the arrays whether they count or not, so
// that they are all under way together.)
template <int FORM>
__device__ __forceinline__ PrefixGroup load_groups(const PagedAttnArgs& a) {
    if constexpr (FORM != PAGED_PREFIX) return {0, 0, 0};
    const int g = threadIdx.x & 63;
    PrefixGroup y = prefix_group(a.group_start, a.prefix_len, min(g, a.f.n_groups - 1), a.n_seqs, a.f.max_prefix);
    if (g >= a.f.n_groups) y = {0, 0, 0};
    return y;
}
struct Span {
    SeqSpan sp;
    SlotGap gap;  // (a 128-row tile of a window has its own)
    __device__ __forceinline__ int slots() const { return max(0, sp.n_kv - gap.skip); }
};
// Lane i: sequence s0 + i.
template <int FORM>
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, const PrefixGroup& gr, int s0) {
    const int s = s0 + (int)(threadIdx.x & 63);
    Span y = {{0, 0, 0}, {0, 0}};
    if constexpr (FORM == PAGED_ALL) {
        if (s < a.n_seqs) y.sp = seq_span(a.q_start, a.kv_len, s, a.n_tokens, a.max_kv);
        return y;
    }
    y.sp = seq_span(a.q_start, a.kv_len, min(s, a.n_seqs - 1), a.n_tokens, a.max_kv);
    if (s >= a.n_seqs) y.sp = {0, 0, 0};
    if constexpr (FORM == PAGED_WINDOW) y.gap = window_gap(y.sp.n_kv - y.sp.n_q, y.sp.n_kv, a.f.window, a.f.sinks, 32);
    if constexpr (FORM == PAGED_PREFIX) {
        int first, last, n;
        if (a.f.n_groups == 1) {
            first = __builtin_amdgcn_readfirstlane(gr.s0), last = __builtin_amdgcn_readfirstlane(gr.s1), n = __builtin_amdgcn_readfirstlane(gr.n);
        } else {  // the last group that begins at s or before
            int g = 0;
            for (int step = 1 << (31 - __builtin_clz(a.f.n_groups - 1)); step; step >>= 1) {
                const int next = g + step, begin = __shfl(gr.s0, next % WAVE);
                if (next < a.f.n_groups && begin <= s) g = next;
            }
            first = __shfl(gr.s0, g), last = __shfl(gr.s1, g), n = __shfl(gr.n, g);
        }
        if (s >= first && s < last) y.gap.skip = n;
    }
    return y;
}
// The last slot of a prefix of n slots that this lane's token t sees; true if all tokens of the group's sequences
// see all of it.
__device__ __forceinline__ bool prefix_last(const PagedAttnArgs& a, int s0, int s1, int n, int t, int& last) {
    bool all = true;
    last = n - 1;
    for (int b = s0; b < s1; b += WAVE) {
        SeqSpan x = {0, 0, 0};
        if (b + (int)(threadIdx.x & 63) < s1) x = seq_span(a.q_start, a.kv_len, b + (threadIdx.x & 63), a.n_tokens, a.max_kv);
        uint64_t few = __ballot(x.n_q > 0 && x.n_kv - x.n_q < n - 1);
        for (; few; few &= few - 1) {
            all = false;
            const int j = __ffsll((unsigned long long)few) - 1;
            const int t0 = __builtin_amdgcn_readlane(x.t0, j), m = __builtin_amdgcn_readlane(x.n_q, j), kv = __builtin_amdgcn_readlane(x.n_kv, j);
            if (t >= t0 && t < t0 + m) last = min(last, kv - m + t - t0);
        }
    }
    return all;
}

// Sequences with at most 16 query rows a KV head (single tokens, drafts).  Their slots, in units of a step
// of all waves of a workgroup, are dealt out evenly: workgroup w of a KV head's `few.n` has units w * per ..
// of all sequences in a row, whatever the sequences' lengths.  A sequence that lies in one workgroup is
// done there; of the others each workgroup leaves a partial, at most two: a sequence's end, or a part from
// its middle, as the first and a beginning as the second.
//
// One workgroup a (sequence, KV head, range of slots) instead, as even as the longest sequence allows, takes
// half again as long for lengths that differ by factors of up to 8.
constexpr int ROWS_TILE = 16, ROWS_STEP = 32;
constexpr int ROWS_PITCH = 80;  // 16-byte places of a wave's results of one dt
// Of the forms with a gap each wave keeps its 64 sequences in LDS, not in registers: places of `kept` and `more`.
template <int NW>
constexpr size_t rows_lds(int form) { return NW * (8 * ROWS_PITCH * 16 + 16 * 8 + (form == PAGED_ALL ? 0 : WAVE * 32)); }

// Lane i: sequence s0 + i, its units (0: the chunk kernel's, or none) and those up to its end since s0; `sum`:
// of all 64.
struct FewUnits {
    Span x;
    int n, end, sum;
};
template <int FORM>
__device__ __forceinline__ FewUnits few_units(const PagedAttnArgs& a, const PrefixGroup& gr, int group, int s0) {
    const int lane = threadIdx.x & 63;
    FewUnits u = {span_of<FORM>(a, gr, s0), 0, 0, 0};
    if (u.x.sp.n_q > 0 && u.x.sp.n_q * group <= ROWS_TILE) u.n = max(1, (u.x.slots() + a.few.unit - 1) / a.few.unit);
    u.end = u.n;
    for (int o = 1; o < min(WAVE, a.n_seqs); o <<= 1) {
        const int y = __shfl_up(u.end, o);
        if (lane >= o) u.end += y;
    }
    u.sum = __builtin_amdgcn_readlane(u.end, min(WAVE, a.n_seqs) - 1);
    return u;
}
// Units a workgroup takes, of this many.
__device__ __forceinline__ int few_per(const PagedAttnArgs& a, int total) {
    const int per = max(a.few.least, (int)(((unsigned)total + a.few.n - 1) / (unsigned)a.few.n));
    return per > a.few.twice ? 2 * per : per;
}

// A workgroup of NW waves: its waves take 32-slot steps of a sequence in turn and join through LDS.  K and V
// go from memory to registers, as each is used by one tile alone, a step ahead of its products: two waves a SIMD
// with a step in flight each; three or four without one are no faster, and a step ahead with three does not fit
// the registers.  A step's latency is 2.4 us from memory, the queries' and tables' before it some 2 us, so a
// single token over 4096 slots is bound by latency: 9 us, and 4 to join.  Long caches are bound by memory: eight
// tokens over up to 32768 fp16 slots 115 us, 5.4 TB/s; 64 tokens over up to 8192 q8 slots 105 us, 4.7 TB/s (a q8
// step is some 450 instructions, 2.7 us of a wave), 113 with fp32 queries.  Those spill 15 registers (fp16 slots)
// and 5 (q8), fp16 queries none.
template <int FORM, int TYPE, int FMT, int NW>
__device__ __forceinline__ void rows_work(const PagedAttnArgs& a, int index, uint8_t* lds) {
    // fp32 probabilities in two parts.  With fp16 queries and q8, two parts of V cost as much as two of the
    // probabilities and leave the smaller error (2.5e-4 for 2.9e-4 of the outputs' rms, 2.1e-4 the output's own).
    constexpr bool PLO = TYPE == TYPE_F32, VLO = VOp<TYPE, FMT>::LO;
    f32x4* const so = (f32x4*)lds;                                  // [NW][8][ROWS_PITCH]
    float2* const sml = (float2*)(lds + NW * 8 * ROWS_PITCH * 16);  // [NW][16]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, r16 = lane & 15;
    const int g = index % a.map.n_kv, w = index / a.map.n_kv, group = a.n_heads / a.map.n_kv;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4* const kept = (i32x4*)(lds + NW * (8 * ROWS_PITCH * 16 + 16 * 8)) + wave * 2 * WAVE;  // (t0, n_q, n_kv, units)
    i32x4* const more = kept + WAVE;                                                           // (units up to its end, gap)
    FewUnits u;
    PrefixGroup gr = load_groups<FORM>(a);
    auto keep = [&]() __attribute__((always_inline)) {
        if constexpr (FORM != PAGED_ALL) {
            kept[lane] = i32x4{u.x.sp.t0, u.x.sp.n_q, u.x.sp.n_kv, u.n};
            more[lane] = i32x4{u.end, u.x.gap.from, u.x.gap.skip, 0};
        }
    };
    // Whole windows: sequence w, if it is one of these, without a look at those before.
    const bool one = FORM == PAGED_WINDOW && a.few.whole;
    int s0 = one ? w / WAVE * WAVE : 0, before = 0, pos, end;
    u = few_units<FORM>(a, gr, group, s0);
    if (one) {
        end = __builtin_amdgcn_readlane(u.end, w % WAVE);
        pos = end - __builtin_amdgcn_readlane(u.n, w % WAVE);
    } else {
        int total = u.sum;
        for (int s1 = WAVE; s1 < a.n_seqs; s1 += WAVE) total += few_units<FORM>(a, gr, group, s1).sum;
        const int per = few_per(a, total);
        pos = w * per;
        end = min(total, pos + per);
    }
    keep();
    while (pos < end) {
        // The sequence that has unit pos, and where its units begin.
        const uint64_t past = __ballot(before + (FORM == PAGED_ALL ? u.end : more[lane][0]) > pos);
        if (!past) {
            before += u.sum;
            s0 += WAVE;
            if (s0 >= a.n_seqs) return;
            gr = load_groups<FORM>(a);
            u = few_units<FORM>(a, gr, group, s0);
            keep();
            continue;
        }
        const int at_lane = __ffsll((unsigned long long)past) - 1;
        i32x4 k = {}, x = {};
        if constexpr (FORM == PAGED_ALL) {
            k = i32x4{__builtin_amdgcn_readlane(u.x.sp.t0, at_lane), __builtin_amdgcn_readlane(u.x.sp.n_q, at_lane), __builtin_amdgcn_readlane(u.x.sp.n_kv, at_lane), __builtin_amdgcn_readlane(u.n, at_lane)};
            x[0] = __builtin_amdgcn_readlane(u.end, at_lane);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                k[i] = __builtin_amdgcn_readfirstlane(kept[at_lane][i]);
                x[i] = __builtin_amdgcn_readfirstlane(more[at_lane][i]);
            }
        }
        const int seq_end = before + x[0], seq_units = k[3], first = pos - (seq_end - seq_units), count = min(end, seq_end) - pos;
        const SeqSpan sp = {k[0], k[1], k[2]};
        const bool whole = count == seq_units;
        pos += count;
        const RowOf row = row_of(sp, r16, group, g);
        // Slots that some row sees: 0 .. lim - 1; all of them see those up to `all`.  (Of a window: and those of its own.)
        const int start = first * a.few.unit;
        const int lim = sp.n_kv, all = sp.n_kv - sp.n_q;
        const SlotGap gap = {FORM == PAGED_WINDOW ? x[1] : 0, x[2]};
        const bool joined = FORM == PAGED_PREFIX && gap.skip > 0;  // to its prefix's part
        const int c1 = min(FORM == PAGED_ALL ? lim : max(0, lim - gap.skip), start + count * a.few.unit);  // of numbers without the gap
        // Whether this lane's row sees a slot, and whether no row does.  (Without short cuts: selects, no branches.  Where
        // p[i] = -inf comes after branches inside branches, the compiler, ROCm 7.2's, joins the copies of p's tuple of
        // registers so that the write is lost: its block is an s_and_saveexec with its s_or right behind it, empty.)
        auto sees = [&](int slot) __attribute__((always_inline)) -> bool {
            if constexpr (FORM != PAGED_WINDOW) return slot <= row.last;
            return (slot <= row.last) & ((slot < a.f.sinks) | (slot > row.last - a.f.window));
        };
        auto unseen = [&](int slot) __attribute__((always_inline)) -> bool {
            if constexpr (FORM != PAGED_WINDOW) return false;
            return (slot >= a.f.sinks) & (slot <= all - a.f.window);
        };
        const int32_t* table = a.tables + (int64_t)(s0 + at_lane) * a.table_width;
        // Lane i: the pool row of tile i % 2 of this wave's step i / 2 from `sub` on (-1: no such page).
        auto step_slot = [&](int sub, int i) { return sub + ROWS_STEP * (wave + NW * i); };
        auto lookup = [&](int sub) {
            const int slot = step_slot(sub, lane / 2) + PAGED_TILE * (lane % 2);
            return slot < c1 ? seq_slot_row(a.map, table, a.table_width, gap_slot(gap, slot)) : -1;
        };
        constexpr int SUB = NW * ROWS_STEP * (WAVE / 2);
        int rows = lookup(start);

        f32x4 O[8];
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = NEG_INF, l = 0.f;
        int sub = start;
        auto fetch = [&](int i, Tile<FMT>* t) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
                load_tile<FMT>(a, max(__builtin_amdgcn_readlane(rows, 2 * i + k), 0) + g * a.map.page_slots, lane, t[k]);
        };
        // This wave's steps of the window that begin below c1.
        auto steps = [&]() {
            const int left = c1 - step_slot(sub, 0);
            return left <= 0 ? 0 : min(WAVE / 2, (left + NW * ROWS_STEP - 1) / (NW * ROWS_STEP));
        };
        const QueryRow<TYPE> qrow = load_query<TYPE>(a, row, q);
        Tile<FMT> A[2], B[2];
        no_tile<FMT>(A);
        no_tile<FMT>(B);
        int n = steps();
        if (n > 0) fetch(0, A);
        const Query<TYPE> y = query_of<TYPE>(qrow, a.scale);
        auto step = [&](int i, Tile<FMT>* t) __attribute__((always_inline)) {
            const int at = gap_slot(gap, step_slot(sub, i));
            const int ok[2] = {__builtin_amdgcn_readlane(rows, 2 * i) < 0 ? 0 : lim, __builtin_amdgcn_readlane(rows, 2 * i + 1) < 0 ? 0 : lim};
            float p[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x4 sc = tile_scores<TYPE, FMT>(t[k], y);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[4 * k + e] = sc[e] * y.c;
            }
            uint32_t odd = 0;
            bool masked = at + ROWS_STEP - 1 > all || ok[0] == 0 || ok[1] == 0;
            if constexpr (FORM == PAGED_WINDOW) masked |= at + ROWS_STEP > a.f.sinks && at <= lim - 1 - a.f.window;
            if (masked) {
                asm volatile("");
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int slot = at + 16 * k + 4 * q + e;
                        if (!sees(slot) | (slot >= ok[k])) p[4 * k + e] = NEG_INF;
                        // Values of slots that no row sees may be anything: they take no part.
                        if ((slot >= ok[k]) | unseen(slot)) {
                            t[k].v[e] = 0;
                            if constexpr (FMT == FMT_Q8) t[k].vs[e] = 0;
                        }
                    }
            }
            float mb = NEG_INF;
#pragma unroll
            for (int e = 0; e < 8; ++e) mb = fmaxf(mb, p[e]);
            mb = max_x4(mb);
            if (__ballot(mb > m + P_SLACK)) {
                asm volatile("");
                const float m_new = fmaxf(m, mb);
                const float corr = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= corr;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) O[dt] *= corr;
            }
            const float base = m == NEG_INF ? 0.f : m - P_SHIFT;
            v8h ph, pl;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(p[e] - base);
                l += x;
                ph[e] = (f16)x;
                if constexpr (PLO) pl[e] = (f16)(x - (float)ph[e]);
            }
            // q8: groups of slots with scales beyond V_TOP, or that are no numbers, are kept out of the products
            // (scale 0) and added in fp32.
            bool beyond = false;
            if constexpr (FMT == FMT_Q8) {
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                u16x2 top = {0, 0};
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        t[k].v[e] ^= 0x80808080u;
                        if (e % 2 == 0)
                            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, ((uint32_t)t[k].vs[e] | (uint32_t)t[k].vs[e + 1] << 16) & 0x7FFF7FFFu));
                    }
                beyond = __ballot(max(top.x, top.y) > V_TOP) != 0;
                if (beyond) {
                    asm volatile("");
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (beyond_fp16(t[k].vs[e])) t[k].vs[e] = 0;
                }
            }
            // f16, slots that some rows see and others do not: values there that are no numbers are kept out of
            // the products and go to the rows that see them.
            auto values = [&](auto finite) __attribute__((always_inline)) {
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    VOp<TYPE, FMT> v = v_operand<TYPE, FMT>(t, dt);
                    if constexpr (finite) keep_finite(v.hi, odd);
                    O[dt] = mfma(v.hi, ph, O[dt]);
                    if constexpr (PLO) O[dt] = mfma(v.hi, pl, O[dt]);
                    if constexpr (VLO) O[dt] = mfma(v.lo, ph, O[dt]);
                }
            };
            if constexpr (FMT == FMT_Q8)
                values(std::false_type());
            else if (masked)
                values(std::true_type());
            else
                values(std::false_type());
            if (beyond)
                for (int j = 0; j < ROWS_STEP; ++j) {
                    const int r = __builtin_amdgcn_readlane(rows, 2 * i + j / PAGED_TILE);
                    if (r < 0 || at + j >= lim) continue;
                    // The row's probability is lane (r16, j % 16 / 4)'s, element 4 (j / 16) + j % 4.
                    auto of_slot = [&](const v8h& p8) __attribute__((always_inline)) {
                        const u32x4 w = __builtin_bit_cast(u32x4, p8);
                        const uint32_t two = j & 16 ? (j & 2 ? w[3] : w[2]) : (j & 2 ? w[1] : w[0]);
                        return h2f((uint16_t)(__shfl((int)two, r16 + 16 * (j % 16 / 4)) >> (16 * (j & 1))));
                    };
                    float pj = of_slot(ph);
                    if constexpr (PLO) pj += of_slot(pl);
                    const int64_t vrow = (int64_t)r + g * a.map.page_slots + j % PAGED_TILE;
                    const uint16_t scale = ((const uint16_t*)a.v_sb)[vrow * NG + q];  // dims 32 q .. + 31 are group q
                    const uint32_t seen = sees(at + j) ? 0xFFFFFFFFu : 0;
                    if (!beyond_fp16(scale)) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int dt = 0; dt < 8; ++dt) {
                            const float x = row_value<FMT>(a.v, a.v_sb, vrow, 32 * q + 8 * e + dt);
                            O[dt][e] += no_number(as_u32(x)) ? as_f32(as_u32(x) & seen) : pj * x;
                        }
                }
            if (__ballot(odd != 0))
                for (int j = 0; j < ROWS_STEP; ++j) {
                    const int r = __builtin_amdgcn_readlane(rows, 2 * i + j / PAGED_TILE);
                    if (r < 0 || at + j >= lim) continue;
                    const int64_t vrow = (int64_t)r + g * a.map.page_slots + j % PAGED_TILE;
                    const uint32_t seen = sees(at + j) ? 0xFFFFFFFFu : 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int dt = 0; dt < 8; ++dt) {
                            const uint32_t x = as_u32(row_value<FMT>(a.v, a.v_sb, vrow, 32 * q + 8 * e + dt));
                            O[dt][e] += as_f32(x & seen & no_number(x));
                        }
                }
        };
        while (n > 0) {
            for (int i = 0; i < n; i += 2) {
                if (i + 1 < n) fetch(i + 1, B);
                step(i, A);
                if (i + 1 < n) {
                    if (i + 2 < n) fetch(i + 2, A);
                    step(i + 1, B);
                }
            }
            sub += SUB;
            if (sub >= c1) break;
            rows = lookup(sub);
            n = steps();
            if (n > 0) fetch(0, A);
        }
        // Join the waves: lane (r16, q) of each has dims 32 q + 8 i + dt of row r16.  They go through LDS, [wave][dt]
        // [q][r16][i], the rows of q padded by four so that the lanes that read it meet no bank twice.
        l = sum_x4(l);
        __syncthreads();  // the sequence before is read
        if (q == 0) sml[wave * 16 + r16] = make_float2(m, l);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) so[(wave * 8 + dt) * ROWS_PITCH + q * 20 + r16] = O[dt];
        __syncthreads();
        // A thread writes DIMS values of a row.
        constexpr int DIMS = 8 * 4 / NW;
        const int at = threadIdx.x * DIMS, d0 = at % HD, orow = at / HD;
        const RowOf out = row_of(sp, orow, group, g);
        if (out.t >= 0 && (whole || orow < a.few.rows)) {
            float mt = NEG_INF, lt = 0.f;
            float2 ml[NW];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                ml[w] = sml[w * 16 + orow];
                mt = fmaxf(mt, ml[w].x);
            }
            float x[DIMS] = {};
            const float* src = (const float*)so + (d0 % 8) * ROWS_PITCH * 4 + (d0 / 32) * 80 + orow * 4 + d0 / 8 % 4;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = ml[w].x == mt ? 1.f : __builtin_amdgcn_exp2f(ml[w].x - mt);
                lt += ml[w].y * f;
#pragma unroll
                for (int k = 0; k < DIMS; ++k) x[k] += src[(w * 8 + k) * ROWS_PITCH * 4] * f;
            }
            const bool partial = !whole || joined;
            const float inv = partial ? 1.f : mt == NEG_INF && lt == 0.f ? 0.f : 1.f / lt;  // no slot seen: zeros
            int64_t part = ((int64_t)index * 2 + (first == 0)) * a.few.rows + orow;
            if (joined && whole) {
                part = a.part_at + ((int64_t)out.t * a.n_heads + out.head) * a.big.n;
            }
#pragma unroll
            for (int k = 0; k < DIMS; k += 4) {
                const f32x4 y = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]} * inv;
                if (partial)
                    *(f32x4*)(a.few_part + part * HD + d0 + k) = y;
                else
                    store4<TYPE>(a.out, (int64_t)out.t * a.out_stride + out.head * HD + d0 + k, y);
            }
            if (partial && d0 == 0) a.few_ml[part] = make_float2(mt, lt);
        }
    }
}

template <int FORM, int TYPE, int FMT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_rows_kernel(PagedAttnArgs a) {
    __shared__ __align__(16) uint8_t lds[rows_lds<4>(FORM)];
    rows_work<FORM, TYPE, FMT, 4>(a, blockIdx.x, lds);
}
// Eight waves a workgroup, for whole sequences.
template <int FORM, int TYPE, int FMT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_rows8_kernel(PagedAttnArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    rows_work<FORM, TYPE, FMT, 8>(a, blockIdx.x, lds);
}

// Sequences with more query rows: 128 rows of a (sequence, KV head) a workgroup, eight waves.  Wave w has
// rows 32 (w & 3) .. + 31 and of each 128 slots the half w >> 2; the two halves keep softmax states of their
// own, joined through LDS at the end.  (Windows over fp16 slots: four waves and 64 slots, two workgroups a CU, so
// that one's first loads and last stores are under the other's products: a prompt of 4096 tokens through a window of
// 512 and 16 first slots 38 us, where eight waves take 45, with fp32 queries 54 and 65.  q8 has registers for eight
// only, 156 us of a batch that took 100; one group's prefix beside 64 tokens 35 us for 32.)
//
// v_mfma_f32_32x32x16_f16, transposed as above: 32 query rows as columns, lane (column, h) has slots
// 8 b + 4 h + 0 .. 3 of a 32-slot block, b = 0 .. 3; V^T operands come from row-major V by transposing LDS reads.
//
// K and V are staged in LDS, two stages of 128 slots, by copies that run under the products: fp16 from memory
// to LDS directly; q8 through registers, as the exact codes in fp16, whose scales go to the groups' sums in fp32
// and to the probabilities.  (Dequantised K, rounded to fp16, doubles the error of a batch of prompts, 4.8e-4
// for 2.9e-4; it took 107 us where this took 138, both in their first calls.)
//
// A staged row is 16 chunks of 16 bytes, chunk c at place c ^ swizzle(row): the operand reads of K (16 rows
// at one chunk) and of V (4 rows at four chunks) then spread over all banks.  With only the low three bits
// of the place changed they met in half of them, and the reads took twice as long.
//
// Bound by the issue of instructions: for 128 slots a SIMD's two waves issue 470 vector instructions (64 of them
// exponentials, 64 products of 32 cycles), 200 scalar ones and 100 of LDS, in some 4300 cycles; products fill 38 %
// of them, vector instructions 41 %, LDS 20 %.  Wave priorities and a start of half the waves apart change nothing.
// A workgroup's first K and V are there 5 us after it starts, and 3 us join and write its rows.  A prompt of 4096
// tokens, 16 heads, fp16 queries: 87 us, 0.79 PFLOP/s of the causal half; q8 142 us.  With fp32 queries, twice the
// products (f16 pool) and also a split of each group's products (q8): 138 and 303 us; they spill 17 and 15 registers.
//
// q8, 12 sessions of chunks and single tokens, 121 us: vector instructions fill 53 % of the SIMDs' cycles, LDS 41 %
// of the CUs' (an eighth of that conflicts), products 19 %.
constexpr int CH_ROWS = 128, CH_HALF = 64;
constexpr int CH_MAT = CH_HALF * HD * 2;        // bytes of a half's K or V
constexpr int CH_SCALES = 8 * CH_HALF * 2;      // q8: a half's scales [K, V][group][slot]
// And for the eight tiles of two stages whether V has values that are no numbers, whether the page exists, and
// (q8, fp16 queries) the power of two that V's scales are below.
constexpr int ch_flags(int halves) { return 2 * halves * (2 * CH_MAT + CH_SCALES); }
constexpr int ch_lds(int halves) { return ch_flags(halves) + 192; }
// Halves of an iteration's slots, of four waves each.
constexpr int ch_halves(int form, int fmt) { return form == PAGED_WINDOW && fmt == FMT_F16 ? 1 : 2; }

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

__device__ __constant__ const u32x4 g_zeros = {0, 0, 0, 0};  // what slots that are not there are copied from

__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }
__device__ __forceinline__ f32x16 mfma32(v8h a, v8h b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The sequence and tile (of `rows` query rows a KV head) that number `index` stands for, over the
// sequences with more than ROWS_TILE rows; false past the last one.  A wave looks at 64 sequences at a time,
// and takes those with the most slots first, so that the last workgroups to run are short.  Every workgroup
// looks through the sequences before its own, so a batch's time has a part that grows with their square:
// 9 tokens over 200 slots of each of 1024 sequences 0.65 ms, of 16384 (the most in a call) 49 ms.
template <int FORM>
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, const PrefixGroup& gr, int group, int rows, int index, int& s, int& tile, int& tiles, Span& span) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.n_seqs; s0 += WAVE) {
        const int count = min(WAVE, a.n_seqs - s0);
        const Span x = span_of<FORM>(a, gr, s0);
        const int n = x.sp.n_q * group > ROWS_TILE ? (x.sp.n_q * group + rows - 1) / rows : 0, slots = FORM == PAGED_PREFIX ? x.slots() : x.sp.n_kv;
        int sum = n;
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) sum += __shfl_xor(sum, o);
        sum = __builtin_amdgcn_readfirstlane(sum);
        if (index >= sum) {
            index -= sum;
            continue;
        }
        int begin = 0;  // tiles of the sequences that come before lane's
        for (int j = 0; j < count; ++j) {
            const int kv = __builtin_amdgcn_readlane(slots, j), add = __builtin_amdgcn_readlane(n, j);
            if (kv > slots || (kv == slots && j < lane)) begin += add;
        }
        const uint64_t mine = __ballot(index >= begin && index < begin + n);
        const int i = __ffsll((unsigned long long)mine) - 1;
        tile = index - __builtin_amdgcn_readlane(begin, i);
        tiles = __builtin_amdgcn_readlane(n, i);
        span.sp = {__builtin_amdgcn_readlane(x.sp.t0, i), __builtin_amdgcn_readlane(x.sp.n_q, i), __builtin_amdgcn_readlane(x.sp.n_kv, i)};
        span.gap = {__builtin_amdgcn_readlane(x.gap.from, i), __builtin_amdgcn_readlane(x.gap.skip, i)};
        s = s0 + i;
        return true;
    }
    return false;
}

// The sequence of s0 .. s1 - 1 through whose table the group's first n slots are read, where s0 has fewer (an idle place,
// a session that is still to get some of them): the first one with n slots, or of those with the most.
__device__ __forceinline__ int longest_sequence(const PagedAttnArgs& a, int s0, int s1, int n) {
    const int lane = threadIdx.x & 63;
    int at = s0, most = 0;
    for (int b = s0; b < s1 && most < n; b += WAVE) {
        const int len = b + lane < s1 ? min(a.kv_len[b + lane], n) : 0;
        int top = len;
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) top = max(top, __shfl_xor(top, o));
        if (top > most) {
            most = __builtin_amdgcn_readfirstlane(top);
            at = b + __ffsll((unsigned long long)__ballot(len == top)) - 1;
        }
    }
    return at;
}

// The same for the groups' tokens over their prefixes: sequences s0 .. s1 - 1, of which s has the table.
__device__ __forceinline__ bool find_prefix_tile(const PagedAttnArgs& a, const PrefixGroup& gr, int group, int index, int& s, int& s0, int& s1, int& tile, int& tiles, Span& span) {
    int t0 = 0, t1 = 0, slots = 0;
    if (gr.n) {
        t0 = min(max(a.q_start[gr.s0], 0), a.n_tokens);
        t1 = min(max(a.q_start[gr.s1], t0), a.n_tokens);
        slots = a.kv_len[gr.s0];
    }
    const int n = ((t1 - t0) * group + CH_ROWS - 1) / CH_ROWS;
    for (int g = 0; g < a.f.n_groups; ++g) {
        tiles = __builtin_amdgcn_readlane(n, g);
        if (index < tiles) {
            s0 = __builtin_amdgcn_readlane(gr.s0, g);
            s1 = __builtin_amdgcn_readlane(gr.s1, g);
            tile = index;
            span = {{__builtin_amdgcn_readlane(t0, g), __builtin_amdgcn_readlane(t1, g) - __builtin_amdgcn_readlane(t0, g), __builtin_amdgcn_readlane(gr.n, g)}, {0, 0}};
            s = __builtin_amdgcn_readlane(slots, g) >= span.sp.n_kv ? s0 : longest_sequence(a, s0, s1, span.sp.n_kv);
            return true;
        }
        index -= tiles;
    }
    return false;
}

template <int FORM, int TYPE, int FMT>
__global__ __launch_bounds__(256 * ch_halves(FORM, FMT)) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_chunk_kernel(PagedAttnArgs a) {
    constexpr int HALVES = ch_halves(FORM, FMT), STEP = HALVES * CH_HALF;
    constexpr bool HL = TYPE == TYPE_F32, CODES = FMT == FMT_Q8;
    extern __shared__ __align__(1024) uint8_t lds[];
    int* const tile_odd = (int*)(lds + ch_flags(HALVES));
    int *const tile_there = tile_odd + 16, *const tile_top = tile_odd + 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31, h = lane >> 5;
    const int par = HALVES == 1 ? 0 : wave >> 2, wi = wave & 3, group = a.n_heads / a.map.n_kv;
    // The first workgroups have the shared prefixes, the last ones the sequences of few rows: they are short, and
    // bound by memory.
    int index = blockIdx.x;
    bool pre = false;
    PagedSplit parts = a.big;
    if constexpr (FORM == PAGED_PREFIX) {
        pre = index < a.pre_tiles * a.map.n_kv * a.pre.n;
        if (pre)
            parts = a.pre;
        else
            index -= a.pre_tiles * a.map.n_kv * a.pre.n;
    }
    const int few = index - a.tiles * a.map.n_kv * a.big.n;
    if (!pre && few >= 0) {
        rows_work<FORM, TYPE, FMT, 4 * HALVES>(a, few, lds);
        return;
    }
    const int g = index % a.map.n_kv, at = index / a.map.n_kv, split = at % parts.n;
    const PrefixGroup gr = load_groups<FORM>(a);
    int s, tile, tiles, group_s0 = 0, group_s1 = 0;
    Span span;
    if (!(pre ? find_prefix_tile(a, gr, group, at / parts.n, s, group_s0, group_s1, tile, tiles, span) : find_tile<FORM>(a, gr, group, CH_ROWS, at / parts.n, s, tile, tiles, span))) return;
    tile = tiles - 1 - tile;  // those that see the most slots first
    const SeqSpan sp = span.sp;
    const int before = sp.n_kv - sp.n_q;  // token i sees slots up to before + i
    const int r0 = tile * CH_ROWS + 32 * wi;
    const bool active = r0 < sp.n_q * group;
    int w_first = before + r0 / group, w_last = before + min(sp.n_q - 1, (r0 + 31) / group);
    int all_seen = before + tile * CH_ROWS / group;  // slots up to this one all rows of the workgroup see
    int lim = max(0, before + min(sp.n_q - 1, (tile * CH_ROWS + CH_ROWS - 1) / group) + 1);
    RowOf row = row_of(sp, r0 + c32, group, g);
    // Iterations are of 64 slots a half, numbered without those that are skipped, 64 or a multiple of it: a half of an
    // iteration is a run of slots.  (Skipped 128 at a time, 16 first slots cost a window of 512 one iteration of 6.)
    SlotGap gap = {0, 0};
    bool joined = false;
    if constexpr (FORM == PAGED_WINDOW) gap = window_gap(all_seen, lim, a.f.window, a.f.sinks, CH_HALF);
    if constexpr (FORM == PAGED_PREFIX) {
        gap.skip = span.gap.skip;
        joined = pre || gap.skip > 0;
        if (pre) {
            lim = sp.n_kv;
            w_first = w_last = all_seen = lim - 1;
            row.last = lim - 1;
        }
    }
    auto slot_of = [&](int v) __attribute__((always_inline)) { return FORM == PAGED_ALL ? v : FORM == PAGED_PREFIX ? v + gap.skip : gap_slot(gap, v); };
    const int left = FORM == PAGED_ALL ? lim : max(0, lim - gap.skip);
    const int c0 = min(left, split * parts.chunk), c1 = min(left, c0 + parts.chunk);
    const int it0 = c0 / STEP, it1 = c1 > c0 ? (c1 + STEP - 1) / STEP : it0;
    // A window's rows see slots from first_own on, those of this wave from w_low .. w_high, and the first ones.
    const int first_own = row.last - a.f.window + 1, w_low = w_first - a.f.window + 1, w_high = w_last - a.f.window + 1;

    // Query operands: dims 16 ks + 8 h .. + 7 of the column's row.  Loaded first, then the first K and V are
    // asked for, and what both take is waited for once.
    u32x4 qrow[HL ? 16 : 8];
    {
        const int64_t qa = (int64_t)row.t * a.q_stride + row.head * HD + 8 * h;
#pragma unroll
        for (int k = 0; k < (HL ? 16 : 8); ++k)
            qrow[k] = row.t < 0 ? u32x4{} : HL ? *(const u32x4*)((const float*)a.q + qa + 16 * (k / 2) + 4 * (k % 2)) : *(const u32x4*)((const f16*)a.q + qa + 16 * k);
    }

    // What the loop seldom needs is read again from the arguments where it is needed, so that it takes no
    // registers in between.
    auto arguments = []() __attribute__((always_inline)) {
        auto p = (__attribute__((address_space(4))) const PagedAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return p;
    };
    // Staging: wave w copies 16-slot tile w of an iteration's.  Lane i of `rows`: the pool row of this
    // wave's tile in iteration sub + i (-1: no such page).
    int rows = -1, sub = it0 - WAVE;
    const int head_row = g * a.map.page_slots;
    auto tile_row = [&](int it) __attribute__((always_inline)) {
        if (it >= sub + WAVE) {
            auto b = arguments();
            const PageMap map = {b->map.n_pages, b->map.n_kv, b->map.page_slots};
            sub = it;
            const int slot = slot_of((sub + lane) * STEP + 16 * wave);
            rows = slot < (FORM == PAGED_ALL ? c1 : lim) ? seq_slot_row(map, b->tables + (int64_t)s * b->table_width, b->table_width, slot) : -1;
        }
        return __builtin_amdgcn_readlane(rows, it - sub);
    };
    const uint8_t *k_base = (const uint8_t*)a.k, *v_base = (const uint8_t*)a.v;
    // LDS: half hb of K (kv = 0) or V (1) in stage st, and the scales of a half.
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto half_at = [&](int kv, int st, int hb) { return (uint32_t)((kv * 2 + st) * HALVES + hb) * CH_MAT; };
    auto scales_at = [&](int st, int hb) { return (f16*)(lds + 4 * HALVES * CH_MAT + (st * HALVES + hb) * CH_SCALES); };
    // fp16: this wave's tile of iteration it, pool row r, from memory to LDS; slots that are not there become
    // zeros.  Row l / 16 (+ 4 j) of the tile, place l % 16.
    int src_off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) src_off[j] = (4 * j + lane / 16) * (HD * 2) + (((lane & 15) ^ swizzle(4 * j + lane / 16)) << 4);
    auto copy = [&](int kv, int it, int r) __attribute__((always_inline)) {
        const int n = r < 0 ? 0 : lim - slot_of(it * STEP + 16 * wave);
        const uint32_t dst = lds0 + half_at(kv, it & 1, par) + wi * 16 * HD * 2;
        const uint8_t* src = (kv ? v_base : k_base) + (int64_t)(max(r, 0) + head_row) * (HD * 2);
        if (!kv && lane == 0) tile_there[(it & 1) * 8 + wave] = r >= 0;
        if (n >= 16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) copy_to_lds(src, src_off[j], dst + j * 1024);
        } else {
            asm volatile("");
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* p = 4 * j + lane / 16 < n ? src + src_off[j] : (const uint8_t*)&g_zeros;
                copy_to_lds(p, dst + j * 1024);
            }
        }
    };
    // q8: a lane has a group of a row of the tile, fetched before the products and put to LDS after them.  Lane l of row
    // l % 16: the rows of 16 lanes meet no bank twice when they are put (12 sessions of chunks and single tokens 125 us,
    // 132 with lane l of row l / 4, whose loads are of fewer lines: prefixes, whose short ranges wait for them, 64 us of
    // drafts for 65).
    const int q_row = FORM == PAGED_PREFIX ? lane >> 2 : lane & 15, q_group = FORM == PAGED_PREFIX ? lane & 3 : lane >> 4;
    u32x4 codes[2][2];
    uint16_t scale[2] = {0, 0};
    auto fetch = [&](int kv, int it, int r) __attribute__((always_inline)) {
        const int n = r < 0 ? 0 : lim - slot_of(it * STEP + 16 * wave);
        if (!kv && lane == 0) tile_there[(it & 1) * 8 + wave] = r >= 0;
        codes[kv][0] = codes[kv][1] = u32x4{0, 0, 0, 0};
        scale[kv] = 0;
        if (q_row < n) {
            const int64_t at = (int64_t)r + head_row + q_row;
            const uint8_t* c = (kv ? v_base : k_base) + at * HD + 32 * q_group;
            codes[kv][0] = *(const u32x4*)c;
            codes[kv][1] = *(const u32x4*)(c + 16);
            scale[kv] = ((const uint16_t*)(kv ? a.v_sb : a.k_sb))[at * NG + q_group];
        }
    };
    auto put = [&](int kv, int it) __attribute__((always_inline)) {
        uint8_t* dst = lds + half_at(kv, it & 1, par);
        const int r = 16 * wi + q_row;
        // V with a scale that is no number is kept out of the products, for the rows that may not see it.
        const bool odd = kv && __ballot(!(fabsf(h2f(scale[1])) <= 65504.f));
        if (kv && lane == 0) tile_odd[(it & 1) * 8 + wave] = odd;
        if (kv && !(fabsf(h2f(scale[1])) <= 65504.f)) scale[1] = 0;
        f16 sc = __builtin_bit_cast(f16, scale[kv]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u32x4 w = codes[kv][k / 2];
            u32x4 y;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f16x2 c[2];
                codes_h2(w[2 * (k % 2) + x], c);
#pragma unroll
                for (int e = 0; e < 2; ++e) y[2 * x + e] = h2_bits(c[e]);
            }
            *(u32x4*)(dst + r * (HD * 2) + (((4 * q_group + k) ^ swizzle(r)) << 4)) = y;
        }
        if (kv && !HL) {  // the power of two that the largest scale is below; where less than 1, scales are raised by it
            int top = scale[1] & 0x7FFF;  // fp16 bits rise with the value
            top = max(top, __builtin_amdgcn_update_dpp(0, top, 0x124, 0xF, 0xF, true));  // row_ror:4, 8: within 16 lanes
            top = max(top, __builtin_amdgcn_update_dpp(0, top, 0x128, 0xF, 0xF, true));
            auto r16 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
            top = max((int)r16[0], (int)r16[1]);
            auto r32 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = max((int)r32[0], (int)r32[1]);
            top = max(top, __builtin_amdgcn_update_dpp(0, top, DPP_XOR1, 0xF, 0xF, true));
            top = max(top, __builtin_amdgcn_update_dpp(0, top, DPP_XOR2, 0xF, 0xF, true));
            top = (top >> 10) - 14;
            if (lane == 0) tile_top[(it & 1) * 8 + wave] = top;
            sc *= __builtin_bit_cast(f16, (uint16_t)((15 - min(top, 0)) << 10));
        }
        scales_at(it & 1, par)[kv * 4 * CH_HALF + q_group * CH_HALF + r] = sc;
    };

    auto stage = [&](int it) __attribute__((always_inline)) {
        const int r = tile_row(it);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            if constexpr (FMT == FMT_F16)
                copy(kv, it, r);
            else
                fetch(kv, it, r);
        }
    };
    auto staged = [&](int it) __attribute__((always_inline)) {
        if constexpr (FMT == FMT_Q8) {
            put(0, it);
            put(1, it);
        }
    };
    if (it0 < it1) stage(it0);
    // Scores are masked before they are scaled, so the scale is positive: a negative one's sign goes to
    // the query.
    v8h Qh[8], Ql[HL ? 8 : 1];
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    float qc = fabsf(a.scale) * 1.4426950408889634f;
    if constexpr (!HL) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) Qh[ks] = __builtin_bit_cast(v8h, qrow[ks]) * (f16)sign;
    } else {
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(as_f32(qrow[k][e])));
        amax = max_x2(amax);
        const int k2 = query_shift(amax);
        qc = ldexpf(qc, -k2);
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = sign * ldexpf(as_f32(qrow[k][e]), k2);
                const f16 hi = (f16)v;
                Qh[k / 2][4 * (k % 2) + e] = hi;
                Ql[k / 2][4 * (k % 2) + e] = (f16)(v - (float)hi);
            }
    }
    qc = fmaxf(qc, 1e-37f);  // and not zero: products are below 2^40, so this makes scores of 2^-80 at most

    // Whether the table has pages outside the pool.
    bool bad_pages = false;
    auto look_at_pages = [&](int c0, int c1) {
        const int32_t* table = a.tables + (int64_t)s * a.table_width;
        const int last_page = c1 > c0 ? (c1 - 1) / a.map.page_slots : -1;
        for (int p = c0 / a.map.page_slots; p <= last_page; p += WAVE)
            if (__ballot(p + lane <= last_page && page_row(a.map, table[min(p + lane, last_page)], 0) < 0)) bad_pages = true;
    };
    if constexpr (FORM == PAGED_ALL) {
        look_at_pages(c0, c1);
    } else {
        look_at_pages(c0, min(c1, gap.from));
        look_at_pages(max(c0, gap.from) + gap.skip, c1 + gap.skip);
    }
    if constexpr (FORM == PAGED_PREFIX)
        if (pre && !prefix_last(a, group_s0, group_s1, lim, row.t, row.last)) w_first = all_seen = __builtin_amdgcn_readfirstlane(-1);
    if (it0 < it1) staged(it0);

    f32x16 O[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) O[dt] = f32x16{};
    float m = NEG_INF, l = 0.f;
    auto base_of = [&](int it) __attribute__((always_inline)) { return slot_of(it * STEP + CH_HALF * par); };
    // LDS addresses of operands in stage 0.  K of block 0: slot c32, dims 16 ks + 8 h .. + 7, at k_at ^ (ks <<
    // 5).  V^T: dims 32 dt + c32 of slots 4 h + {0 .. 3} (k = 1: + 8, the operand's other half), at v_at[k] ^
    // (dt << 6).  (A row's place in a stage is a multiple of its 256 bytes.)
    const uint32_t k_at = lds0 + half_at(0, 0, par) + c32 * (HD * 2) + ((h ^ swizzle(c32)) << 4);
    uint32_t v_at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = 8 * k + 4 * h + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        v_at[k] = lds0 + half_at(1, 0, par) + r * (HD * 2) + ((chunk ^ swizzle(r)) << 4) + 8 * (lane & 1);
    }
    auto k_operand = [&](uint32_t block, int ks) __attribute__((always_inline)) {
        return *(__attribute__((address_space(3))) const v8h*)((k_at + block) ^ (ks << 5));
    };
    auto v_operand = [&](uint32_t block, int c, int dt) __attribute__((always_inline)) {
        v4s half[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            half[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(
                ((v_at[k] + block) ^ (dt << 6)) + c * 16 * HD * 2));
        return __builtin_bit_cast(v8h, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // Scores of a block are unscaled; element i: slot 8 (i / 4) + 4 h + i % 4.
    auto mask = [&](int it, int kt, f32x16& S) __attribute__((always_inline)) {
        const int base = base_of(it) + 32 * kt;
        const bool ends = FORM == PAGED_WINDOW && base + 31 >= a.f.sinks && base < w_high;  // before some row's window
        if (base + 31 <= w_first && !bad_pages && !ends) return;
        asm volatile("");  // keeps the branch: the selects are not made where they are not needed
        const int seen = row.last - base - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + i % 4 > seen) S[i] = NEG_INF;
        if (ends) {
            const int from = a.f.sinks - base - 4 * h, to = first_own - base - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((8 * (i / 4) + i % 4 >= from) & (8 * (i / 4) + i % 4 < to)) S[i] = NEG_INF;
        }
        if (bad_pages) {
            const int2 there = *(const int2*)(tile_there + (it & 1) * 8 + 4 * par + 2 * kt);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(i < 8 ? there.x : there.y)) S[i] = NEG_INF;
        }
    };
    auto block_max = [&](const f32x16& S) __attribute__((always_inline)) {
        float mb = NEG_INF;
#pragma unroll
        for (int i = 0; i < 16; ++i) mb = fmaxf(mb, S[i]);
        return mb;
    };
    // The maximum that is subtracted follows the true one when that is more than 2^P_SLACK ahead.  q8 with fp16
    // queries: the values' sums have a maximum of their own, m + mv, of scores plus the power of two e that V's
    // scales of their half are below.  mv is a whole number; m is not, so that the probability of the largest
    // score is a power of two and its products with scales are exact (2.9e-4 of error, 3.3e-4 with a whole m).
    constexpr bool WEIGHED = CODES && !HL;
    float mv = 0.f;
    auto follow_max = [&](float mb, float e) __attribute__((always_inline)) {
        mb = max_x2(mb) * qc;
        if constexpr (WEIGHED) {
            if (__builtin_amdgcn_ballot_w64(mb > m + P_SLACK || mb + e > m + mv + P_SLACK)) {
                asm volatile("");
                const float m_new = fmaxf(m, mb);
                // (2^-7: what rounding adds to a whole number does not make it the next.)
                const float mv_new = m_new == NEG_INF ? 0.f : __builtin_ceilf(fmaxf(m + mv, mb + e) - m_new - 0.0078125f);
                const float down = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                const float corr = m == NEG_INF ? 0.f : down * __builtin_amdgcn_exp2f(mv - mv_new);
                l *= down;
                m = m_new;
                mv = mv_new;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) O[dt] *= corr;
            }
        } else if (__builtin_amdgcn_ballot_w64(mb > m + P_SLACK)) {
            asm volatile("");
            const float m_new = fmaxf(m, mb);
            const float corr = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) O[dt] *= corr;
        }
    };
    // One half of an iteration: scores, their softmax, values, written in the order in which it is to be
    // issued.  Operands are read six (K) and eight (V) products ahead, the exponentials of 16 slots are among
    // the products of the 16 before; the denominator sums the probabilities as the products take them.
    auto half_step = [&](int it) __attribute__((always_inline)) {
        f32x16 S[2] = {f32x16{}, f32x16{}};
        const uint32_t st = (it & 1) * HALVES * CH_MAT;
        v8h kf[8];
#pragma unroll
        for (int k = 0; k < 6; ++k) kf[k] = k_operand(st + (k % 2) * 32 * HD * 2, k / 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (k + 6 < 16) kf[(k + 6) % 8] = k_operand(st + (k % 2) * 32 * HD * 2, (k + 6) / 2);
            S[k % 2] = mfma32(kf[k % 8], Qh[k / 2], S[k % 2]);
            if constexpr (HL) S[k % 2] = mfma32(kf[k % 8], Ql[k / 2], S[k % 2]);
            __builtin_amdgcn_sched_barrier(0);
        }
        mask(it, 0, S[0]);
        mask(it, 1, S[1]);
        v8h vf[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) vf[k] = v_operand(st, k / 4, k % 4);
        follow_max(fmaxf(block_max(S[0]), block_max(S[1])), 0.f);
        const float sub_m = m == NEG_INF ? 0.f : m - P_SHIFT;
        const f16x2 ones = {(f16)1.f, (f16)1.f};
        float sum[2] = {0.f, 0.f};
        v8h hi[4], lo[HL ? 4 : 1];
        auto exponentials = [&](int c) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[c / 2][8 * (c % 2) + e], qc, -sub_m));
                hi[c][e] = (f16)p;
                if constexpr (HL) lo[c][e] = (f16)(p - (float)hi[c][e]);
            }
        };
        exponentials(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int c = k / 4, dt = k % 4;
            if (dt == 0 && c < 3) exponentials(c + 1);
            O[dt] = mfma32(vf[k % 8], hi[c], O[dt]);
            if constexpr (HL) O[dt] = mfma32(vf[k % 8], lo[c], O[dt]);
            sum[dt % 2] = dot2(f16x2{hi[c][2 * dt], hi[c][2 * dt + 1]}, ones, sum[dt % 2]);
            if constexpr (HL) sum[dt % 2] = dot2(f16x2{lo[c][2 * dt], lo[c][2 * dt + 1]}, ones, sum[dt % 2]);
            if (k + 8 < 16) vf[k % 8] = v_operand(st, (k + 8) / 4, (k + 8) % 4);
            if (dt == 3) __builtin_amdgcn_sched_barrier(0);
        }
        l += sum[0] + sum[1];
    };
    // q8: codes are exact in fp16, and scales go to the sums of a group's products, in fp32, and to the
    // probabilities.  Block kt's sums of group gr take their slots' scales.
    auto scale_scores = [&](int it, int kt, int gr, const f32x16& y, f32x16& S) __attribute__((always_inline)) {
        const f16* scales = scales_at(it & 1, par) + gr * CH_HALF + 32 * kt + 4 * h;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const v4h sc = *(const v4h*)(scales + 8 * b);
#pragma unroll
            for (int e = 0; e < 4; ++e) S[4 * b + e] = __builtin_fmaf(y[4 * b + e], (float)sc[e], S[4 * b + e]);
        }
    };
    auto codes_scores = [&](int it, f32x16 S[2]) __attribute__((always_inline)) {
        const uint32_t st = (it & 1) * HALVES * CH_MAT;
        f32x16 y[2];
        S[0] = S[1] = f32x16{};
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                y[kt] = f32x16{};
#pragma unroll
                for (int ks = 2 * gr; ks < 2 * gr + 2; ++ks) {
                    const v8h kf = k_operand(st + kt * 32 * HD * 2, ks);
                    y[kt] = mfma32(kf, Qh[ks], y[kt]);
                    if constexpr (HL) y[kt] = mfma32(kf, Ql[ks], y[kt]);
                }
                // Under these products, those of the block before are scaled.
                if (2 * gr + kt) scale_scores(it, 1 - kt, gr - 1 + kt, y[1 - kt], S[1 - kt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        scale_scores(it, 1, NG - 1, y[1], S[1]);
    };
    // Values, fp16 queries.  A probability p, of 2^P_SHIFT at a score of m, becomes p 2^(e - mv) for the sums,
    // e <= 0 the power of two that its 16 slots' scales were raised by: so p and its products with scales are both
    // rounded where they have all of fp16's bits, whatever the size of V's values, and the products end below 2^15.
    // Next to a scale 2^d larger among the same 64 slots, seen or not, terms have steps of 2^(d - 33) of the
    // row's largest: d = 21 is where that shows (2e-3 of error instead of 1e-3 at most for a row).
    auto codes_values = [&](int it, const f32x16 S[2], const int4& tops) __attribute__((always_inline)) {
        const float sub_m = m == NEG_INF ? 0.f : m - P_SHIFT;
        const uint32_t st = (it & 1) * HALVES * CH_MAT;
        const f16* scales = scales_at(it & 1, par) + 4 * CH_HALF + 4 * h;
        const f16x2 ones = {(f16)1.f, (f16)1.f};
        float sum[2] = {0.f, 0.f};
        f16x2 p[2][4];
        auto exponentials = [&](int c) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                p[c % 2][e / 2][e % 2] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(S[c / 2][8 * (c % 2) + e], qc, -sub_m));
        };
        // 2^(e - mv): at most 2^14, as mv is -14 or more.
        auto factor = [&](int c) __attribute__((always_inline)) {
            const int e = c == 0 ? tops.x : c == 1 ? tops.y : c == 2 ? tops.z : tops.w;
            const f16 y = (f16)__builtin_amdgcn_exp2f((float)min(e, 0) - mv);
            return f16x2{y, y};
        };
        exponentials(0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const f16x2 g = factor(c);
            f16x2 pg[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) pg[k] = p[c % 2][k] * g;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                u32x4 ph;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x2 sc = *(const u32x2*)(scales + dt * CH_HALF + 16 * c + 8 * k);
#pragma unroll
                    for (int e = 0; e < 2; ++e) ph[2 * k + e] = h2_bits(pg[2 * k + e] * as_h2(sc[e]));
                }
                O[dt] = mfma32(v_operand(st, c, dt), __builtin_bit_cast(v8h, ph), O[dt]);
                sum[dt % 2] = dot2(p[c % 2][dt], ones, sum[dt % 2]);
                if (dt == 1 && c < 3) exponentials(c + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum[0] + sum[1];
    };
    // fp32 queries: a block's dims 32 dt .. + 31 are one group, whose scales go to the probabilities.  A row's
    // products of the two, by the power of two that puts the largest in [2^14, 2^15), are split into fp16 hi + lo
    // parts, and the power goes to the sum: values that the row does not see, or gives little weight, take nothing
    // from its accuracy, however large.  (By the power of the largest scale instead, a value of 65504 at a later
    // token left 4e-4 of error to rows of small values.)
    auto exact_values = [&](int it, int kt, const f32x16& S) __attribute__((always_inline)) {
        const float sub_m = m == NEG_INF ? 0.f : m - P_SHIFT;
        const uint32_t Vs = (it & 1) * HALVES * CH_MAT + kt * 32 * HD * 2;
        const f16* scales = scales_at(it & 1, par) + 4 * CH_HALF + 32 * kt + 4 * h;
        float p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], qc, -sub_m));
            l += p[i];
        }
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
            float x[16], top = 0.f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const v4h sc = *(const v4h*)(scales + dt * CH_HALF + 8 * b);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[4 * b + e] = p[4 * b + e] * (float)sc[e];
                    top = fmaxf(top, fabsf(x[4 * b + e]));
                }
            }
            const int e2 = max(__builtin_amdgcn_frexp_expf(max_x2(top)), -100) - 15;
            const float down = ldexpf(1.f, -e2), up = ldexpf(1.f, e2);
            f32x16 y = {};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                v8h ph, pl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float z = x[8 * c + e] * down;
                    // One value for both parts: else the compiler rounds the product itself to fp16 for one
                    // of them, which next to a tie is not its fp32 value rounded.
                    asm("" : "+v"(z));
                    ph[e] = (f16)z;
                    pl[e] = (f16)(z - (float)ph[e]);
                }
                const v8h v = v_operand(Vs, c, dt);
                y = mfma32(v, ph, y);
                y = mfma32(v, pl, y);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) O[dt][i] += up * y[i];
        }
    };
    // Whether some row of the workgroup does not see all of an iteration: of an f16 pool, all of its values are
    // made finite then, also for waves whose rows see them.
    auto cleaned = [&](int it) __attribute__((always_inline)) {
        if constexpr (FORM != PAGED_WINDOW) return slot_of(it * STEP) + STEP - 1 > all_seen;
        bool some = false;
        for (int half = 0; half < HALVES; ++half) {
            const int at = slot_of(it * STEP + CH_HALF * half);
            some |= (at + CH_HALF - 1 > all_seen) | ((at + CH_HALF > a.f.sinks) & (at <= lim - 1 - a.f.window));
        }
        return some;
    };
    // Values that are no numbers were kept out of the products: they go to the rows that see them.
    auto add_odd_values = [&](int it) __attribute__((always_inline)) {
        const int base = base_of(it);
        if (FMT == FMT_F16 && !cleaned(it)) return;
        const int4 odd = *(const int4*)(tile_odd + (it & 1) * 8 + 4 * par);
        if (!__builtin_amdgcn_readfirstlane(odd.x | odd.y | odd.z | odd.w)) return;
        auto b = arguments();
        const PageMap map = {b->map.n_pages, b->map.n_kv, b->map.page_slots};
        for (int j = 0; j < CH_HALF && base + j < lim; ++j) {
            const int r = seq_slot_row(map, b->tables + (int64_t)s * b->table_width, b->table_width, base + j);
            if (r < 0) continue;
            const bool own = FORM != PAGED_WINDOW || (base + j < a.f.sinks) | (base + j >= first_own);
            const uint32_t sees = (base + j <= row.last) & own ? 0xFFFFFFFFu : 0;
#pragma unroll
            for (int k = 0; k < 16; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = as_u32(row_value<FMT>(b->v, b->v_sb, (int64_t)r + head_row, 32 * (k / 4) + 8 * (k % 4) + 4 * h + e));
                    O[k / 4][4 * (k % 4) + e] += as_f32(x & sees & no_number(x));
                }
        }
    };
    // Slots that some rows of the workgroup see and others do not may hold values that are no numbers: in
    // iterations that have such slots each wave makes its tile of V finite.  (q8: when it is put to LDS.)
    auto clean_values = [&](int it) __attribute__((always_inline)) {
        if (!cleaned(it)) return;
        asm volatile("");
        uint32_t odd = 0;
        uint8_t* vt = lds + half_at(1, it & 1, par) + wi * 16 * HD * 2 + lane * 16;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v8h v = *(const v8h*)(vt + 1024 * k);
            keep_finite(v, odd);
            *(v8h*)(vt + 1024 * k) = v;
        }
        const bool any = __ballot(odd != 0) != 0;
        if (lane == 0) tile_odd[(it & 1) * 8 + wave] = any;
        staged_barrier<63>();
    };
    // Iterations whose half some row of this wave sees.
    const int v_last = FORM == PAGED_ALL || w_last < gap.from ? w_last : max(gap.from - 1, w_last - gap.skip);  // w_last's number
    const int my1 = active && base_of(it0) <= w_last ? min(it1, (v_last - CH_HALF * par) / STEP + 1) : it0;
    for (int it = it0; it < it1; ++it) {
        staged_barrier<0>();
        if (it + 1 < it1) stage(it + 1);
        if constexpr (FMT == FMT_F16) clean_values(it);
        if (it < my1 && (FORM != PAGED_WINDOW || base_of(it) < a.f.sinks || base_of(it) + CH_HALF > w_low)) {
            if constexpr (!CODES) {
                half_step(it);
            } else {
                f32x16 S[2];
                codes_scores(it, S);
                mask(it, 0, S[0]);
                mask(it, 1, S[1]);
                int4 tops = {0, 0, 0, 0};
                if constexpr (!HL) tops = *(const int4*)(tile_top + (it & 1) * 8 + 4 * par);
                follow_max(fmaxf(block_max(S[0]), block_max(S[1])), (float)max(max(tops.x, tops.y), max(tops.z, tops.w)));
                if constexpr (HL) {
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) exact_values(it, kt, S[kt]);
                } else {
                    codes_values(it, S, tops);
                }
            }
            add_odd_values(it);
        }
        if (it + 1 < it1) staged(it + 1);
    }

    if constexpr (WEIGHED) {  // the sums relative to m again
        const float f = __builtin_amdgcn_exp2f(mv);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) O[dt] *= f;
    }

    // The halves' states join: waves 4 .. 7 hand theirs to waves 0 .. 3.
    f32x4* const mo = (f32x4*)lds;                          // [4 waves][16][64 lanes]
    float2* const mml = (float2*)(lds + 4 * 16 * 64 * 16);  // [4 waves][64 lanes]
    l = swap32_add(l, l);
    float mt = m, lt = l, f0 = 1.f, f1 = 0.f;
    if constexpr (HALVES == 2) {
        staged_barrier<0>();
        if (par == 1) {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                mo[(wi * 16 + k) * 64 + lane] = f32x4{O[k / 4][4 * (k % 4)], O[k / 4][4 * (k % 4) + 1], O[k / 4][4 * (k % 4) + 2], O[k / 4][4 * (k % 4) + 3]};
            mml[wi * 64 + lane] = make_float2(m, l);
        }
        staged_barrier<0>();
        if (par == 1) return;
        const float2 ml = mml[wi * 64 + lane];
        mt = fmaxf(m, ml.x);
        f0 = m == mt ? 1.f : __builtin_amdgcn_exp2f(m - mt);
        f1 = ml.x == mt ? 1.f : __builtin_amdgcn_exp2f(ml.x - mt);
        lt = l * f0 + ml.y * f1;
    }
    if (row.t < 0) return;
    const bool partial = parts.n > 1 || joined;
    const float inv = partial ? 1.f : mt == NEG_INF && lt == 0.f ? 0.f : 1.f / lt;  // no slot seen: zeros
    const int64_t out_row = ((int64_t)row.t * a.n_heads + row.head) * parts.n + split;
    float* const part = FORM != PAGED_PREFIX ? a.part : a.few_part + (pre ? a.pre_at : a.part_at) * HD;
    float2* const part_ml = FORM != PAGED_PREFIX ? a.part_ml : a.few_ml + (pre ? a.pre_at : a.part_at);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = O[k / 4][4 * (k % 4) + e];
        if constexpr (HALVES == 2) {
            const f32x4 o1 = mo[(wi * 16 + k) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = y[e] * f0 + o1[e] * f1;
        }
        y *= inv;
        const int d = 32 * (k / 4) + 8 * (k % 4) + 4 * h;
        if (partial)
            *(f32x4*)(part + out_row * HD + d) = y;
        else
            store4<TYPE>(a.out, (int64_t)row.t * a.out_stride + row.head * HD + d, y);
    }
    if (partial && h == 0) part_ml[out_row] = make_float2(mt, lt);
}

// Joins the partials of a row, at part_at(0 .. n - 1): 32 lanes have a partial's 128 values, four each, so a
// wave reads two at a time, eight loads in flight; all of them are independent of the weights.
template <int TYPE, typename AT>
__device__ __forceinline__ void merge_row(const PagedAttnArgs& a, int t, int head, const float* part, const float2* part_ml, int n, AT part_at) {
    const int lane = threadIdx.x & 63, d = 4 * (lane & 31);
    float2 ml = make_float2(NEG_INF, 0.f);
    if (lane < n) ml = part_ml[part_at(lane)];
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float f = 0.f, m = 0.f, l = 0.f;
    for (int i0 = 0; i0 < n; i0 += 16) {
        f32x4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = *(const f32x4*)(part + part_at(min(i0 + 2 * k + (lane >> 5), n - 1)) * HD + d);
        if (i0 == 0) {
            m = wave_max(ml.x);
            f = ml.x == NEG_INF ? 0.f : ml.x == m ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
            l = wave_sum(ml.y * f);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + 2 * k + (lane >> 5);
            // 0 past the last; by all lanes, as an inactive one hands nothing over.  A partial without weight is added
            // too: one that is no number (of a slot of V that the row sees) makes the output none.
            o += x[k] * __shfl(f, i);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = swap32_add(o[e], o[e]);
    const float inv = m == NEG_INF && l == 0.f ? 0.f : 1.f / l;
    if (lane < 32) store4<TYPE>(a.out, (int64_t)t * a.out_stride + head * HD + d, o * inv);
}

// The workgroups of a KV head that share few-row sequence s: `n` of them from w0 on.
struct FewParts {
    int w0, n;
};
template <int FORM>
__device__ __forceinline__ FewParts few_parts(const PagedAttnArgs& a, const PrefixGroup& gr, int s) {
    const int group = a.n_heads / a.map.n_kv;
    int total = 0, begin = 0, n = 0;  // units of all sequences, those before s, its own
    for (int s0 = 0; s0 < a.n_seqs; s0 += WAVE) {
        const FewUnits u = few_units<FORM>(a, gr, group, s0);
        if (s >= s0 && s < s0 + WAVE) {
            n = __builtin_amdgcn_readlane(u.n, s - s0);
            begin = total + __builtin_amdgcn_readlane(u.end, s - s0) - n;
        }
        total += u.sum;
    }
    const int per = few_per(a, total), w0 = begin / per;
    return {w0, (begin + n - 1) / per - w0 + 1};
}
// Partial i of its row r, KV head g.
__device__ __forceinline__ int64_t few_at(const PagedAttnArgs& a, const FewParts& p, int g, int r, int i) {
    return (((int64_t)(p.w0 + i) * a.map.n_kv + g) * 2 + (i == 0)) * a.few.rows + r;
}

// Row r of a few-row sequence s and KV head g, if workgroups share the sequence.
template <int FORM, int TYPE>
__device__ __forceinline__ void merge_few(const PagedAttnArgs& a, int s, const SeqSpan& sp, int g, int r) {
    const int group = a.n_heads / a.map.n_kv;
    const FewParts p = few_parts<FORM>(a, PrefixGroup{}, s);
    if (p.n < 2 || r >= a.few.rows) return;
    merge_row<TYPE>(a, sp.t0 + r / group, g * group + r % group, a.few_part, a.few_ml, p.n, [&](int i) { return few_at(a, p, g, r, i); });
}

// Where only sequences of few rows are split: a workgroup has four of the at most 16 rows of a (sequence, KV
// head), a wave one.
template <int FORM, int TYPE>
__global__ __launch_bounds__(256) void paged_merge_rows_kernel(PagedAttnArgs a) {
    const int r = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = blockIdx.x / a.map.n_kv, g = blockIdx.x % a.map.n_kv;
    const SeqSpan sp = seq_span(a.q_start, a.kv_len, s, a.n_tokens, a.max_kv);
    const int rows = sp.n_q * (a.n_heads / a.map.n_kv);
    if (rows > ROWS_TILE || r >= rows) return;
    merge_few<FORM, TYPE>(a, s, sp, g, r);
}

// Row (t, head) of sequence s with prefixes: the partials of its group's, then its own.  Those of a few-row sequence
// that one workgroup has done are in its place in `part`.
template <int TYPE>
__device__ __forceinline__ void merge_prefix(const PagedAttnArgs& a, int t, int head, int s, const SeqSpan& sp) {
    const int lane = threadIdx.x & 63, group = a.n_heads / a.map.n_kv;
    const int64_t row = (int64_t)t * a.n_heads + head;
    const PrefixGroup gr = load_groups<PAGED_PREFIX>(a);
    const bool few = sp.n_q * group <= ROWS_TILE;
    const int pre = __ballot(gr.n > 0 && s >= gr.s0 && s < gr.s1) ? a.pre.n : 0;
    FewParts own = {0, a.big.n};
    if (few)
        own = few_parts<PAGED_PREFIX>(a, gr, s);
    else if (!a.tiles)
        return;  // more tokens than max_q
    if (!pre && own.n < 2) return;  // written already
    merge_row<TYPE>(a, t, head, a.few_part, a.few_ml, pre + own.n, [&](int i) {
        if (i < pre) return a.pre_at + row * a.pre.n + i;
        i -= pre;
        return few && own.n > 1 ? few_at(a, own, head / group, (t - sp.t0) * group + head % group, i) : a.part_at + row * a.big.n + i;
    });
}

// Else a wave a row, over all tokens; rows of no sequence stay as they are.
template <int FORM, int TYPE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int lane = threadIdx.x & 63, group = a.n_heads / a.map.n_kv;
    if (row >= (int64_t)a.n_tokens * a.n_heads) return;
    const int t = (int)(row / a.n_heads), head = (int)(row - (int64_t)t * a.n_heads);
    for (int s0 = 0; s0 < a.n_seqs; s0 += WAVE) {  // its sequence, looked for 64 at a time
        SeqSpan x = {0, 0, 0};
        if (s0 + lane < a.n_seqs) x = seq_span(a.q_start, a.kv_len, s0 + lane, a.n_tokens, a.max_kv);
        const uint64_t mine = __ballot(t >= x.t0 && t < x.t0 + x.n_q);
        if (!mine) continue;
        const int i = __ffsll((unsigned long long)mine) - 1;
        const SeqSpan sp = {__builtin_amdgcn_readlane(x.t0, i), __builtin_amdgcn_readlane(x.n_q, i), __builtin_amdgcn_readlane(x.n_kv, i)};
        if constexpr (FORM == PAGED_PREFIX)
            merge_prefix<TYPE>(a, t, head, s0 + i, sp);
        else if (sp.n_q * group <= ROWS_TILE)
            merge_few<FORM, TYPE>(a, s0 + i, sp, head / group, (t - sp.t0) * group + head % group);
        else
            merge_row<TYPE>(a, t, head, a.part, a.part_ml, a.big.n, [&](int k) { return row * a.big.n + k; });
        return;
    }
}

}  // namespace

hipError_t launch_paged_store(int fmt, int type, int q_type, const PagedStoreArgs& a, hipStream_t s) {
    const int64_t vecs = (int64_t)a.n_tokens * (a.n_heads + 2 * a.map.n_kv);
    const dim3 grid((unsigned)((vecs + 15) / 16));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    const int which = (fmt == FMT_Q8) * 4 + (type == TYPE_F16) * 2 + (q_type == TYPE_F16);
    switch (which) {
        case 0: go(paged_store_kernel<TYPE_F32, TYPE_F32, FMT_F16>); break;
        case 1: go(paged_store_kernel<TYPE_F32, TYPE_F16, FMT_F16>); break;
        case 2: go(paged_store_kernel<TYPE_F16, TYPE_F32, FMT_F16>); break;
        case 3: go(paged_store_kernel<TYPE_F16, TYPE_F16, FMT_F16>); break;
        case 4: go(paged_store_kernel<TYPE_F32, TYPE_F32, FMT_Q8>); break;
        case 5: go(paged_store_kernel<TYPE_F32, TYPE_F16, FMT_Q8>); break;
        case 6: go(paged_store_kernel<TYPE_F16, TYPE_F32, FMT_Q8>); break;
        case 7: go(paged_store_kernel<TYPE_F16, TYPE_F16, FMT_Q8>); break;
    }
    return hipGetLastError();
}

hipError_t launch_paged_load(int fmt, int type, const PagedLoadArgs& a, hipStream_t s) {
    const int64_t rows = (int64_t)a.n_rows * a.map.n_kv;
    const dim3 grid((unsigned)((rows + 15) / 16));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (fmt == FMT_Q8)
        type == TYPE_F32 ? go(paged_load_kernel<TYPE_F32, FMT_Q8>) : go(paged_load_kernel<TYPE_F16, FMT_Q8>);
    else
        type == TYPE_F32 ? go(paged_load_kernel<TYPE_F32, FMT_F16>) : go(paged_load_kernel<TYPE_F16, FMT_F16>);
    return hipGetLastError();
}

// Splits of max_kv slots among `per` workgroups of each (sequence, rows, KV head) that make up to `want`
// in all, each a multiple of 128 slots.
static PagedSplit split_slots(int64_t groups, int64_t want, int max_kv, int max_splits) {
    const int64_t most = std::max(1, (max_kv + 127) / 128);
    const int n = (int)std::min<int64_t>({std::max<int64_t>(1, want / std::max<int64_t>(1, groups)), most, max_splits});
    const int chunk = std::max(128, ((max_kv + n - 1) / n + 127) / 128 * 128);
    return {std::max(1, (max_kv + chunk - 1) / chunk), chunk};
}

// Units of few-row sequences among `want` workgroups: no sequence in more than max_splits of them.
//
// 512 workgroups are what the registers let run at once: 64 q8 sequences of up to 8192 slots take 110 us with 512,
// 143 with 256, 127 with 768 and 116 with 1024.  fp16 steps are twice a q8 step's bytes, and half as many workgroups
// read long caches faster: eight sequences of up to 32768 slots 121 us, 128 without the doubled shares.
static PagedFew few_of(int64_t want, int unit, int twice, int n_kv, int n_seqs, int rows, int max_kv, int max_splits) {
    const int most = std::max(1, (max_kv + unit - 1) / unit);
    const int n = (int)std::min(std::max<int64_t>(1, want / n_kv), (int64_t)n_seqs * most);
    return {n, unit, most < 2 ? 1 : (most - 2) / (max_splits - 1) + 1, twice, rows, 4, 0};
}

// The most tiles that sequences of more rows may have.
static int64_t big_tiles(int n_tokens, int group, int n_seqs) {
    return (int64_t)n_tokens * group / CH_ROWS + std::min<int64_t>(n_seqs, (int64_t)n_tokens * group / (ROWS_TILE + 1));
}

PagedPlan paged_plan(int fmt, int n_heads, int n_kv, int n_seqs, int n_tokens, int max_q, int max_kv, const PagedFormSizes& f) {
    PagedPlan p{};
    const bool prefix = f.form == PAGED_PREFIX;
    const int group = n_heads / n_kv, few = (int)std::min<int64_t>(ROWS_TILE, (int64_t)max_q * group);
    const int halves = ch_halves(f.form, fmt);  // of a workgroup of the chunk kernel: one, and two workgroups a CU, or two
    const int max_splits = prefix ? PAGED_MAX_SPLITS / 2 : PAGED_MAX_SPLITS;  // a row has partials of two spans
    if (f.form == PAGED_WINDOW) max_kv = window_slots(max_kv, f.window, f.sinks);
    p.big = {1, std::max(128, (max_kv + 127) / 128 * 128)};
    p.pre = {1, std::max(128, (f.max_prefix + 127) / 128 * 128)};
    const bool big = (int64_t)max_q * group > ROWS_TILE;
    int64_t shares = 256;  // workgroups that few-row sequences have beside prefixes
    if (prefix && n_tokens) {
        // As many tiles as there may be; one of a group at least, and about half of its last one is in use.
        const int64_t rows = (int64_t)n_tokens * group, groups = std::min<int64_t>(f.n_groups, rows);
        const int64_t tiles = std::max<int64_t>(groups, (rows + 63 * groups) / CH_ROWS), steps = (f.max_prefix + 127) / 128;
        p.pre_tiles = (int)((rows + 127 * groups) / CH_ROWS);
        // us of a tile's 128 slots, and of a sequence's 256; what sequences have of their own is six tenths of the most.
        const double step = fmt == FMT_F16 ? 2.5 : 5., unit = fmt == FMT_F16 ? 3. : 3.5;
        const int own = max_kv - f.max_prefix;
        const int64_t wgs = tiles * n_kv;
        double least = 1e30;
        int64_t ranges = 1;
        if (big) {
            // Beside chunks: the least of the CUs' time for all tiles, or of the longest workgroup, and of what a range more
            // costs to join.  (6 sessions, chunks of up to 300 tokens behind 1008 slots: 45 us with the two ranges that this
            // takes, 40 with one, 51 with the three that fill the CUs; 4 sessions, chunks of 60 behind 3200: 26 us with 8
            // ranges, 36 with 25.)
            const double rest = (double)big_tiles(n_tokens, group, n_seqs) * n_kv * (8. + 0.6 * own / 128 * step);
            const double join = 0.5 + (double)n_tokens * n_heads * (HD + 2) * 8 / 5e6;
            for (int64_t n = 1; n <= std::min<int64_t>(steps, max_splits); ++n) {
                const double longest = 8. + (steps + n - 1) / n * step, us = std::max(longest, (n * wgs * longest + rest) / 256) + n * join;
                if (us < least) least = us, ranges = n;
            }
        } else {
            // Beside few-row sequences: all workgroups at a time, one a CU, as many ranges of slots as end with the
            // sequences' shares.  64 tokens behind 7680 slots 29 us with 10 ranges and 176 shares, 32 with 384 shares in a
            // second round; 20 sequences of 8 tokens and fp32 queries, three prefixes, over q8 65 us with 6 ranges and 112
            // shares, 74 with 11 and 384.
            const int64_t units = (int64_t)(n_seqs * std::max(1., 0.6 * own / 256 + 0.5));
            for (int64_t n = 1; n <= std::min<int64_t>(steps, max_splits) && (n == 1 || n * wgs + n_kv <= 256); ++n) {
                const int64_t share = std::max<int64_t>(1, (256 - n * wgs % 256) / n_kv);
                const double us = 0.1 * n + std::max(8. + (steps + n - 1) / n * step, 6. + (units + share - 1) / share * unit);
                if (us < least) least = us, ranges = n, shares = share * n_kv;
            }
        }
        p.pre = split_slots(1, ranges, f.max_prefix, max_splits);
    }
    if (big) {
        p.tiles = (int)big_tiles(n_tokens, group, n_seqs);
        // (Windows that go through up to 512 slots, 258 and no first ones, are not split: 1024 tokens, windows of 128: 18
        // us, 27 in two parts, joined.)
        p.big = split_slots((int64_t)p.tiles * n_kv, 512 / halves, max_kv, f.form == PAGED_WINDOW && max_kv <= 512 ? 1 : max_splits);
    }
    // Windows are much of one length: where the (sequence, KV head) pairs fill 256 workgroups of eight waves, or whole
    // rounds of 512 of four, to four fifths, each has a workgroup of its own, and nothing is left to join.  (32 windows
    // of 1024 fp16 slots 36 us, q8 25, 64 of them 63; in even shares, joined: 42, 34 and 68.  40 windows, 52 us so or so,
    // and 96 short ones, 41 us and 44 in three rounds of 256, are in even shares.)
    const int64_t pairs = (int64_t)n_seqs * n_kv, rounds = (pairs + 511) / 512;
    const int waves = pairs <= 256 && 5 * pairs >= 4 * 256 ? 8 : 5 * pairs >= 4 * 512 * rounds ? 4 : 0;
    // Beside prompts windows that go through up to 1536 slots, 1282 and no first ones, are whole, too: 32 sessions, chunks
    // of 100 tokens and single ones, windows of 1000, 58 us for 63.  (Of 2048 over q8 they end last: 109 us for 101.)  Workgroup w has sequence w then, without a
    // search (1024 single tokens 100 us, searched for 379; 600 sessions, chunks and single tokens, 299 and 430), but in
    // smaller batches of both, where workgroups of chunks' numbers, which end at once, leave half the CUs idle (40
    // sessions over q8 46 us, 40 searched for; 150 as long).
    const bool whole = f.form == PAGED_WINDOW && (big ? max_kv <= 1536 : waves > 0);
    const int unit = 4 * halves * ROWS_STEP;  // slots of a step of a workgroup of the chunk kernel
    if (whole)
        p.few = {n_seqs, (max_kv + 8 * ROWS_STEP - 1) / (8 * ROWS_STEP) * (8 * ROWS_STEP), 1, INT32_MAX, few, big ? 4 : waves, !big || n_seqs > 128};
    else if (big || p.pre_tiles)
        p.few = few_of(big ? 512 / halves : shares, unit, INT32_MAX, n_kv, n_seqs, few, max_kv, max_splits);
    else
        p.few = few_of(512, 4 * ROWS_STEP, fmt == FMT_F16 ? 4 : INT32_MAX, n_kv, n_seqs, few, max_kv, max_splits);
    if (p.big.n > 1 || prefix) p.part_rows = (size_t)n_tokens * n_heads * p.big.n;
    if (prefix) p.pre_rows = (size_t)n_tokens * n_heads * p.pre.n;
    if (p.few.n > 1 && max_kv > p.few.unit) p.few_rows = (size_t)p.few.n * n_kv * 2 * few;
    return p;
}

template <int FORM, int TYPE, int FMT>
static hipError_t attention_of(const PagedAttnArgs& a, hipStream_t s) {
    const unsigned few = (unsigned)a.few.n * a.map.n_kv;
    hipError_t e;
    if (a.tiles || a.pre_tiles) {
        constexpr int halves = ch_halves(FORM, FMT), lds = std::max(ch_lds(halves), (int)rows_lds<4 * halves>(FORM));
        e = hipFuncSetAttribute((const void*)paged_chunk_kernel<FORM, TYPE, FMT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        const unsigned tiles = (unsigned)a.tiles * a.map.n_kv * a.big.n + (unsigned)a.pre_tiles * a.map.n_kv * a.pre.n;
        hipLaunchKernelGGL((paged_chunk_kernel<FORM, TYPE, FMT>), dim3(few + tiles), dim3(256 * halves), lds, s, a);
    } else if constexpr (FORM != PAGED_PREFIX) {  // (prefixes have tiles)
        if constexpr (FORM == PAGED_WINDOW)
            if (a.few.waves == 8) {
                e = hipFuncSetAttribute((const void*)paged_rows8_kernel<FORM, TYPE, FMT>, hipFuncAttributeMaxDynamicSharedMemorySize, rows_lds<8>(FORM));
                if (e != hipSuccess) return e;
                hipLaunchKernelGGL((paged_rows8_kernel<FORM, TYPE, FMT>), dim3(few), dim3(512), rows_lds<8>(FORM), s, a);
                return hipGetLastError();
            }
        hipLaunchKernelGGL((paged_rows_kernel<FORM, TYPE, FMT>), dim3(few), dim3(256), 0, s, a);
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.part)
        hipLaunchKernelGGL((paged_merge_kernel<FORM, TYPE>), dim3((unsigned)(((int64_t)a.n_tokens * a.n_heads + 3) / 4)), dim3(256), 0, s, a);
    else if (a.few_part)
        hipLaunchKernelGGL((paged_merge_rows_kernel<FORM, TYPE>), dim3((unsigned)a.n_seqs * a.map.n_kv, (unsigned)(a.few.rows + 3) / 4), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int FORM>
static hipError_t attention_form(int fmt, int type, const PagedAttnArgs& a, hipStream_t s) {
    if (fmt == FMT_Q8) return type == TYPE_F32 ? attention_of<FORM, TYPE_F32, FMT_Q8>(a, s) : attention_of<FORM, TYPE_F16, FMT_Q8>(a, s);
    return type == TYPE_F32 ? attention_of<FORM, TYPE_F32, FMT_F16>(a, s) : attention_of<FORM, TYPE_F16, FMT_F16>(a, s);
}

hipError_t launch_paged_attention(int fmt, int type, const PagedAttnArgs& a, hipStream_t s) {
    if (a.f.form == PAGED_WINDOW) return attention_form<PAGED_WINDOW>(fmt, type, a, s);
    if (a.f.form == PAGED_PREFIX) return attention_form<PAGED_PREFIX>(fmt, type, a, s);
    return attention_form<PAGED_ALL>(fmt, type, a, s);
}

}  // namespace icua
