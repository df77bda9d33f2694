// Operators on paged K/V caches, gfx950: store (per-head RMSNorm and rotation of new queries and keys,
// keys and values written to their slots as fp16 or q8), attention of every sequence's new tokens over
// its slots, load (slots read back).  A pool's K and V are row-major .icua matrices of 128 columns,
// rows [page][KV head][slot]: a (page, head)'s slots are contiguous, so a 16-slot tile is one run of
// 4 KiB (fp16) or 2 KiB of codes and 128 bytes of scales (q8).
#include <algorithm>

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
// the converter's quantiser (Convert.swift:215-241), so a stored row has the bytes that quantising
// the float32 row as a matrix gives.
__device__ __forceinline__ uint32_t q8_codes(f32x4 v, uint16_t& scale) {
#pragma clang fp contract(off)
    float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    amax = fmaxf(amax, dpp<DPP_XOR1>(amax));
    amax = fmaxf(amax, dpp<DPP_XOR2>(amax));
    amax = fmaxf(amax, dpp<DPP_HALF_MIRROR>(amax));
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
// and its queries, keys and values written once.
template <int TYPE, int QTYPE, int FMT>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedStoreArgs a) {
    const int nvec = a.n_heads + 2 * a.map.n_kv;
    const int64_t v = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (v >= (int64_t)a.n_tokens * nvec) return;
    const int t = (int)(v / nvec), vec = (int)(v - (int64_t)t * nvec), l = threadIdx.x % 16;
    const bool is_q = vec < a.n_heads, is_v = vec >= a.n_heads + a.map.n_kv;
    const int pos = a.pos ? a.pos[t] : 0;
    const bool pos_ok = !a.rot || (pos >= 0 && pos < a.rope_rows);
    const int row = is_q ? 0 : pool_slot_row(a.map, a.slots[t]);
    if (!is_q && (row < 0 || !pos_ok)) return;
    const int64_t at = (int64_t)t * a.qkv_stride + vec * HD;
    f32x4 x[2] = {load4<TYPE>(a.qkv, at + 4 * l), load4<TYPE>(a.qkv, at + 64 + 4 * l)};
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
// Read-back: 16 lanes a (row, KV head), 8 values a lane, K and V by one lane.
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
// operand takes its slots in that order.  Exponentials are taken of base-2 scores, shifted by 2^15 (of
// numerator and denominator alike): fp16 probabilities down to 2^-39 of the largest keep their value,
// where unshifted ones would round to nothing below 2^-24, which adds up over long caches.
//
// fp32 queries and probabilities are split into fp16 hi + lo parts, two products each; queries are
// first scaled by a power of two that puts the row's largest value in [2^9, 2^10), so that neither
// part leaves fp16's range.

constexpr float P_SHIFT = 15.0f;

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
template <int TYPE>
__device__ __forceinline__ Query<TYPE> load_query(const PagedAttnArgs& a, const RowOf& r, int q) {
    Query<TYPE> y;
    y.c = a.scale * 1.4426950408889634f;
    const int64_t at = (int64_t)r.t * a.q_stride + r.head * HD + 8 * q;
    if constexpr (TYPE == TYPE_F16) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) y.hi[ks] = r.t < 0 ? v8h{} : *(const v8h*)((const f16*)a.q + at + 32 * ks);
    } else {
        f32x4 x[8];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] = r.t < 0 ? f32x4{} : *(const f32x4*)((const float*)a.q + at + 32 * (k / 2) + 4 * (k % 2));
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(x[k][e]));
        }
        amax = max_x4(amax);
        const int k2 = amax > 0.f && amax < __builtin_inff() ? 10 - __builtin_amdgcn_frexp_expf(amax) : 0;
        y.c = ldexpf(y.c, -k2);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = ldexpf(x[k][e], k2);
                const f16 h = (f16)v;
                y.hi[k / 2][4 * (k % 2) + e] = h;
                y.lo[k / 2][4 * (k % 2) + e] = (f16)(v - (float)h);
            }
    }
    return y;
}

__device__ __forceinline__ f32x4 mfma(v8h a, v8h b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Two 16-slot tiles of K or V as a lane reads them from memory (K: slot r16, dims 32 ks + 8 q .. + 7;
// V: slots 4 q .. + 3, dims 8 r16 .. + 7), with a scale for each 8 values (q8).
template <int FMT>
struct KTile {
    u32x4 w[4];
};
template <>
struct KTile<FMT_Q8> {
    u32x2 w[4];
    u32x4 s[2];  // scales of slots 4 q .. + 3, four each
};
template <int FMT>
struct VTile {
    u32x4 w[4];
};
template <>
struct VTile<FMT_Q8> {
    u32x2 w[4];
    uint16_t s[4];
};

template <int FMT>
__device__ __forceinline__ void load_k(const PagedAttnArgs& a, int row, int lane, KTile<FMT>& t) {
    const int q = lane >> 4, r16 = lane & 15;
    if constexpr (FMT == FMT_F16) {
        const uint8_t* p = (const uint8_t*)a.k + (int64_t)row * (HD * 2) + r16 * (HD * 2) + q * 16;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) t.w[ks] = *(const u32x4*)(p + 64 * ks);
    } else {
        const uint8_t* p = (const uint8_t*)a.k + (int64_t)row * HD + r16 * HD + q * 8;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) t.w[ks] = *(const u32x2*)(p + 32 * ks);
        const uint8_t* s = (const uint8_t*)a.k_sb + (int64_t)row * (NG * 2) + q * 32;
        t.s[0] = *(const u32x4*)s;
        t.s[1] = *(const u32x4*)(s + 16);
    }
}
template <int FMT>
__device__ __forceinline__ void load_v(const PagedAttnArgs& a, int row, int lane, VTile<FMT>& t) {
    const int q = lane >> 4, r16 = lane & 15;
    if constexpr (FMT == FMT_F16) {
        const uint8_t* p = (const uint8_t*)a.v + (int64_t)row * (HD * 2) + q * 4 * (HD * 2) + r16 * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) t.w[j] = *(const u32x4*)(p + j * HD * 2);
    } else {
        const uint8_t* p = (const uint8_t*)a.v + (int64_t)row * HD + q * 4 * HD + r16 * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) t.w[j] = *(const u32x2*)(p + j * HD);
        const uint16_t* s = (const uint16_t*)a.v_sb + (int64_t)row * NG + q * 4 * NG + r16 / 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) t.s[j] = s[j * NG];
    }
}

// Eight int8 codes as exact fp16 values.
__device__ __forceinline__ v8h codes_f16(u32x2 c) {
    v8h y;
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = (f16)(float)(int8_t)(c[k / 4] >> (8 * (k % 4)));
    return y;
}

// Scores of a tile, products with the column's query: fp16 rows directly; q8 codes are exact in fp16
// and a 32-value group is one product's depth, so each group's sum takes its scale in fp32.
template <int TYPE, int FMT>
__device__ __forceinline__ f32x4 tile_scores(const KTile<FMT>& t, const Query<TYPE>& y) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        if constexpr (FMT == FMT_F16) {
            const v8h k = __builtin_bit_cast(v8h, t.w[ks]);
            s = mfma(k, y.hi[ks], s);
            if constexpr (TYPE == TYPE_F32) s = mfma(k, y.lo[ks], s);
        } else {
            const v8h k = codes_f16(t.w[ks]);
            f32x4 p = mfma(k, y.hi[ks], f32x4{0.f, 0.f, 0.f, 0.f});
            if constexpr (TYPE == TYPE_F32) p = mfma(k, y.lo[ks], p);
            // The scale of slot 4 q + i, group ks: half 4 i + ks of t.s.
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[i] += p[i] * h2f((uint16_t)(t.s[i / 2][2 * (i % 2) + ks / 2] >> (16 * (ks % 2))));
        }
    }
    return s;
}

// The V^T operands of two tiles: dims 8 r16 + dt over this lane's eight slots (4 q .. + 3 of each tile),
// hi and, for q8 with fp32 queries, lo parts of the exact products code x scale.
template <int TYPE, int FMT>
struct VOps {
    static constexpr bool LO = FMT == FMT_Q8 && TYPE == TYPE_F32;
    v8h hi[8], lo[LO ? 8 : 1];
};
template <int TYPE, int FMT>
__device__ __forceinline__ void v_operands(const VTile<FMT>* t, VOps<TYPE, FMT>& o) {
    if constexpr (FMT == FMT_F16) {
        // Word w of output dim 2 w (+ 1): the low (high) halves of word w of two rows, one byte select.
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            u32x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = __builtin_amdgcn_perm(t[j / 2].w[2 * (j % 2) + 1][dt / 2], t[j / 2].w[2 * (j % 2)][dt / 2],
                                             dt % 2 ? 0x07060302u : 0x05040100u);
            o.hi[dt] = __builtin_bit_cast(v8h, y);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float s = h2f(t[j / 4].s[j % 4]);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                const float v = s * (float)(int8_t)(t[j / 4].w[j % 4][dt / 4] >> (8 * (dt % 4)));
                o.hi[dt][j] = (f16)v;
                if constexpr (VOps<TYPE, FMT>::LO) o.lo[dt][j] = (f16)(v - (float)o.hi[dt][j]);
            }
        }
    }
}

template <int TYPE, int FMT>
__device__ __forceinline__ f32x4 pv(const VOps<TYPE, FMT>& v, int dt, v8h ph, v8h pl, f32x4 c) {
    c = mfma(v.hi[dt], ph, c);
    if constexpr (TYPE == TYPE_F32) c = mfma(v.hi[dt], pl, c);
    if constexpr (VOps<TYPE, FMT>::LO) c = mfma(v.lo[dt], ph, c);
    return c;
}

// Query rows in tiles of 16: a workgroup has one tile of a (sequence, KV head) and a range of its
// slots, its four waves take 32-slot steps of it in turn and join through LDS.  K and V go from memory to
// registers: each is used by one tile alone.  Bound by memory for single tokens and drafts.
constexpr int ROWS_STEP = 32, ROWS_SUB = WAVE * PAGED_TILE;

template <int TYPE, int FMT>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedAttnArgs a) {
    __shared__ f32x4 so[4][8][WAVE];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, r16 = lane & 15;
    const int g = blockIdx.y, split = blockIdx.z, group = a.n_heads / a.map.n_kv;
    // The sequence and tile of this workgroup: a sequence has ceil(n_q group / 16) tiles.
    int s = 0, tile = blockIdx.x;
    if (a.one_tile) {
        s = tile;
        tile = 0;
    } else {
        for (;; s += WAVE) {
            if (s >= a.n_seqs) return;
            int n = 0;
            if (s + lane < a.n_seqs)
                n = (seq_span(a.q_start, a.kv_len, s + lane, a.n_tokens, a.max_kv).n_q * group + 15) / 16;
            int end = n;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const int x = __shfl_up(end, o);
                if (lane >= o) end += x;
            }
            const uint64_t past = __ballot(end > tile);
            if (past) {
                const int first = __ffsll((unsigned long long)past) - 1;
                tile -= __shfl(end - n, first);
                s += first;
                break;
            }
            tile -= __shfl(end, 63);
        }
    }
    const SeqSpan sp = seq_span(a.q_start, a.kv_len, s, a.n_tokens, a.max_kv);
    if (tile * 16 >= sp.n_q * group) return;
    const RowOf row = row_of(sp, tile * 16 + r16, group, g);
    // Slots that some row of the tile sees: 0 .. lim - 1; all of them see those up to `all`.
    const int i0 = tile * 16 / group, i1 = min(sp.n_q - 1, (tile * 16 + 15) / group);
    const int lim = max(0, sp.n_kv - sp.n_q + i1 + 1), all = sp.n_kv - sp.n_q + i0;
    const int c0 = min(lim, split * a.chunk), c1 = min(lim, c0 + a.chunk);

    const Query<TYPE> y = load_query<TYPE>(a, row, q);
    f32x4 O[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;
    const int32_t* table = a.tables + (int64_t)s * a.table_width;
    for (int sub = c0; sub < c1; sub += ROWS_SUB) {
        // Lane i: the pool row of the range's tile i (-1: beyond the range, or no such page).
        int rows = -1;
        if (sub + lane * PAGED_TILE < c1) rows = seq_slot_row(a.map, table, a.table_width, sub + lane * PAGED_TILE);
        const int end = min(c1, sub + ROWS_SUB);
        for (int at = sub + wave * ROWS_STEP; at < end; at += 4 * ROWS_STEP) {
            KTile<FMT> kt[2];
            VTile<FMT> vt[2];
            int ok[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = __builtin_amdgcn_readlane(rows, (at - sub) / PAGED_TILE + t);
                ok[t] = r < 0 ? 0 : lim;  // slots from here on are not there
                const int base = max(r, 0) + g * a.map.page_slots;
                load_k<FMT>(a, base, lane, kt[t]);
                load_v<FMT>(a, base, lane, vt[t]);
            }
            float p[8], mb = NEG_INF;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 sc = tile_scores<TYPE, FMT>(kt[t], y);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = at + 16 * t + 4 * q + i;
                    p[4 * t + i] = slot > row.last || slot >= ok[t] ? NEG_INF : sc[i] * y.c;
                    mb = fmaxf(mb, p[4 * t + i]);
                }
            }
            mb = max_x4(mb);
            const float m_new = fmaxf(m, mb);
            const float corr = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
            const float base = m_new == NEG_INF ? 0.f : m_new - P_SHIFT;
            m = m_new;
            v8h ph, pl;
            l *= corr;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = __builtin_amdgcn_exp2f(p[i] - base);
                l += e;
                ph[i] = (f16)e;
                pl[i] = TYPE == TYPE_F32 ? (f16)(e - (float)ph[i]) : (f16)0.f;
            }
            // Values of slots that no row sees may be anything: they take no part.
            if (at + ROWS_STEP > min(ok[0], ok[1]))
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (at + 16 * t + 4 * q + j >= ok[t]) {
                            vt[t].w[j] = 0;
                            if constexpr (FMT == FMT_Q8) vt[t].s[j] = 0;
                        }
            VOps<TYPE, FMT> vo;
            v_operands<TYPE, FMT>(vt, vo);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) O[dt] *= corr;
            // Slots that some rows see and others do not: a value there that is no number must not
            // reach the rows that do not see it, so each such step is checked, and where one is found the
            // slots are added one by one to the rows that see them.
            bool plain = true;
            if (at + ROWS_STEP - 1 > all) {
                bool finite = true;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int j = 0; j < 8; ++j) finite &= __builtin_fabsf16(vo.hi[dt][j]) <= (f16)65504.f;
                plain = __ballot(!finite) == 0;
            }
            if (plain) {
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) O[dt] = pv<TYPE, FMT>(vo, dt, ph, pl, O[dt]);
            } else {
                for (int j = 0; j < ROWS_STEP; ++j) {
                    const bool sees = at + j <= row.last;
#pragma unroll
                    for (int dt = 0; dt < 8; ++dt) {
                        VOps<TYPE, FMT> one;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool mine = 16 * (e / 4) + 4 * q + e % 4 == j;
                            one.hi[dt][e] = mine ? vo.hi[dt][e] : (f16)0.f;
                            if constexpr (VOps<TYPE, FMT>::LO) one.lo[dt][e] = mine ? vo.lo[dt][e] : (f16)0.f;
                        }
                        const f32x4 c = pv<TYPE, FMT>(one, dt, ph, pl, O[dt]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) O[dt][i] = sees ? c[i] : O[dt][i];
                    }
                }
            }
        }
    }
    // Join the waves: lane (r16, q) of each has dims 8 (4 q + i) + dt of row r16.
    l = sum_x4(l);
    if (q == 0) {
        sm[wave][r16] = m;
        sl[wave][r16] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) so[wave][dt][lane] = O[dt];
    __syncthreads();
    float mt = NEG_INF, lt = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, sm[w][r16]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = sm[w][r16] == mt ? 1.f : __builtin_amdgcn_exp2f(sm[w][r16] - mt);
        lt += sl[w][r16] * f[w];
    }
    if (row.t < 0) return;
    // Wave w writes dims 8 (4 q + i) + 2 w, + 1.
    const float inv = a.nsplit > 1 ? 1.f : mt == NEG_INF && lt == 0.f ? 0.f : 1.f / lt;  // no slot seen: zeros
    const int64_t out_row = (int64_t)row.t * a.n_heads + row.head;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y2[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int w = 0; w < 4; ++w) y2[h] += so[w][2 * wave + h][lane][i] * f[w];
        const int d = 8 * (4 * q + i) + 2 * wave;
        if (a.nsplit > 1) {
            *(float2*)(a.part + (out_row * a.nsplit + split) * HD + d) = make_float2(y2[0], y2[1]);
        } else {
            const int64_t o = (int64_t)row.t * a.out_stride + row.head * HD + d;
            if constexpr (TYPE == TYPE_F32)
                *(float2*)((float*)a.out + o) = make_float2(y2[0] * inv, y2[1] * inv);
            else
                *(f16x2*)((f16*)a.out + o) = f16x2{(f16)(y2[0] * inv), (f16)(y2[1] * inv)};
        }
    }
    if (a.nsplit > 1 && wave == 0 && q == 0) a.part_ml[out_row * a.nsplit + split] = make_float2(mt, lt);
}

// Joins the splits of a row: one wave a row, two dims a lane.
template <int TYPE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)a.n_tokens * a.n_heads) return;
    const int t = (int)(row / a.n_heads), head = (int)(row - (int64_t)t * a.n_heads);
    // Rows of no sequence stay as they are.
    if (t < max(0, a.q_start[0]) || t >= a.q_start[a.n_seqs]) return;
    float2 ml = make_float2(NEG_INF, 0.f);
    if (lane < a.nsplit) ml = a.part_ml[row * a.nsplit + lane];
    const float m = wave_max(ml.x);
    const float f = ml.x == NEG_INF ? 0.f : ml.x == m ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
    const float l = wave_sum(ml.y * f);
    float2 o = make_float2(0.f, 0.f);
    for (int i = 0; i < a.nsplit; ++i) {
        const float w = as_f32(__builtin_amdgcn_readlane(as_u32(f), i));
        if (w == 0.f) continue;
        const float2 p = *(const float2*)(a.part + (row * a.nsplit + i) * HD + 2 * lane);
        o.x += w * p.x;
        o.y += w * p.y;
    }
    const float inv = m == NEG_INF && l == 0.f ? 0.f : 1.f / l;
    const int64_t at = (int64_t)t * a.out_stride + head * HD + 2 * lane;
    if constexpr (TYPE == TYPE_F32)
        *(float2*)((float*)a.out + at) = make_float2(o.x * inv, o.y * inv);
    else
        *(f16x2*)((f16*)a.out + at) = f16x2{(f16)(o.x * inv), (f16)(o.y * inv)};
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

PagedPlan paged_plan(int n_heads, int n_kv, int n_seqs, int n_tokens, int max_q, int max_kv) {
    PagedPlan p{};
    const int group = n_heads / n_kv;
    p.one_tile = (int64_t)max_q * group <= 16;
    const int64_t tiles = p.one_tile ? n_seqs : (int64_t)n_tokens * group / 16 + n_seqs;
    p.tiles = (int)std::min<int64_t>(tiles, 1 << 30);
    // Slots are split among workgroups until there are four of them for each of the 256 CUs.
    const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, tiles * n_kv));
    const int most = std::max(1, (max_kv + 127) / 128);  // at least a step for each wave
    p.nsplit = (int)std::min<int64_t>({want, most, PAGED_MAX_SPLITS});
    p.chunk = ((max_kv + p.nsplit - 1) / p.nsplit + 127) / 128 * 128;
    p.nsplit = std::max(1, (max_kv + p.chunk - 1) / std::max(1, p.chunk));
    if (p.nsplit > 1) {
        p.part_floats = (size_t)n_tokens * n_heads * p.nsplit * HD;
        p.ml_floats = (size_t)n_tokens * n_heads * p.nsplit * 2;
    }
    return p;
}

hipError_t launch_paged_attention(int fmt, int type, const PagedAttnArgs& a, hipStream_t s) {
    const dim3 grid(a.tiles, a.map.n_kv, a.nsplit);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (fmt == FMT_Q8)
        type == TYPE_F32 ? go(paged_rows_kernel<TYPE_F32, FMT_Q8>) : go(paged_rows_kernel<TYPE_F16, FMT_Q8>);
    else
        type == TYPE_F32 ? go(paged_rows_kernel<TYPE_F32, FMT_F16>) : go(paged_rows_kernel<TYPE_F16, FMT_F16>);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    const dim3 mgrid((unsigned)(((int64_t)a.n_tokens * a.n_heads + 3) / 4));
    if (type == TYPE_F32)
        hipLaunchKernelGGL(paged_merge_kernel<TYPE_F32>, mgrid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(paged_merge_kernel<TYPE_F16>, mgrid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace icua
