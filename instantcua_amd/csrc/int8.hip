// Products on 8-bit integers with a scale for each token and each output channel, gfx950: the tokens' rows are
// (normalised and) quantised, multiplied by a matrix of codes on the int8 matrix cores, and scaled into rows of y.
#include <algorithm>

#include "icua_device.h"
#include "icua_int8.h"
#include "icua_kernels.h"

namespace icua {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef f16 v8h __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------------------------------
// Quantisation of rows.  y = x norm / sqrt(mean(x^2) + eps), or x:  scale = max |y| / 127, code = y / scale rounded
// to the nearest, ties to even.  The root mean square is common to a row's values and leaves the codes as they are
// without it: code = 127 t / max |t| of t = x norm.  The maximum, its scale and the mean are of 64 bits, where t is
// exact.  A quotient t (127 / max) in fp32 is less than 3 2^-24 of its at most 127 off, 2.3e-5: it rounds as the exact
// one but within 4e-5 of half way between two codes (and in rows whose maximum is not near fp32's middle), where the
// 64-bit one decides, and within 2^-40 of it, where that may be off too, the exact sign of 254 t - (2 k + 1) max |t|:
// codes are those of the definition.  (Without a norm t has 24 bits, quotients that are no ties are 2^-25 from one, and a
// division tells them.)

// t 127 / top to the nearest, ties to even, for a quotient next to half way between two codes.  Values are products of
// two fp32 numbers, so that the difference of the two products below is a few steps of the last place of either.
__device__ __forceinline__ double code_next_to_tie(double t, double top, double q) {
#pragma clang fp contract(off)  // a and b are the rounded products
    const double below = floor(q), odd = 2. * below + 1.;
    const double a = 254. * t, b = odd * top;
    const double off = (a - b) + (fma(254., t, -a) - fma(odd, top, -b));
    return off > 0. ? below + 1. : off < 0. ? below : 2. * __builtin_rint(0.5 * below + 0.25);
}

// Eight values.
template <int TYPE>
__device__ __forceinline__ void load_x(const void* p, int64_t i, float* x) {
    if constexpr (TYPE == TYPE_F32) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const f32x4 v = *(const f32x4*)((const float*)p + i + 4 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = v[e];
        }
    } else {
        const v8h h = *(const v8h*)((const f16*)p + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
    }
}

// Over the lanes of a wave, every lane gets the result.
template <typename T, typename OP>
__device__ __forceinline__ T wave_reduce(T v, OP op) {
    auto other = [&](auto swap) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(T, swap(__builtin_bit_cast(int, v)));
        } else {
            const uint64_t b = __builtin_bit_cast(uint64_t, v);
            return __builtin_bit_cast(T, (uint64_t)(uint32_t)swap((int)(uint32_t)b) | (uint64_t)(uint32_t)swap((int)(uint32_t)(b >> 32)) << 32);
        }
    };
    v = op(v, other([](int x) { return dpp_i<DPP_MIRROR>(x); }));
    v = op(v, other([](int x) { return dpp_i<DPP_HALF_MIRROR>(x); }));
    v = op(v, other([](int x) { return dpp_i<DPP_XOR2>(x); }));
    v = op(v, other([](int x) { return dpp_i<DPP_XOR1>(x); }));
    v = op(v, other([](int x) { return __shfl_xor(x, 16); }));
    return op(v, other([](int x) { return __shfl_xor(x, 32); }));
}

constexpr int QUANT_ROWS = 1 << 20;  // of a launch's first dimension, which has fewer than 2^32 threads

// A workgroup a row; a thread has vectors of eight values 8 threadIdx.x + 2048 i, in registers where KEEP of them hold
// the row, else read a second time.  Bound by memory for many rows: 4096 of 6144 fp16 values, 76 MB, in 17 us, 4.5 TB/s
// (in 64 bits throughout 23), of 2048 fp32 ones 8 us, with a norm 10; by a chain of two loads and a reduction for few,
// 2.6 us.  4096 of 16384 fp16 values 45 us kept, 55 read twice; with a norm, which takes as many registers again, 8192
// fp32 ones 70 us kept and 46 read twice.
template <int TYPE, bool NORM, int KEEP>
__global__ __launch_bounds__(256) void i8_quantize_kernel(I8QuantArgs a) {
    __shared__ double s_top[4], s_sum[4];
    __shared__ int s_none[4];
    const int row = blockIdx.y * QUANT_ROWS + blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (row >= a.n_rows) return;
    const int64_t at = (int64_t)row * a.x_stride;
    constexpr int N = KEEP ? KEEP : 1;
    float x[N][8], w[NORM ? N : 1][8];
    auto load = [&](int k, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
        if constexpr (NORM)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[k][e] = 1.f;
        if (i >= a.n_cols) return;
        load_x<TYPE>(a.x, at + i, x[k]);
        if constexpr (NORM) load_x<TYPE_F32>(a.norm, i, w[k]);
    };
    uint32_t bits = 0;  // without a norm: the largest magnitude's bits, an infinity's or more if some y is none
    double top = 0., sum = 0., odd = 0.;  // odd: no number if some y is none
    auto look = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (NORM) {
                const double v = x[k][e], t = v * (double)w[k][e];
                top = fmax(top, fabs(t));
                sum = fma(v, v, sum);
                odd = fma(t, t, odd);
            } else {
                bits = max(bits, as_u32(x[k][e]) & 0x7FFFFFFFu);
            }
        }
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) load(k, 8 * threadIdx.x + 2048 * k);
#pragma unroll
        for (int k = 0; k < KEEP; ++k) look(k);
    } else {
        for (int i = 8 * threadIdx.x; i < a.n_cols; i += 2048) {
            load(0, i);
            look(0);
        }
    }
    bool none;
    if constexpr (NORM) {
        top = wave_reduce(top, [](double p, double q) { return fmax(p, q); });
        sum = wave_reduce(sum, [](double p, double q) { return p + q; });
        none = __ballot(!(odd < __builtin_inf())) != 0;
    } else {
        bits = wave_reduce(bits, [](uint32_t p, uint32_t q) { return max(p, q); });
        top = as_f32(bits);
        none = bits >= 0x7F800000u;
    }
    if (lane == 0) {
        s_top[wave] = top;
        s_sum[wave] = sum;
        s_none[wave] = none;
    }
    __syncthreads();
    top = fmax(fmax(s_top[0], s_top[1]), fmax(s_top[2], s_top[3]));
    none = (s_none[0] | s_none[1] | s_none[2] | s_none[3]) != 0;
    if (threadIdx.x == 0) {
        sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        const double r = NORM ? 1. / sqrt(sum / a.n_cols + (double)a.eps) : 1.;
        a.scales[row] = none ? __builtin_nanf("") : top == 0. ? 0.f : (float)(top * r / 127.);  // (r of zeros may be infinite)
    }
    const double to = none || top == 0. ? 0. : 127. / top;
    const bool middle = to == 0. || (top > 0x1p-60 && top < 0x1p60);  // no product of fp32 values leaves its range
    const float to32 = middle ? (float)to : 0.f;
    auto store = [&](int k, int i) __attribute__((always_inline)) {
        if (i >= a.n_cols) return;
        int code[8];
        float off = middle ? 0.f : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q = (none ? 0.f : NORM ? x[k][e] * w[k][e] : x[k][e]) * to32, r = __builtin_rintf(q);
            off = fmaxf(off, fabsf(q - r));
            code[e] = (int)r;
        }
        if (__builtin_expect(off > 0.49996f, 0)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double t = NORM ? (double)x[k][e] * (double)w[k][e] : (double)x[k][e], q = t * to;
                double r = __builtin_rint(q);
                if (__builtin_expect(fabs(q - r) > 0.5 - 0x1p-40, 0)) r = NORM ? code_next_to_tie(t, top, q) : __builtin_rint(t * 127. / top);
                code[e] = (int)r;
            }
        }
        uint2 word;
        word.x = (code[0] & 255) | (code[1] & 255) << 8 | (code[2] & 255) << 16 | (uint32_t)code[3] << 24;
        word.y = (code[4] & 255) | (code[5] & 255) << 8 | (code[6] & 255) << 16 | (uint32_t)code[7] << 24;
        *(uint2*)(a.codes + (int64_t)row * a.codes_stride + i) = word;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) store(k, 8 * threadIdx.x + 2048 * k);
    } else {
        for (int i = 8 * threadIdx.x; i < a.n_cols; i += 2048) {
            load(0, i);
            store(0, i);
        }
    }
}

template <int TYPE, bool NORM>
hipError_t quantize_of(const I8QuantArgs& a, hipStream_t s) {
    const dim3 grid(std::min(a.n_rows, QUANT_ROWS), (a.n_rows + QUANT_ROWS - 1) / QUANT_ROWS);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (a.n_cols <= 2048)
        go(i8_quantize_kernel<TYPE, NORM, 1>);
    else if (a.n_cols <= 6144)
        go(i8_quantize_kernel<TYPE, NORM, 3>);
    else if (!NORM && a.n_cols <= 16384)
        go(i8_quantize_kernel<TYPE, NORM, NORM ? 0 : 8>);
    else
        go(i8_quantize_kernel<TYPE, NORM, 0>);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------
// Products.  y[m][n] = x_scales[m] w_scales[n] sum_k x[m][k] w[n][k] (+ add[m][n]), the sums exact in 32-bit integers
// (|sum| <= 127^2 2^17 < 2^31); or, of two matrices, silu(gate) up.

__device__ __constant__ const u32x4 g_zero_codes = {0, 0, 0, 0};  // what lies behind a row's last code

// g / (1 + exp(-g)) u, by e = exp(-|g|) <= 1: g / (1 + e) u for g >= 0, e g / (1 + e) u else.  Up to |g| = GATE_NEAR
// e is a normal number of fp32 (the instructions make others zero), and so is what it is multiplied with: u comes last,
// whose product is below fp32's range where the result is.
constexpr float GATE_NEAR = 80.f;
__device__ __forceinline__ float gated_up(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(fabsf(g) * -1.4426950408889634f);
    const float s = __builtin_amdgcn_rcpf(1.f + e);
    return g * s * (g >= 0.f ? 1.f : e) * u;
}
// The same for gates of any size: e = x 2^n, and for g < 0 the power goes to the product in two parts, before u, where
// the product is below 1, and behind it.
__device__ __forceinline__ float gated_up_far(float g, float u) {
    const float n = fmaxf(__builtin_rintf(fabsf(g) * -1.4426950408889634f), -1000.f);
    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(fabsf(g), -1.4426950408889634f, -n));
    const int i = (int)n, half = i >> 1;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_ldexpf(x, i));
    if (!(g < 0.f)) return g * s * u;
    return __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(g * s * x, half) * u, i - half);
}

// A tile of BM tokens and BN matrix rows a workgroup, WM x WN of it a wave, on v_mfma_i32_32x32x32_i8 (twice the rate
// of the 16x16x64 one: 4.6 and 2.6 POPS of products of zeros, 3.5 and 2.2 of random codes, where the chip's power is
// the limit): tokens are the result's rows, channels its columns, so that a wave's stores are runs of 32 channels.
// Rows are staged in LDS 128 codes at a time, NS stages, by copies that run under the products; row r's 16-byte chunk
// c lies at place c ^ (r / 2 & 7), so that sixteen rows' reads of one chunk meet no bank twice.  KW groups of waves have the
// tile's 128 codes in turn, for few tiles, and join their sums through LDS.  Gated: half of a wave's matrix rows are
// gates, the other half the same channels' ups.
//
// The order of issue is written out: under each product one operand of the 32 codes ahead is read, and two of them in
// four carry the copies of a later stage (all in one of the four: 126 us where this took 111).  Large tiles, 8192^3 of
// random codes in 480 to 515 us, 2.1 to 2.3 POPS, are bound by their copies: on the same data 438 us without those of
// later stages, and no faster with half of either operand's reads.  256 x 256 x 128 codes are 64 KB of copies and 192 KB
// of reads; waves of 128 x 128, with 128 KB of reads, were no faster, nor were two groups of waves in turn, or 64 codes
// a stage in four.
template <int TYPE, bool GATED, int BM, int BN, int WM, int WN, int KW, int NS>
__global__ __launch_bounds__(BM / WM * (BN / WN) * KW * 64) void i8_matmul_kernel(I8MatmulArgs a, int tiles_m, int tiles_n) {
    constexpr int BK = 128, THREADS = BM / WM * (BN / WN) * 64, STAGE = (BM + BN) * BK, KS = BK / 32;
    constexpr int CX = BM * 8 / THREADS, CW = BN * 8 / THREADS, NI = WM / 32, NJ = WN / 32;
    constexpr int OUT = GATED ? BN / 2 : BN, WOUT = GATED ? WN / 2 : WN;  // channels of y of the tile, of a wave
    extern __shared__ __align__(1024) uint8_t lds[];
    float* const s_scale = (float*)(lds + KW * NS * STAGE);  // the tokens' scales
    const int part = KW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS), tid = threadIdx.x - part * THREADS;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + part * NS * STAGE;
    const int wm = wave % (BM / WM), wn = wave / (BM / WM), c32 = lane & 31, h = lane >> 5;
    // Consecutive workgroups go to the eight XCDs in turn: each XCD has a run of tiles, four of x by as many of the
    // matrix, whose rows its L2 holds for all of them.
    const int tile = (int)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    if (tile >= tiles_m * tiles_n) return;
    const int band = tile / (4 * tiles_n), bm = min(4, tiles_m - 4 * band), in_band = tile - band * 4 * tiles_n;
    const int m0 = (4 * band + in_band % bm) * BM, n0 = in_band / bm * OUT;
    // Copy i of a thread: 16 bytes of row (i * THREADS + tid) / 8 of the tile's x, or of its matrix rows.
    auto chunk = [&](int i) __attribute__((always_inline)) { return 16 * (tid % 8 ^ ((i < CX ? i : i - CX) * THREADS + tid) / 16 % 8); };
    const uint8_t *x0 = (const uint8_t*)a.x + m0 * a.x_stride, *w0 = (const uint8_t*)a.w + n0 * a.w_stride;
    uint32_t offset[CX + CW];
#pragma unroll
    for (int i = 0; i < CX + CW; ++i) {
        const int r = ((i < CX ? i : i - CX) * THREADS + tid) / 8, o = r / WN * WOUT + r % WN % WOUT;
        offset[i] = (uint32_t)(i < CX ? min(r, a.n_rows - 1 - m0) * (int)a.x_stride : min(o, a.n_out - 1 - n0) * (int)a.w_stride) + chunk(i);
    }
    const int64_t ups = GATED ? a.n_out * a.w_stride : 0;
    // Iteration it of this part of the waves is of codes first_k(it) .. + 127; `steps` are the workgroup's, this part's
    // last ones may be none.
    const int all_steps = (a.n_in + BK - 1) / BK, steps = (all_steps + KW - 1) / KW, mine = (all_steps - part + KW - 1) / KW;
    const int whole = a.n_in / BK < part ? 0 : (a.n_in / BK - part + KW - 1) / KW;
    auto first_k = [&](int it) __attribute__((always_inline)) { return (it * KW + part) * BK; };
    auto copy = [&](int it, int i) __attribute__((always_inline)) {
        const uint32_t dst = lds0 + it % NS * STAGE + wave * 1024 + (i < CX ? i : i - CX) * THREADS * 16;
        if (i < CX) {
            copy_to_lds(x0 + first_k(it), offset[i], dst);
        } else {
            const bool up = GATED && ((i - CX) * THREADS + wave * 64) / 8 % WN >= WOUT;  // the same for a wave's eight rows
            copy_to_lds(w0 + (up ? ups : 0) + first_k(it), offset[i], dst + BM * BK);
        }
    };
    // A stage that the last code lies in: zeros of x behind it, any of the matrix.
    auto copy_end = [&](int it) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CX + CW; ++i) {
            const bool there = first_k(it) + chunk(i) < a.n_in;
            const uint32_t dst = lds0 + it % NS * STAGE + wave * 1024 + (i < CX ? i : i - CX) * THREADS * 16;
            const bool up = GATED && i >= CX && ((i - CX) * THREADS + wave * 64) / 8 % WN >= WOUT;
            if (i < CX)
                copy_to_lds(there ? x0 + offset[i] + first_k(it) : (const uint8_t*)&g_zero_codes, dst);
            else
                copy_to_lds(w0 + (up ? ups : 0) + (there ? offset[i] + first_k(it) : offset[i] - chunk(i)), dst + BM * BK);
        }
    };
    auto stage = [&](int it) __attribute__((always_inline)) {
        if (it < whole) {
#pragma unroll
            for (int i = 0; i < CX + CW; ++i) copy(it, i);
        } else {
            copy_end(it);
        }
    };
    i32x16 acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = i32x16{};
#pragma unroll
    for (int it = 0; it < NS; ++it)
        if (it < mine) stage(it);
    // What the outputs take is asked for behind the first codes, and waited for with them.
    constexpr int NO = WOUT / 32, SIZE = TYPE == TYPE_F32 ? 4 : 2;
    const int first_m = m0 + wm * WM, first_n = n0 + wn * WOUT;
    static_assert(BM <= THREADS * KW);
    float x_scale = 0.f, sw[NO], su[NO];
    if ((int)threadIdx.x < BM) x_scale = a.x_scales[min(m0 + (int)threadIdx.x, a.n_rows - 1)];
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        const int n = min(first_n + 32 * j + c32, a.n_out - 1);
        sw[j] = a.w_scales[n];
        su[j] = GATED ? a.w_scales[a.n_out + n] : 0.f;
    }
    staged_barrier<0>();
    constexpr int HALF = (CX + CW + 1) / 2;  // of a stage's copies: with these products, the rest with the next ones
    i32x4 x[2][NI], w[2][NJ];
    const uint32_t x_at = lds0 + (wm * WM + c32) * BK, w_at = lds0 + (BM + wn * WN + c32) * BK;
    // Operand k of the codes 32 ks .. + 31 of the stage at `at`.
    auto read = [&](int at, int ks, int k) __attribute__((always_inline)) {
        const uint32_t c = ((2 * ks + h) ^ (c32 >> 1 & 7)) << 4;
        if (k < NI)
            x[ks & 1][k] = *(__attribute__((address_space(3))) const i32x4*)(x_at + at + c + 32 * BK * k);
        else
            w[ks & 1][k - NI] = *(__attribute__((address_space(3))) const i32x4*)(w_at + at + c + 32 * BK * (k - NI));
    };
    // The products of 32 codes; under them the next ones' operands and (`more`) a later stage are asked for.
    auto products = [&](int ks, int next, int at, int it, bool more) __attribute__((always_inline)) {
        constexpr int C = (HALF + NI * NJ - 1) / (NI * NJ), R = (NI + NJ + NI * NJ - 1) / (NI * NJ);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < NI * NJ; ++k) {
            acc[k / NJ][k % NJ] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[ks & 1][k / NJ], w[ks & 1][k % NJ], acc[k / NJ][k % NJ], 0, 0, 0);
#pragma unroll
            for (int i = R * k; i < R * k + R && i < NI + NJ; ++i) read(at, next, i);
            if (ks == KS - 1 && more)
#pragma unroll
                for (int i = C * k; i < C * k + C && i < HALF; ++i) copy(it, i);
            if (ks == 0 && more)
#pragma unroll
                for (int i = HALF + C * k; i < HALF + C * k + C && i < CX + CW; ++i) copy(it, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int k = 0; k < NI + NJ; ++k) read(0, 0, k);
#pragma unroll 1
    for (int it = 0; it < steps; ++it) {
        if (KW > 1 && it >= mine) {
            staged_barrier<0>();
            break;
        }
        const int at = it % NS * STAGE, next = (it + 1) % NS * STAGE;
#pragma unroll
        for (int ks = 0; ks < KS - 1; ++ks) products(ks, ks + 1, at, it - 1 + NS, ks == 0 && it > 0 && it - 1 + NS < whole);
        // All of this stage has been read, the next one is there.
        if (it + NS <= mine)
            staged_barrier<(NS - 2) * (CX + CW)>();
        else
            staged_barrier<0>();
        if (it + NS == whole && whole < mine) copy_end(it + NS);
        products(KS - 1, 0, next, it + NS, it + NS < whole);
    }
    if ((int)threadIdx.x < BM) s_scale[threadIdx.x] = x_scale;
    staged_barrier<0>();
    if constexpr (KW > 1) {  // the first part adds the others' sums to its own
        constexpr int PLACE = NI * NJ * 16 * 64 * 4;  // bytes of a wave's
        constexpr int WAVES = THREADS / 64;
        if (part > 0) {
            i32x4* const to = (i32x4*)(lds + ((part - 1) * WAVES + wave) * PLACE);
#pragma unroll
            for (int i = 0; i < NI * NJ * 4; ++i) {
                const i32x16& v = acc[i / 4 / NJ][i / 4 % NJ];
                to[i * 64 + lane] = i32x4{v[i % 4 * 4], v[i % 4 * 4 + 1], v[i % 4 * 4 + 2], v[i % 4 * 4 + 3]};
            }
        }
        staged_barrier<0>();
        if (part > 0) return;
#pragma unroll
        for (int p = 0; p < KW - 1; ++p)
#pragma unroll
            for (int i = 0; i < NI * NJ * 4; ++i) {
                const i32x4 v = ((const i32x4*)(lds + (p * WAVES + wave) * PLACE))[i * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i / 4 / NJ][i / 4 % NJ][i % 4 * 4 + e] += v[e];
            }
    }
    // Element e of a block: token 8 (e / 4) + 4 h + e % 4, channel c32.  Buffer accesses from the wave's first token and
    // channel: rows behind the last one lie behind the buffer's end, and are not stored; so do channels, moved there.
    const int left_m = a.n_rows - first_m, left_n = a.n_out - first_n;
    auto resource = [&](const void* p, int64_t stride, int size) __attribute__((always_inline)) {
        const int64_t bytes = left_m > 0 && left_n > 0 ? ((left_m - 1) * stride + left_n) * size : 0;
        return __builtin_amdgcn_make_buffer_rsrc((uint8_t*)p + (first_m * stride + first_n) * size, 0, (int)(uint32_t)min(bytes, (int64_t)0xBFFFFFF0), 0x00020000);
    };
    const auto y0 = resource(a.y, a.y_stride, SIZE), add0 = resource(a.add, a.add_stride, a.add ? 4 : 0);
    const uint32_t y_row = (uint32_t)a.y_stride * SIZE, add_row = (uint32_t)a.add_stride * 4;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        f32x4 sx[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) sx[b] = *(const f32x4*)(s_scale + wm * WM + 32 * i + 4 * h + 8 * b);
#pragma unroll
        for (int j = 0; j < NO; ++j) {
            const bool there = 32 * j + c32 < left_n;
            const uint32_t y_at = there ? (32 * i + 4 * h) * y_row + (32 * j + c32) * SIZE : 0xC0000000u;
            float add[16];
            if (a.add) {
                const uint32_t at = there ? (32 * i + 4 * h) * add_row + (32 * j + c32) * 4 : 0xC0000000u;
#pragma unroll
                for (int e = 0; e < 16; ++e) add[e] = as_f32(__builtin_amdgcn_raw_buffer_load_b32(add0, at + (8 * (e / 4) + e % 4) * add_row, 0, 0));
            }
            float value[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) value[e] = (float)acc[i][j][e] * sx[e / 4][e % 4] * sw[j];
            if constexpr (GATED) {
                float up[16], top = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    up[e] = (float)acc[i][j + NO][e] * sx[e / 4][e % 4] * su[j];
                    top = fmaxf(top, fabsf(value[e]));
                }
                if (__builtin_expect(__ballot(top > GATE_NEAR) != 0, 0)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) value[e] = gated_up_far(value[e], up[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) value[e] = gated_up(value[e], up[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float y = value[e];
                if (a.add) y += add[e];
                const uint32_t at = y_at + (8 * (e / 4) + e % 4) * y_row;
                if constexpr (TYPE == TYPE_F32)
                    __builtin_amdgcn_raw_buffer_store_b32(as_u32(y), y0, at, 0, 0);
                else
                    __builtin_amdgcn_raw_buffer_store_b16(f2h(y), y0, at, 0, 0);
            }
        }
    }
}

template <int TYPE, bool GATED, int BM, int BN, int WM, int WN, int KW, int NS>
hipError_t matmul_tiles(const I8MatmulArgs& a, hipStream_t s) {
    constexpr int stages = KW * NS * (BM + BN) * 128, lds = stages + BM * 4;
    static_assert((KW - 1) * BM * BN * 4 <= stages);
    const auto kernel = i8_matmul_kernel<TYPE, GATED, BM, BN, WM, WN, KW, NS>;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const int out = GATED ? BN / 2 : BN, tm = (a.n_rows + BM - 1) / BM, tn = (a.n_out + out - 1) / out;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)tm * tn + 7) / 8 * 8), dim3(BM / WM * (BN / WN) * KW * 64), lds, s, a, tm, tn);
    return hipGetLastError();
}

// Few tokens: a matrix value takes part in few products, and goes from memory to registers.  A workgroup has ROWS matrix
// rows (gated: as many gates and their ups) and 16 MB tokens; its eight waves take 128 codes of all rows in turn, on
// v_mfma_i32_16x16x64_i8 (matrix rows as the result's rows, tokens as its columns), and join their sums through LDS.  A
// row's 128 codes are one line of memory: lane (row, q) has 32 of them, and the tokens' operands take theirs in the same
// order.  Bound by memory and its latency: 8 tokens, 4096 channels, 2048 deep, 8 MB, in 4.0 us; 16 tokens of 6144 gated
// channels, 25 MB, in 8.5 us, 3.0 TB/s.
template <int TYPE, bool GATED, int RB, int MB, int DEPTH>
__global__ __launch_bounds__(512) void i8_stream_kernel(I8MatmulArgs a) {
    constexpr int NW = 8, SETS = GATED ? 2 : 1, ROWS = 16 * RB, TOKENS = 16 * MB, VALUES = ROWS * TOKENS;
    constexpr int PER = (VALUES + 511) / 512;  // outputs of a thread
    __shared__ __align__(16) int s_sum[NW][SETS * RB * MB][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * ROWS, m0 = blockIdx.y * TOKENS;
    const int8_t *wp[SETS][RB], *xp[MB];
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < RB; ++i) wp[s][i] = a.w + (min(n0 + 16 * i + r16, a.n_out - 1) + (s ? (int64_t)a.n_out : 0)) * a.w_stride + 32 * q;
#pragma unroll
    for (int j = 0; j < MB; ++j) xp[j] = a.x + min(m0 + 16 * j + r16, a.n_rows - 1) * a.x_stride + 32 * q;
    // What the outputs of this thread take, asked for before the products: value v is of token v / ROWS, channel v % ROWS.
    float sx[PER], sw[PER], su[PER], add[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int v = i * 512 + tid, m = min(m0 + v / ROWS, a.n_rows - 1), n = min(n0 + v % ROWS, a.n_out - 1);
        sx[i] = a.x_scales[m];
        sw[i] = a.w_scales[n];
        su[i] = GATED ? a.w_scales[a.n_out + n] : 0.f;
        add[i] = !GATED && a.add ? a.add[m * a.add_stride + n] : 0.f;
    }
    struct Step {
        i32x4 w[SETS][RB][2], x[MB][2];
    };
    const int steps = (a.n_in + 127) / 128;
    auto load = [&](int it, Step& t) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = it * 128 + 16 * k, at = c + 32 * q < a.n_in ? c : -32 * q;  // behind the last code: the first ones
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int i = 0; i < RB; ++i) t.w[s][i][k] = *(const i32x4*)(wp[s][i] + at);
#pragma unroll
            for (int j = 0; j < MB; ++j) t.x[j][k] = *(const i32x4*)(xp[j] + at);
        }
    };
    i32x4 acc[SETS][RB][MB];
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j) acc[s][i][j] = i32x4{};
    auto products = [&](int it, Step& t) __attribute__((always_inline)) {
        if (it == steps - 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (it * 128 + 16 * k + 32 * q >= a.n_in)
#pragma unroll
                    for (int j = 0; j < MB; ++j) t.x[j][k] = i32x4{};
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int i = 0; i < RB; ++i)
#pragma unroll
                    for (int j = 0; j < MB; ++j) acc[s][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(t.w[s][i][k], t.x[j][k], acc[s][i][j], 0, 0, 0);
    };
    Step t[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + NW * d < steps) load(wave + NW * d, t[d]);
    for (int it = wave; it < steps; it += NW * DEPTH)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (it + NW * d < steps) {
                products(it + NW * d, t[d]);
                if (it + NW * (d + DEPTH) < steps) load(it + NW * (d + DEPTH), t[d]);
            }
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j) *(i32x4*)&s_sum[wave][(s * RB + i) * MB + j][4 * lane] = acc[s][i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int v = i * 512 + tid, m = v / ROWS, n = v % ROWS;
        if (v >= VALUES || m0 + m >= a.n_rows || n0 + n >= a.n_out) continue;
        const int block = n / 16 * MB + m / 16, at = (n % 16 / 4 * 16 + m % 16) * 4 + n % 4;
        int sum[SETS] = {};
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int w = 0; w < NW; ++w) sum[s] += s_sum[w][s * RB * MB + block][at];
        float y = (float)sum[0] * sx[i] * sw[i];
        if constexpr (GATED) {
            const float up = (float)sum[SETS - 1] * sx[i] * su[i];
            y = fabsf(y) > GATE_NEAR ? gated_up_far(y, up) : gated_up(y, up);
        }
        if (a.add) y += add[i];
        const int64_t o = (int64_t)(m0 + m) * a.y_stride + n0 + n;
        if constexpr (TYPE == TYPE_F32)
            ((float*)a.y)[o] = y;
        else
            ((f16*)a.y)[o] = (f16)y;
    }
}

template <int TYPE, bool GATED, int RB, int MB, int DEPTH>
hipError_t matmul_stream(const I8MatmulArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((i8_stream_kernel<TYPE, GATED, RB, MB, DEPTH>), dim3((a.n_out + 16 * RB - 1) / (16 * RB), (a.n_rows + 16 * MB - 1) / (16 * MB)), dim3(512), 0, s, a);
    return hipGetLastError();
}

template <int TYPE, bool GATED>
hipError_t matmul_of(const I8MatmulArgs& a, hipStream_t s) {
    const I8FormId form = i8_form(GATED, a.n_rows, a.n_out, a.n_in);
    switch (form) {
        case I8_STREAM_16: return matmul_stream<TYPE, GATED, 1, 1, 2>(a, s);
        case I8_STREAM_32: return matmul_stream<TYPE, GATED, 1, 2, 2>(a, s);
        case I8_64x128: return matmul_tiles<TYPE, GATED, 64, 128, 32, 64, 1, 3>(a, s);
        case I8_128x128: return matmul_tiles<TYPE, GATED, 128, 128, 64, 64, 1, 2>(a, s);
        case I8_128x256: return matmul_tiles<TYPE, GATED, 128, 256, 64, 64, 1, 2>(a, s);
        case I8_128x256_DEEP: return matmul_tiles<TYPE, GATED, 128, 256, 64, 64, 1, 3>(a, s);
        case I8_256x256: return matmul_tiles<TYPE, GATED, 256, 256, 128, 64, 1, 2>(a, s);
        default: break;
    }
    if constexpr (!GATED) {  // waves of 32 x 32, which do not hold gates and ups
        switch (form) {
            case I8_32x32: return matmul_tiles<TYPE, GATED, 32, 32, 32, 32, 8, 2>(a, s);
            case I8_32x64: return matmul_tiles<TYPE, GATED, 32, 64, 32, 32, 4, 3>(a, s);
            case I8_64x64_DEEP: return matmul_tiles<TYPE, GATED, 64, 64, 32, 32, 1, 4>(a, s);
            case I8_64x64: return matmul_tiles<TYPE, GATED, 64, 64, 32, 32, 1, 2>(a, s);
            default: break;
        }
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_i8_quantize(int type, const I8QuantArgs& a, hipStream_t s) {
    if (a.norm) return type == TYPE_F32 ? quantize_of<TYPE_F32, true>(a, s) : quantize_of<TYPE_F16, true>(a, s);
    return type == TYPE_F32 ? quantize_of<TYPE_F32, false>(a, s) : quantize_of<TYPE_F16, false>(a, s);
}

hipError_t launch_i8_matmul(int type, bool gated, const I8MatmulArgs& a, hipStream_t s) {
    if (type == TYPE_F32) return gated ? matmul_of<TYPE_F32, true>(a, s) : matmul_of<TYPE_F32, false>(a, s);
    return gated ? matmul_of<TYPE_F16, true>(a, s) : matmul_of<TYPE_F16, false>(a, s);
}

}  // namespace icua
