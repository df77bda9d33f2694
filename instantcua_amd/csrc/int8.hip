// Products on 8-bit integers with a scale for each token and each output channel, gfx950: the tokens' rows are
// (normalised and) quantised, multiplied by a matrix of codes on the int8 matrix cores, and scaled into rows of y.
#include "icua_device.h"
#include "icua_kernels.h"

namespace icua {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------
// Quantisation of rows.  y = x norm / sqrt(mean(x^2) + eps), or x:  scale = max |y| / 127, code = y / scale rounded
// to the nearest, ties to even.  The root mean square is common to a row's values and leaves the codes as they are
// without it: code = 127 t / max |t| of t = x norm.  All of it in 64 bits, where t is exact and the quotient rounds
// as the exact one does but for ties, which the division decides: codes are those of the definition.

template <int TYPE>
__device__ __forceinline__ f32x4 load_x(const void* p, int64_t i) {
    if constexpr (TYPE == TYPE_F32) return *(const f32x4*)((const float*)p + i);
    const v4h h = *(const v4h*)((const f16*)p + i);
    return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

// A workgroup a row.
template <int TYPE>
__global__ __launch_bounds__(256) void i8_quantize_kernel(I8QuantArgs a) {
    __shared__ double s_top[4], s_sum[4];
    __shared__ int s_odd[4];
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t at = (int64_t)row * a.x_stride;
    double top = 0., sum = 0.;
    bool odd = false;
    for (int i = 4 * threadIdx.x; i < a.n_cols; i += 1024) {
        const f32x4 x = load_x<TYPE>(a.x, at + i);
        f32x4 w = {1.f, 1.f, 1.f, 1.f};
        if (a.norm) w = *(const f32x4*)(a.norm + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double t = (double)x[e] * (double)w[e];
            odd |= !(fabs(t) < __builtin_inf());
            top = fmax(top, fabs(t));
            sum += (double)x[e] * (double)x[e];
        }
    }
    for (int o = 1; o < WAVE; o <<= 1) {
        top = fmax(top, __shfl_xor(top, o));
        sum += __shfl_xor(sum, o);
    }
    odd = __ballot(odd) != 0;
    if (lane == 0) {
        s_top[wave] = top;
        s_sum[wave] = sum;
        s_odd[wave] = odd;
    }
    __syncthreads();
    top = fmax(fmax(s_top[0], s_top[1]), fmax(s_top[2], s_top[3]));
    sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    odd = (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3]) != 0;
    if (threadIdx.x == 0) {
        const double r = a.norm ? 1. / sqrt(sum / a.n_cols + (double)a.eps) : 1.;
        a.scales[row] = odd ? __builtin_nanf("") : (float)(top * r / 127.);
    }
    for (int i = 4 * threadIdx.x; i < a.n_cols; i += 1024) {
        const f32x4 x = load_x<TYPE>(a.x, at + i);
        f32x4 w = {1.f, 1.f, 1.f, 1.f};
        if (a.norm) w = *(const f32x4*)(a.norm + i);
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double t = (double)x[e] * (double)w[e];
            const int code = odd || top == 0. ? 0 : (int)__builtin_rint(127. * t / top);
            word |= (uint32_t)(code & 255) << (8 * e);
        }
        *(uint32_t*)(a.codes + (int64_t)row * a.codes_stride + i) = word;
    }
}

// ------------------------------------------------------------------------------------------
// Products.  y[m][n] = x_scales[m] w_scales[n] sum_k x[m][k] w[n][k] (+ add[m][n]), the sums exact in 32-bit integers
// (|sum| <= 127^2 2^17 < 2^31); or, of two matrices, silu(gate) up.

__device__ __constant__ const u32x4 g_zero_codes = {0, 0, 0, 0};  // what lies behind a row's last code

// A tile of BM tokens and BN matrix rows a workgroup, WM x WN of it a wave, on v_mfma_i32_32x32x32_i8: tokens are
// the result's rows, channels its columns, so that a wave's stores are runs of 32 channels.  Rows are staged in LDS
// 128 codes at a time, two stages, by copies that run under the products; row r's 16-byte chunk c lies at place c ^
// (r & 7), so that eight rows' reads of one chunk meet no bank twice.  Gated: half of a wave's matrix rows are
// gates, the other half the same channels' ups.
template <int TYPE, bool GATED, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void i8_matmul_kernel(I8MatmulArgs a, int tiles_m, int tiles_n) {
    constexpr int THREADS = BM / WM * (BN / WN) * 64, STAGE = (BM + BN) * 128;
    constexpr int CX = BM * 8 / THREADS, CW = BN * 8 / THREADS, NI = WM / 32, NJ = WN / 32;
    constexpr int OUT = GATED ? BN / 2 : BN, WOUT = GATED ? WN / 2 : WN;  // channels of y of the tile, of a wave
    extern __shared__ __align__(1024) uint8_t lds[];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % (BM / WM), wn = wave / (BM / WM), c32 = lane & 31, h = lane >> 5;
    const int m0 = blockIdx.x % tiles_m * BM, n0 = blockIdx.x / tiles_m * OUT;

    const int8_t *xp[CX], *wp[CW];
#pragma unroll
    for (int i = 0; i < CX; ++i) {
        const int r = (i * THREADS + tid) / 8, m = min(m0 + r, a.n_rows - 1);
        xp[i] = a.x + (int64_t)m * a.x_stride;
    }
#pragma unroll
    for (int i = 0; i < CW; ++i) {
        const int r = (i * THREADS + tid) / 8, w = r / WN, o = r % WN;
        int64_t n = min(n0 + w * WOUT + o % WOUT, a.n_out - 1);
        if (GATED && o >= WOUT) n += a.n_out;
        wp[i] = a.w + n * a.w_stride;
    }
    const int chunk = 16 * ((tid & 7) ^ ((tid >> 3) & 7));  // of every row that this thread copies
    const int steps = (a.n_in + 127) / 128;
    auto stage = [&](int it) __attribute__((always_inline)) {
        const int k = it * 128 + chunk;
        const bool there = k < a.n_in;  // behind the last code: zeros of x, any of the matrix
        const uint32_t dst = lds0 + (it & 1) * STAGE + wave * 1024;
#pragma unroll
        for (int i = 0; i < CX; ++i)
            copy_to_lds(there ? (const uint8_t*)xp[i] + k : (const uint8_t*)&g_zero_codes, dst + i * THREADS * 16);
#pragma unroll
        for (int i = 0; i < CW; ++i)
            copy_to_lds((const uint8_t*)wp[i] + (there ? k : 0), dst + BM * 128 + i * THREADS * 16);
    };
    i32x16 acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = i32x16{};
    auto operand = [&](int at, int r, int ks) __attribute__((always_inline)) {
        return *(const i32x4*)(lds + at + r * 128 + (((2 * ks + h) ^ (r & 7)) << 4));
    };
    stage(0);
    for (int it = 0; it < steps; ++it) {
        staged_barrier<0>();
        if (it + 1 < steps) stage(it + 1);
        const int at = (it & 1) * STAGE;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            i32x4 x[NI], w[NJ];
#pragma unroll
            for (int i = 0; i < NI; ++i) x[i] = operand(at, wm * WM + 32 * i + c32, ks);
#pragma unroll
            for (int j = 0; j < NJ; ++j) w[j] = operand(at + BM * 128, wn * WN + 32 * j + c32, ks);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[i], w[j], acc[i][j], 0, 0, 0);
        }
    }
    // Element e of a block: token 8 (e / 4) + 4 h + e % 4, channel c32.
    constexpr int NO = WOUT / 32;
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        const int n = n0 + wn * WOUT + 32 * j + c32;
        if (n >= a.n_out) continue;
        const float sw = a.w_scales[n], su = GATED ? a.w_scales[a.n_out + n] : 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm * WM + 32 * i + 8 * (e / 4) + 4 * h + e % 4;
                if (m >= a.n_rows) continue;
                const float sx = a.x_scales[m];
                float y = (float)acc[i][j][e] * sx * sw;
                if constexpr (GATED) {
                    const float up = (float)acc[i][j + NO][e] * sx * su;
                    y = y / (1.f + __expf(-y)) * up;
                }
                if (a.add) y += a.add[(int64_t)m * a.add_stride + n];
                const int64_t o = (int64_t)m * a.y_stride + n;
                if constexpr (TYPE == TYPE_F32)
                    ((float*)a.y)[o] = y;
                else
                    ((f16*)a.y)[o] = (f16)y;
            }
    }
}

template <int TYPE, bool GATED, int BM, int BN, int WM, int WN>
hipError_t matmul_tiles(const I8MatmulArgs& a, hipStream_t s) {
    constexpr int lds = 2 * (BM + BN) * 128;
    const auto kernel = i8_matmul_kernel<TYPE, GATED, BM, BN, WM, WN>;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const int out = GATED ? BN / 2 : BN, tm = (a.n_rows + BM - 1) / BM, tn = (a.n_out + out - 1) / out;
    hipLaunchKernelGGL(kernel, dim3((unsigned)tm * tn), dim3(BM / WM * (BN / WN) * 64), lds, s, a, tm, tn);
    return hipGetLastError();
}

template <int TYPE, bool GATED>
hipError_t matmul_of(const I8MatmulArgs& a, hipStream_t s) { return matmul_tiles<TYPE, GATED, 128, 128, 64, 64>(a, s); }

}  // namespace

hipError_t launch_i8_quantize(int type, const I8QuantArgs& a, hipStream_t s) {
    if (type == TYPE_F32)
        hipLaunchKernelGGL(i8_quantize_kernel<TYPE_F32>, dim3(a.n_rows), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(i8_quantize_kernel<TYPE_F16>, dim3(a.n_rows), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_i8_matmul(int type, bool gated, const I8MatmulArgs& a, hipStream_t s) {
    if (type == TYPE_F32) return gated ? matmul_of<TYPE_F32, true>(a, s) : matmul_of<TYPE_F32, false>(a, s);
    return gated ? matmul_of<TYPE_F16, true>(a, s) : matmul_of<TYPE_F16, false>(a, s);
}

}  // namespace icua
