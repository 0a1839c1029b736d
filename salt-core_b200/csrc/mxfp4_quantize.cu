// Rows to MXFP4: per 32 columns one E8M0 scale and 32 E2M1 codes, two per byte, the even column in the low nibble.
//
//   E = floor(log2(max |x|)), scale byte s = clamp(E - 2 + 127, 0, 254): the largest magnitude lands in [4, 8);
//   code = x * 2^(127 - s) to the nearest E2M1 value (0, .5, 1, 1.5, 2, 3, 4, 6), ties to the even code, 6 beyond;
//   a block with a NaN or an infinity has scale byte 255, which reads as NaN, and codes 0.
// The scale is a power of two, so scaling is exact (values that become subnormal by it are far below half a step) and the only
// rounding is the one to the code, by the conversion instruction.
//
// Four lanes share a block, eight columns each: one or two 16-byte loads, a maximum over four lanes, one 4-byte store.
// Bound by memory.
#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "pdl.cuh"

namespace sb {
bool cuda_ok(cudaError_t e, const char* what);

namespace {

constexpr int MQ_MAX_THREADS = 256;

struct QuantArgs {
    const void* x;
    size_t stride;
    int src_rows, cols, rows, div;
    const int32_t* index;
    uint8_t* codes;
    uint8_t* scales;
    size_t pitch;
    void* values;
};

// A block works on one row, a thread on U pieces of eight columns, whose loads are all in flight before the first is used.
template <int FT, bool VALUES, int U> __global__ void __launch_bounds__(MQ_MAX_THREADS) mxfp4_quantize_kernel(const QuantArgs a) {
    using T = typename FloatType<FT>::T;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x;
    int src = row;
    if (a.index) {
        src = __ldg(a.index + row);
        if (src < 0) return;                             // an index below zero leaves its row as it was
        src = (int)((unsigned)src / (unsigned)a.div);
    }
    if (src >= a.src_rows) return;
    const T* x = (const T*)a.x + (size_t)src * a.stride;
    const int first = blockIdx.y * U * blockDim.x + threadIdx.x, units = a.cols / 8;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int unit = first + u * blockDim.x;         // the four lanes of a block of 32 columns agree on it
#pragma unroll
        for (int i = 0; i < 8; i++) v[u][i] = 0.f;
        if (unit < units) load8<FT>(x + unit * 8, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int unit = first + u * blockDim.x;
        uint32_t top = 0;                                // magnitudes order like their bits, NaN above infinity
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[u][i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t ex = top >> 23;                   // biased exponent; 0: subnormal or zero
        const bool bad = ex == 255u;
        const uint32_t s = bad ? 255u : (ex > 2u ? ex - 2u : 0u);
        const float up = __uint_as_float((254u - min(s, 253u)) << 23);   // 2^(127 - s); s is at most 252 unless bad
        uint32_t packed = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t b;
            asm("{ .reg .b8 q;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 q, %2, %1;\n\t"
                "cvt.u32.u8 %0, q; }\n"
                : "=r"(b)
                : "f"(__fmul_rn(v[u][2 * i], up)), "f"(__fmul_rn(v[u][2 * i + 1], up)));
            packed |= b << (8 * i);
        }
        if (bad) packed = 0;
        if (unit >= units) continue;
        *(uint32_t*)(a.codes + (size_t)row * (a.cols / 2) + unit * 4) = packed;
        if ((unit & 3) == 0) a.scales[(size_t)row * a.pitch + (unit >> 2)] = (uint8_t)s;
        if (VALUES) {
            const float unit_value = __uint_as_float(s == 0u || s == 255u ? (s << 23) | 0x400000u : s << 23);     // 2^(s - 127); NaN
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t h;                              // two codes as halves, exactly
                asm("{ .reg .b8 q;\n\t"
                    "cvt.u8.u32 q, %1;\n\t"
                    "cvt.rn.f16x2.e2m1x2 %0, q; }\n"
                    : "=r"(h)
                    : "r"(packed >> (8 * i)));
                const float2 f = __half22float2(*(const __half2*)&h);
                o[2 * i] = __fmul_rn(f.x, unit_value);
                o[2 * i + 1] = __fmul_rn(f.y, unit_value);
            }
            store8<FT>((T*)a.values + (size_t)row * a.cols + unit * 8, o);
        }
    }
}

template <int FT, bool VALUES> cudaError_t launch_quantize(const QuantArgs& a, cudaStream_t stream) {
    const int units = a.cols / 8;
    // four pieces per thread where the rows fill the SMs, one where a call is nothing but latency
    const int per = a.rows >= 4 * device_sms() ? 4 : 1;
    const int blocks = (units + MQ_MAX_THREADS * per - 1) / (MQ_MAX_THREADS * per);
    const int threads = (((units + blocks - 1) / blocks + per - 1) / per + 31) / 32 * 32;
    const dim3 grid(a.rows, blocks);
    return per == 4 ? launch_pdl(mxfp4_quantize_kernel<FT, VALUES, 4>, grid, dim3(threads), 0, stream, a)
                    : launch_pdl(mxfp4_quantize_kernel<FT, VALUES, 1>, grid, dim3(threads), 0, stream, a);
}

template <int FT> cudaError_t launch_quantize(const QuantArgs& a, cudaStream_t stream) {
    return a.values ? launch_quantize<FT, true>(a, stream) : launch_quantize<FT, false>(a, stream);
}

}  // namespace
}  // namespace sb

extern "C" size_t salt_b200_mxfp4_scale_pitch(int cols) { return cols < 32 ? 16 : ((size_t)cols / 32 + 15) / 16 * 16; }

extern "C" int salt_b200_mxfp4_quantize(const void* d_x, int dtype, size_t row_stride, int src_rows, int cols,
                                        const int32_t* d_row_index, int index_div, int rows, uint8_t* d_codes, uint8_t* d_scales,
                                        void* d_values, void* stream) {
    using namespace sb;
    if (!float_type_ok(dtype) || cols < 32 || cols % 32 || cols > SALT_B200_MXFP4_MAX_COLS || rows < 0 || src_rows < 0 ||
        index_div < 1 || row_stride < (size_t)cols || row_stride > (size_t)1 << 40 || (!d_row_index && rows > src_rows))
        return -1;
    if (rows == 0) return 0;
    const size_t size = float_type_size(dtype);
    if ((!d_x && src_rows > 0) || !d_codes || !d_scales || (uintptr_t)d_x % 16 || row_stride * size % 16 || (uintptr_t)d_codes % 16 ||
        (uintptr_t)d_scales % 16 || (uintptr_t)d_values % 16)
        return -1;
    QuantArgs a;
    a.x = d_x; a.stride = row_stride; a.src_rows = src_rows; a.cols = cols; a.rows = rows; a.div = d_row_index ? index_div : 1; a.index = d_row_index;
    a.codes = d_codes; a.scales = d_scales; a.pitch = salt_b200_mxfp4_scale_pitch(cols); a.values = d_values;
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = dtype == FT_F32    ? launch_quantize<FT_F32>(a, st)
                          : dtype == FT_BF16 ? launch_quantize<FT_BF16>(a, st)
                                             : launch_quantize<FT_F16>(a, st);
    return cuda_ok(e, "mxfp4 quantize") ? 0 : -1;
}
