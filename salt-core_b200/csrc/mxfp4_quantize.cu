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

constexpr int MQ_THREADS = 128;

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

template <int FT, bool VALUES> __global__ void __launch_bounds__(MQ_THREADS) mxfp4_quantize_kernel(const QuantArgs a) {
    using T = typename FloatType<FT>::T;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x;
    long long src = a.index ? (long long)a.index[row] : row;
    if (src < 0) return;                                 // an index below zero leaves its row as it was
    src /= a.div;
    if (src >= a.src_rows) return;
    const int unit = blockIdx.y * MQ_THREADS + threadIdx.x;          // eight columns
    const bool live = unit * 8 < a.cols;                 // the four lanes of a block agree
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) load8<FT>((const T*)a.x + (size_t)src * a.stride + unit * 8, v);
    uint32_t top = 0;                                    // magnitudes order like their bits, NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (!live) return;
    const uint32_t ex = top >> 23;                       // biased exponent; 0: subnormal or zero
    const bool bad = ex == 255u;
    const uint32_t s = bad ? 255u : (ex > 2u ? ex - 2u : 0u);
    const float up = __uint_as_float((254u - min(s, 253u)) << 23);   // 2^(127 - s); s is at most 252 unless bad
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float lo = bad ? 0.f : __fmul_rn(v[2 * i], up), hi = bad ? 0.f : __fmul_rn(v[2 * i + 1], up);
        uint32_t b;
        asm("{ .reg .b8 q;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 q, %2, %1;\n\t"
            "cvt.u32.u8 %0, q; }\n"
            : "=r"(b)
            : "f"(lo), "f"(hi));
        packed |= b << (8 * i);
    }
    *(uint32_t*)(a.codes + (size_t)row * (a.cols / 2) + unit * 4) = packed;
    if ((unit & 3) == 0) a.scales[(size_t)row * a.pitch + (unit >> 2)] = (uint8_t)s;
    if (VALUES) {
        // magnitude of a code: bits m e1 e0 -> by arithmetic on the exponent; 2^(s - 127) has s = 0 as a subnormal
        const float unit_value = __uint_as_float(s == 0u || s == 255u ? (s << 23) | 0x400000u : s << 23);
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t c = (packed >> (4 * i)) & 15u, e = (c >> 1) & 3u, m = c & 1u;
            const float mag = e ? __uint_as_float(((126u + e) << 23) | (m << 22)) : 0.5f * (float)m;
            o[i] = __fmul_rn(c & 8u ? -mag : mag, unit_value);
        }
        store8<FT>((T*)a.values + (size_t)row * a.cols + unit * 8, o);
    }
}

template <int FT> cudaError_t launch_quantize(const QuantArgs& a, cudaStream_t stream) {
    const dim3 grid(a.rows, (a.cols / 8 + MQ_THREADS - 1) / MQ_THREADS);
    return a.values ? launch_pdl(mxfp4_quantize_kernel<FT, true>, grid, dim3(MQ_THREADS), 0, stream, a)
                    : launch_pdl(mxfp4_quantize_kernel<FT, false>, grid, dim3(MQ_THREADS), 0, stream, a);
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
