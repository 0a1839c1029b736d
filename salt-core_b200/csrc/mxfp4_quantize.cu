// Rows to MXFP4: per 32 columns one E8M0 scale and 32 E2M1 codes, two per byte, the even column in the low nibble.
//
//   E = floor(log2(max |x|)), scale byte s = clamp(E - 2 + 127, 0, 254): the largest magnitude lands in [4, 8);
//   code = x * 2^(127 - s) to the nearest E2M1 value (0, .5, 1, 1.5, 2, 3, 4, 6), ties to the even code, 6 beyond;
//   a block with a NaN or an infinity has scale byte 255, which reads as NaN, and codes 0.
// The scale is a power of two, so scaling is exact (values that become subnormal by it are far below half a step) and the only
// rounding is the one to the code, by the conversion instruction.
//
// Two lanes share a block, sixteen columns each: two or four 16-byte loads, a maximum over the two, one 8-byte store of codes.  32-bit
// values are written by four lanes a block: a lane's 64 bytes would be four stores apart (15992 gathered rows of 2816: 44 us
// against 61).  4096 x 5120 bf16: 9.7 us, 5.5 TB/s.
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

// Eight columns as they were loaded.  The largest magnitude is found on the bits (NaN lies above infinity), of 16-bit types two at a
// time, and returned as the bits of a float.
template <int FT> struct Raw8 {
    using T = typename FloatType<FT>::T;
    uint4 q = make_uint4(0, 0, 0, 0);
    __device__ __forceinline__ void load(const T* p) { q = *(const uint4*)p; }
    __device__ __forceinline__ uint32_t top() const {    // of the even and of the odd columns
        constexpr uint32_t M = 0x7fff7fffu;
        return __vmaxu2(__vmaxu2(q.x & M, q.y & M), __vmaxu2(q.z & M, q.w & M));
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t t) {
        t = max(t & 0xffffu, t >> 16);
        if (FT == FT_BF16) return t << 16;
        const __half_raw h = {(unsigned short)t};
        return __float_as_uint(__half2float(__half(h)));
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (FT == FT_BF16) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 p = __half22float2(*(const __half2*)&w[i]);
                f[2 * i] = p.x;
                f[2 * i + 1] = p.y;
            }
        }
    }
};
template <> struct Raw8<FT_F32> {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    __device__ __forceinline__ void load(const float* p) { a = ((const float4*)p)[0]; b = ((const float4*)p)[1]; }
    __device__ __forceinline__ void floats(float (&f)[8]) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    __device__ __forceinline__ uint32_t top() const {
        float f[8];
        floats(f);
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) t = max(t, __float_as_uint(f[i]) & 0x7fffffffu);
        return t;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t t) { return t; }
};

// A block works on one row, a thread on U pieces of 8 W columns, whose loads are all in flight before the first is used.
template <int FT, bool VALUES> constexpr int MQ_SIDE = FT == FT_F32 && VALUES ? 1 : 2;

template <int FT, bool VALUES, int U> __global__ void __launch_bounds__(MQ_MAX_THREADS) mxfp4_quantize_kernel(const QuantArgs a) {
    using T = typename FloatType<FT>::T;
    constexpr int W = MQ_SIDE<FT, VALUES>;               // 4 / W lanes share a block
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x;
    int src = row;
    if (a.index) {
        src = a.index[row];
        if (src < 0) return;                             // an index below zero leaves its row as it was
        src = (int)((unsigned)src / (unsigned)a.div);
    }
    if (src >= a.src_rows) return;
    const T* x = (const T*)a.x + (size_t)src * a.stride;
    const int first = blockIdx.y * U * blockDim.x + threadIdx.x, units = a.cols / (8 * W);
    Raw8<FT> v[U][W];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int unit = first + u * blockDim.x;         // the lanes of a block of 32 columns agree on it
        if (unit < units)
#pragma unroll
            for (int h = 0; h < W; h++) v[u][h].load(x + (unit * W + h) * 8);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int unit = first + u * blockDim.x;
        uint32_t most = v[u][0].top();
        if (W == 2) most = Raw8<FT>::larger(most, v[u][W - 1].top());
#pragma unroll
        for (int d = 1; d < 4 / W; d <<= 1) most = Raw8<FT>::larger(most, __shfl_xor_sync(0xffffffffu, most, d));
        const uint32_t top = Raw8<FT>::float_bits(most);
        const uint32_t ex = top >> 23;                   // biased exponent; 0: subnormal or zero
        const bool bad = ex == 255u;
        const uint32_t s = bad ? 255u : (ex > 2u ? ex - 2u : 0u);
        const float up = __uint_as_float((254u - min(s, 253u)) << 23);   // 2^(127 - s); s is at most 252 unless bad
        uint32_t packed[W];
#pragma unroll
        for (int h = 0; h < W; h++) {
            float f[8];
            v[u][h].floats(f);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = __fmul_rn(f[i], up);
            asm("{ .reg .b8 a, b, c, d;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
                "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
                "mov.b32 %0, {a, b, c, d}; }\n"
                : "=r"(packed[h])
                : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
            if (bad) packed[h] = 0;
        }
        if (unit >= units) continue;
        uint8_t* codes = a.codes + (size_t)row * (a.cols / 2) + unit * 4 * W;
        if (W == 2) *(uint2*)codes = make_uint2(packed[0], packed[W - 1]);
        else *(uint32_t*)codes = packed[0];
        if (unit % (4 / W) == 0) a.scales[(size_t)row * a.pitch + unit / (4 / W)] = (uint8_t)s;
        if (VALUES) {
            const float unit_value = __uint_as_float(s == 0u || s == 255u ? (s << 23) | 0x400000u : s << 23);     // 2^(s - 127); NaN
#pragma unroll
            for (int h = 0; h < W; h++) {
                float o[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t p;                          // two codes as halves, exactly
                    asm("{ .reg .b8 q;\n\t"
                        "cvt.u8.u32 q, %1;\n\t"
                        "cvt.rn.f16x2.e2m1x2 %0, q; }\n"
                        : "=r"(p)
                        : "r"(packed[h] >> (8 * i)));
                    const float2 f = __half22float2(*(const __half2*)&p);
                    o[2 * i] = __fmul_rn(f.x, unit_value);
                    o[2 * i + 1] = __fmul_rn(f.y, unit_value);
                }
                store8<FT>((T*)a.values + (size_t)row * a.cols + (unit * W + h) * 8, o);
            }
        }
    }
}

template <int FT, bool VALUES> cudaError_t launch_quantize(const QuantArgs& a, cudaStream_t stream) {
    constexpr int W = MQ_SIDE<FT, VALUES>, MANY = 4 / W;
    const int units = a.cols / (8 * W);
    // 32 columns per thread where the rows fill the SMs, one piece where a call is nothing but latency
    const int per = a.rows >= 4 * device_sms() ? MANY : 1;
    const int blocks = (units + MQ_MAX_THREADS * per - 1) / (MQ_MAX_THREADS * per);
    const int threads = (((units + blocks - 1) / blocks + per - 1) / per + 31) / 32 * 32;
    const dim3 grid(a.rows, blocks);
    return per > 1 ? launch_pdl(mxfp4_quantize_kernel<FT, VALUES, MANY>, grid, dim3(threads), 0, stream, a)
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
        row_stride < (size_t)cols || row_stride > (size_t)1 << 40 || (d_row_index ? index_div < 1 : rows > src_rows))
        return -1;
    if (rows == 0) return 0;
    const size_t size = float_type_size(dtype);
    if ((!d_x && src_rows > 0) || !d_codes || !d_scales || (uintptr_t)d_x % 16 || row_stride * size % 16 || (uintptr_t)d_codes % 16 ||
        (uintptr_t)d_scales % 16 || (uintptr_t)d_values % 16 || (uintptr_t)d_row_index % 4)
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
