// MXFP4 products of few rows: y[t][r] = sum over blocks of 32 columns of 2^(sw + sx - 254) * sum cw cx.
//
// E2M1 values are halves of the integers 0, 1, 2, 3, 4, 6, 8, 12, so a block's sum of products is a whole number of quarters
// below 4608: it is formed without rounding by byte dot products, scaled once and added in 32 bits.  Bound by the weights, which
// are read once per pass of up to eight rows.
//
// A warp owns eight stored rows: r, r + 1 and the same 32, 64 and 96 further on, whose scale bytes share one 32-byte sector per
// 128 columns; a lane owns one block of 32 columns per step, so a weight load is 16 bytes a lane.  The block's activations lie in
// shared memory as signed bytes.  A gated pair's two rows are in one lane's hands at the end.
#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "mxfp4.h"
#include "pdl.cuh"

namespace sb {
namespace {

constexpr int FR_WARPS = 8;
constexpr int FR_ROWS = FR_WARPS * 8;    // stored rows of a block: half a scale tile
constexpr size_t FR_MAX_SMEM = 200 * 1024;

struct FewRowsArgs {
    Mxfp4Weights w;
    Mxfp4Call c;
    int first_pass;
};

// Four codes (the low nibbles' order) as signed bytes, in halves: the selector's top bit makes the byte permutation repeat a
// sign, which is 0 for every table entry, so positives and negatives are looked up apart.
__device__ __forceinline__ uint32_t four_codes(uint32_t sel) {
    constexpr uint32_t LO = 0x03020100u, HI = 0x0c080604u;
    uint32_t p, n;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(p) : "r"(LO), "r"(HI), "r"(sel));
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(n) : "r"(LO), "r"(HI), "r"(sel ^ 0x8888u));
    return p | ((0x80808080u - n) ^ 0x80808080u);
}

__device__ __forceinline__ float scale_value(uint32_t s) {   // 2^(s - 127); 255 is NaN
    return __uint_as_float(s == 0u || s == 255u ? (s << 23) | 0x400000u : s << 23);
}

template <int NT> __global__ void __launch_bounds__(FR_WARPS * 32) mxfp4_few_rows_kernel(const FewRowsArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_find[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nb = a.w.cols / 32;
    uint4* xq = (uint4*)smem;                            // [NT][2][nb]: columns 0..15 and 16..31 of every block, a byte each
    float* xs = (float*)(xq + (size_t)NT * 2 * nb);      // [NT][nb]: a quarter of the scale
    pdl_wait();
    pdl_launch_dependents();
    // the rows of this block's pass
    const int pass = a.first_pass + blockIdx.y;
    int expert = 0, row0 = pass * NT, n = min(NT, a.c.rows - row0);
    if (a.c.offsets) {
        // pass p stands for grouped row p and works where a pass of its group begins
        row0 = pass;
        if (tid == 0) s_find[0] = -1;
        __syncthreads();
        for (int e = tid; e < a.w.experts; e += FR_WARPS * 32) {
            const int b = max(a.c.offsets[e], 0), t = min(a.c.offsets[e + 1], a.c.rows);
            if (row0 >= b && row0 < t && (row0 - b) % NT == 0) { s_find[0] = e; s_find[1] = t; }
        }
        __syncthreads();
        expert = s_find[0];
        if (expert < 0) return;
        n = min(NT, s_find[1] - row0);
    }
    const int words = nb * 4;                            // 32-bit words of a row's codes
    for (int i = tid; i < NT * words; i += FR_WARPS * 32) {
        const int t = i / words, k = i - t * words;      // word k: columns 8 k .. 8 k + 7
        uint32_t q = 0;
        if (t < n) q = ((const uint32_t*)(a.c.codes + (size_t)(row0 + t) * (a.w.cols / 2)))[k];
        const int b = k >> 2, part = (k >> 1) & 1;
        ((uint2*)(xq + (size_t)(t * 2 + part) * nb + b))[k & 1] = make_uint2(four_codes(q), four_codes(q >> 16));
    }
    const size_t pitch = ((size_t)nb + 15) / 16 * 16;
    for (int i = tid; i < NT * nb; i += FR_WARPS * 32) {
        const int t = i / nb, b = i - t * nb;
        xs[i] = t < n ? 0.25f * scale_value(a.c.scales[(size_t)(row0 + t) * pitch + b]) : 0.f;
    }
    __syncthreads();

    const int tile = blockIdx.x >> 1;
    const int r32 = (blockIdx.x & 1) * 16 + warp * 2;    // row % 32 of the warp's first row
    const int r0 = tile * 128 + r32;
    const uint8_t* wc = a.w.codes + (size_t)expert * a.w.stored_rows * (a.w.cols / 2);
    const uint8_t* ws = a.w.scales + ((size_t)expert * a.w.row_tiles + tile) * a.w.col_tiles * 512 + r32 * 16;
    float acc[8][NT];
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[j][t] = 0.f;
    for (int b = lane; b < nb; b += 32) {
        uint4 q[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = min(r0 + (j >> 1) * 32 + (j & 1), a.w.stored_rows - 1);
            q[j] = __ldg((const uint4*)(wc + (size_t)r * (a.w.cols / 2)) + b);
        }
        const uint4 s0 = __ldg((const uint4*)(ws + (size_t)(b >> 2) * 512));
        const uint4 s1 = __ldg((const uint4*)(ws + (size_t)(b >> 2) * 512) + 1);
        const int sh = (b & 3) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint4 s = (j & 1) ? s1 : s0;
            const uint32_t sw = j < 2 ? s.x : j < 4 ? s.y : j < 6 ? s.z : s.w;
            const float wv = scale_value((sw >> sh) & 255u);
            const uint32_t cw[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
            uint32_t w8[8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                w8[2 * k] = four_codes(cw[k]);
                w8[2 * k + 1] = four_codes(cw[k] >> 16);
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint4 x0 = xq[(size_t)(t * 2) * nb + b], x1 = xq[(size_t)(t * 2 + 1) * nb + b];
                int d = __dp4a((int)w8[0], (int)x0.x, 0);
                d = __dp4a((int)w8[1], (int)x0.y, d);
                d = __dp4a((int)w8[2], (int)x0.z, d);
                d = __dp4a((int)w8[3], (int)x0.w, d);
                d = __dp4a((int)w8[4], (int)x1.x, d);
                d = __dp4a((int)w8[5], (int)x1.y, d);
                d = __dp4a((int)w8[6], (int)x1.z, d);
                d = __dp4a((int)w8[7], (int)x1.w, d);
                acc[j][t] = __fmaf_rn((float)d * xs[t * nb + b], wv, acc[j][t]);
            }
        }
    }
    // Sums over the lanes: each of two exchanges halves the row pairs a lane keeps, three more finish; lanes 8 p hold pair p.
#pragma unroll
    for (int t = 0; t < NT; t++) {
        float u[2], v[2];                                // first and second row of two pairs
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const bool high = lane & 16;
            const float a0 = high ? acc[2 * (p + 2)][t] : acc[2 * p][t], b0 = high ? acc[2 * p][t] : acc[2 * (p + 2)][t];
            const float a1 = high ? acc[2 * (p + 2) + 1][t] : acc[2 * p + 1][t], b1 = high ? acc[2 * p + 1][t] : acc[2 * (p + 2) + 1][t];
            u[p] = a0 + __shfl_xor_sync(0xffffffffu, b0, 16);
            v[p] = a1 + __shfl_xor_sync(0xffffffffu, b1, 16);
        }
        const bool high = lane & 8;
        float first = (high ? u[1] : u[0]) + __shfl_xor_sync(0xffffffffu, high ? u[0] : u[1], 8);
        float second = (high ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[1], 8);
#pragma unroll
        for (int d = 4; d; d >>= 1) {
            first += __shfl_xor_sync(0xffffffffu, first, d);
            second += __shfl_xor_sync(0xffffffffu, second, d);
        }
        const int r = r0 + (lane >> 3) * 32;
        if ((lane & 7) == 0 && t < n && r < a.w.stored_rows) {
            const size_t o = (size_t)(row0 + t) * a.c.y_stride;
            if (a.w.activation) {
                store_float(a.c.y, a.c.y_type, o + (r >> 1), gate_act(a.w.activation, first) * second);
            } else {
                store_float(a.c.y, a.c.y_type, o + r, first);
                if (r + 1 < a.w.stored_rows) store_float(a.c.y, a.c.y_type, o + r + 1, second);
            }
        }
    }
}

template <int NT> size_t few_rows_smem(int cols) { return (size_t)NT * (cols + cols / 32 * sizeof(float)); }

template <int NT> cudaError_t launch(const FewRowsArgs& a, cudaStream_t stream) {
    const size_t smem = few_rows_smem<NT>(a.w.cols);
    cudaError_t e;
    if (smem > PLAIN_DYNAMIC_SMEM && (e = ensure_dynamic_smem((const void*)mxfp4_few_rows_kernel<NT>, smem)) != cudaSuccess) return e;
    const int passes = a.c.offsets ? a.c.rows : (a.c.rows + NT - 1) / NT;
    const unsigned row_blocks = 2 * a.w.row_tiles;
    // a launch has at most 65535 blocks along y; the passes beyond follow in launches of their own
    for (int first = 0; first < passes; first += 65535) {
        FewRowsArgs part = a;
        part.first_pass = first;
        e = launch_pdl(mxfp4_few_rows_kernel<NT>, dim3(row_blocks, std::min(65535, passes - first)), dim3(FR_WARPS * 32), smem, stream, part);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_mxfp4_few_rows(const Mxfp4Weights& w, const Mxfp4Call& c, cudaStream_t stream) {
    FewRowsArgs a;
    a.w = w;
    a.c = c;
    a.first_pass = 0;
    // rows of a pass: as many as there are, or as an expert has on average, rounded up; fewer where they do not fit
    const int want = c.offsets ? (c.rows + w.experts - 1) / w.experts : c.rows;
    if (want > 4 && few_rows_smem<8>(w.cols) <= FR_MAX_SMEM) return launch<8>(a, stream);
    if (want > 2 && few_rows_smem<4>(w.cols) <= FR_MAX_SMEM) return launch<4>(a, stream);
    if (want > 1 && few_rows_smem<2>(w.cols) <= FR_MAX_SMEM) return launch<2>(a, stream);
    return launch<1>(a, stream);
}

}  // namespace sb
