// The experts' rows of every token back in token order: y[t] = sum_j w[t][j] * rows[index[t][j]], j ascending, in 32 bits and
// rounded once.  One read of every row that is used and one write per token: bound by memory (1999 tokens of four rows of 5120
// bf16: 18.8 us, 5.4 TB/s).
#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "pdl.cuh"

namespace sb {
bool cuda_ok(cudaError_t e, const char* what);

namespace {

constexpr int CB_THREADS = 128;
constexpr int CB_MAX_TOPK = 32;

struct CombineArgs {
    const void* rows;
    size_t row_stride;
    int n_rows, cols, topk, y_type;
    const int32_t* index;
    const float* weights;
    void* y;
    size_t y_stride;
};

// The token's rows that exist, in their order, without gaps: the loop over them then has no branch between its loads.
struct Picks {
    long long at[CB_MAX_TOPK];
    float w[CB_MAX_TOPK];
    int n;
};
__device__ __forceinline__ void load_picks(const CombineArgs& a, int token, Picks& p) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        long long r = -1;
        float w = 0.f;
        if (lane < a.topk) {
            const long long i = (long long)token * a.topk + lane;
            r = a.index ? (long long)a.index[i] : i;
            w = a.weights[i];
            if (r >= a.n_rows) r = -1;
        }
        const uint32_t live = __ballot_sync(0xffffffffu, r >= 0);
        const int at = __popc(live & ((1u << lane) - 1u));
        if (r >= 0) { p.at[at] = r; p.w[at] = w; }
        if (lane == 0) p.n = __popc(live);
    }
    __syncthreads();
}

// A block = one token and CB_THREADS pieces of eight columns.
template <int FT> __global__ void __launch_bounds__(CB_THREADS) combine_kernel(const CombineArgs a) {
    __shared__ Picks s;
    using T = typename FloatType<FT>::T;
    const int token = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    load_picks(a, token, s);
    const int n = s.n;
    const int c = (blockIdx.y * CB_THREADS + threadIdx.x) * 8;
    if (c >= a.cols) return;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int j = 0; j < n; j++) {
        float v[8];
        load8<FT>((const T*)a.rows + (size_t)s.at[j] * a.row_stride + c, v);
#pragma unroll
        for (int k = 0; k < 8; k++) acc[k] = __fmaf_rn(s.w[j], v[k], acc[k]);
    }
    const size_t o = (size_t)token * a.y_stride + c;
    if (a.y_type == FT_F32) store8<FT_F32>((float*)a.y + o, acc);
    else if (a.y_type == FT_BF16) store8<FT_BF16>((__nv_bfloat16*)a.y + o, acc);
    else store8<FT_F16>((__half*)a.y + o, acc);
}

// Any column count, stride and alignment: a thread per column.
template <int FT> __global__ void __launch_bounds__(CB_THREADS) combine_any_kernel(const CombineArgs a) {
    __shared__ Picks s;
    using T = typename FloatType<FT>::T;
    const int token = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    load_picks(a, token, s);
    const int n = s.n;
    const int c = blockIdx.y * CB_THREADS + threadIdx.x;
    if (c >= a.cols) return;
    float acc = 0.f;
#pragma unroll 4
    for (int j = 0; j < n; j++)
        acc = __fmaf_rn(s.w[j], FloatType<FT>::up(((const T*)a.rows)[(size_t)s.at[j] * a.row_stride + c]), acc);
    store_float(a.y, a.y_type, (size_t)token * a.y_stride + c, acc);
}

template <int FT> cudaError_t launch_combine(const CombineArgs& a, int tokens, bool wide, cudaStream_t stream) {
    const int per = CB_THREADS * (wide ? 8 : 1);
    const dim3 grid(tokens, (a.cols + per - 1) / per);
    return wide ? launch_pdl(combine_kernel<FT>, grid, dim3(CB_THREADS), 0, stream, a)
                : launch_pdl(combine_any_kernel<FT>, grid, dim3(CB_THREADS), 0, stream, a);
}

}  // namespace
}  // namespace sb

extern "C" int salt_b200_combine_experts(const void* d_rows, int dtype, size_t row_stride, int n_rows, int cols,
                                         const int32_t* d_row_index, const float* d_weights, int tokens, int topk, void* d_y,
                                         int y_dtype, size_t y_row_stride, void* stream) {
    using namespace sb;
    if (!float_type_ok(dtype) || !float_type_ok(y_dtype) || n_rows < 0 || cols < 1 || cols > 65535 * CB_THREADS || tokens < 0 ||
        topk < 1 || topk > CB_MAX_TOPK || row_stride < (size_t)cols || y_row_stride < (size_t)cols ||
        row_stride > (size_t)1 << 40 || y_row_stride > (size_t)1 << 40 || (int64_t)tokens * topk > INT32_MAX)
        return -1;
    if (tokens == 0) return 0;
    const size_t size = float_type_size(dtype), y_size = float_type_size(y_dtype);
    if (!d_weights || !d_y || (!d_rows && n_rows > 0) || (uintptr_t)d_rows % size || (uintptr_t)d_y % y_size ||
        ((uintptr_t)d_row_index | (uintptr_t)d_weights) % 4)
        return -1;
    CombineArgs a;
    a.rows = d_rows; a.row_stride = row_stride; a.n_rows = n_rows; a.cols = cols; a.topk = topk; a.y_type = y_dtype;
    a.index = d_row_index; a.weights = d_weights; a.y = d_y; a.y_stride = y_row_stride;
    // eight columns a thread where every row begins on 16 bytes on both sides
    const bool wide = cols % 8 == 0 && (uintptr_t)d_rows % 16 == 0 && row_stride * size % 16 == 0 && (uintptr_t)d_y % 16 == 0 &&
                      y_row_stride * y_size % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = dtype == FT_F32    ? launch_combine<FT_F32>(a, tokens, wide, st)
                          : dtype == FT_BF16 ? launch_combine<FT_BF16>(a, tokens, wide, st)
                                             : launch_combine<FT_F16>(a, tokens, wide, st);
    return cuda_ok(e, "combine experts") ? 0 : -1;
}
