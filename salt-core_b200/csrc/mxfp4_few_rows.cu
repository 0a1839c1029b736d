// MXFP4 products of few rows: y[t][r] = sum over blocks of 32 columns of 2^(sw + sx - 254) * sum cw cx.
//
// E2M1 values are halves of the integers 0, 1, 2, 3, 4, 6, 8, 12, so a block's sum of products is a whole number of quarters
// below 4608: it is formed without rounding by byte dot products, scaled once and added in 32 bits.  Bound by the weights, which
// are read once per pass of up to eight rows.
//
// A block of 256 threads takes one tile of 128 stored weight rows, a pass of the group's rows, and, in a cluster of 1 to 8 blocks,
// its share of the K chunks (256 columns, 17 KB).  Bulk copies bring the tiles into a ring in shared memory; eight lanes share a
// row, a block of 32 columns each, so a load of packed codes is 16 bytes a lane without bank conflicts.  The rows' codes lie in
// shared memory as signed bytes, made once per block.  The cluster's partial sums are added in rank order through distributed
// shared memory: results do not depend on timing.  Every wait is bounded (SB_ERR_TIMEOUT).
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "mxfp4.h"
#include "pdl.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace sb {
namespace {

constexpr int FR_THREADS = 256;
constexpr int FR_MAX_CLUSTER = 8;
constexpr int FR_MAX_STAGES = 8;
constexpr size_t FR_MAX_SMEM = 220 * 1024;

struct FewRowsArgs {
    Mxfp4Weights w;
    Mxfp4Call c;
    int first_pass, cluster, share, stages;      // share: most chunks of a block
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

// Shared memory: ring of tiles | rows' codes as bytes [NT][2][blocks] of 16 | scales [NT][blocks] | partial sums [NT][128]
template <int NT> size_t few_rows_smem(int share, int stages) {
    const size_t blocks = (size_t)share * 8;
    return (size_t)stages * MX_TILE_BYTES + NT * (blocks * 36 + MX_TILE_ROWS * sizeof(float));
}

template <int NT> __global__ void __launch_bounds__(FR_THREADS) mxfp4_few_rows_kernel(const FewRowsArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bar_full[FR_MAX_STAGES], bar_free[FR_MAX_STAGES];
    __shared__ int s_find[2], s_fail;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = a.cluster > 1 ? (int)blockIdx.x % a.cluster : 0, tile = (int)blockIdx.x / a.cluster;
    const int chunk0 = rank * a.share, chunks = max(0, min(a.share, a.w.chunks - chunk0));
    const int nb = a.share * 8;                          // blocks of 32 columns in the tables
    uint4* xq = (uint4*)(smem + (size_t)a.stages * MX_TILE_BYTES);
    float* xs = (float*)(xq + (size_t)NT * 2 * nb);
    float* part = xs + (size_t)NT * nb;
    if (tid == 0) {
        for (int s = 0; s < a.stages; s++) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_free[s], FR_THREADS / 32);
        }
        s_find[0] = -1;
        s_fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const uint8_t* src = a.w.tiles + ((size_t)tile * a.w.chunks + chunk0) * MX_TILE_BYTES;
    if (!a.c.offsets && tid == 0)                        // a dense product's tiles do not wait for the launch before
        for (int k = 0; k < min(a.stages, chunks); k++) {
            mbar_expect_tx(&bar_full[k], MX_TILE_BYTES);
            bulk_load(smem_u32(smem + (size_t)k * MX_TILE_BYTES), src + (size_t)k * MX_TILE_BYTES, MX_TILE_BYTES, smem_u32(&bar_full[k]));
        }
    pdl_wait();
    pdl_launch_dependents();
    // the rows of this block's pass
    const int pass = a.first_pass + blockIdx.y;
    int row0 = pass * NT, n = min(NT, a.c.rows - row0);
    if (a.c.offsets) {
        // pass p stands for grouped row p and works where a pass of its group begins
        row0 = pass;
        for (int e = tid; e < a.w.experts; e += FR_THREADS) {
            const int b = max(a.c.offsets[e], 0), t = min(a.c.offsets[e + 1], a.c.rows);
            if (row0 >= b && row0 < t && (row0 - b) % NT == 0) { s_find[0] = e; s_find[1] = t; }
        }
        __syncthreads();
        const int expert = s_find[0];
        if (expert < 0) return;                          // the same in every block of the cluster
        n = min(NT, s_find[1] - row0);
        src += (size_t)expert * a.w.row_tiles * a.w.chunks * MX_TILE_BYTES;
        if (tid == 0)
            for (int k = 0; k < min(a.stages, chunks); k++) {
                mbar_expect_tx(&bar_full[k], MX_TILE_BYTES);
                bulk_load(smem_u32(smem + (size_t)k * MX_TILE_BYTES), src + (size_t)k * MX_TILE_BYTES, MX_TILE_BYTES, smem_u32(&bar_full[k]));
            }
    }
    const int all = a.w.cols / 32, first = chunk0 * 8, live = max(0, min(chunks * 8, all - first));
    const size_t pitch = ((size_t)all + 15) / 16 * 16;
    for (int i = tid; i < NT * nb * 4; i += FR_THREADS) {
        const int t = i / (nb * 4), k = i - t * nb * 4, b = k >> 2;      // word k: columns 8 k .. 8 k + 7 of the share
        uint32_t q = 0;
        if (t < n && b < live) q = ((const uint32_t*)(a.c.codes + (size_t)(row0 + t) * (a.w.cols / 2)))[first * 4 + k];
        ((uint2*)(xq + (size_t)(t * 2 + ((k >> 1) & 1)) * nb + b))[k & 1] = make_uint2(four_codes(q), four_codes(q >> 16));
    }
    for (int i = tid; i < NT * nb; i += FR_THREADS) {
        const int t = i / nb, b = i - t * nb;
        xs[i] = t < n && b < live ? 0.25f * scale_value(a.c.scales[(size_t)(row0 + t) * pitch + first + b]) : 0.f;
    }
    __syncthreads();

    volatile int* fail = &s_fail;
    const int c = lane & 7;                              // block of 32 columns within a chunk
    int r[4];
    uint32_t at_code[4], at_scale[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r[i] = warp * 16 + i * 4 + (lane >> 3);
        at_code[i] = r[i] * 128 + ((c ^ (r[i] & 7)) << 4);
        at_scale[i] = MX_CODE_BYTES + (c >> 2) * 512 + (r[i] & 31) * 16 + (r[i] >> 5) * 4 + (c & 3);
    }
    float acc[4][NT];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = 0.f;
    bool ok = true;
    int s = 0, requested = min(a.stages, chunks);        // thread 0 counts
    uint32_t ph = 0;
    for (int kc = 0; kc < chunks; kc++) {
        const uint8_t* st = smem + (size_t)s * MX_TILE_BYTES;
        ok = ok && mbar_wait(&bar_full[s], ph, fail);
        if (__any_sync(0xffffffffu, !ok)) break;
        uint4 q[4];
        float wv[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = *(const uint4*)(st + at_code[i]);
            wv[i] = scale_value(st[at_scale[i]]);
        }
        __syncwarp();
        if (kc + a.stages < chunks) {                    // this warp is done with the stage; the last one's arrival refills it
            if (lane == 0) mbar_arrive(&bar_free[s]);
            if (tid == 0) {
                if (mbar_wait(&bar_free[s], ph, fail)) {
                    mbar_expect_tx(&bar_full[s], MX_TILE_BYTES);
                    bulk_load(smem_u32(st), src + (size_t)(kc + a.stages) * MX_TILE_BYTES, MX_TILE_BYTES, smem_u32(&bar_full[s]));
                    requested++;
                }
            }
            __syncwarp();
        }
        const int b = kc * 8 + c;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t cw[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
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
                acc[i][t] = __fmaf_rn((float)d * xs[t * nb + b], wv[i], acc[i][t]);
            }
        }
        if (++s == a.stages) { s = 0; ph ^= 1u; }
    }
    // eight lanes hold parts of a row
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int d = 4; d; d >>= 1) acc[i][t] += __shfl_xor_sync(0xffffffffu, acc[i][t], d);
            if (c == 0) part[t * MX_TILE_ROWS + r[i]] = acc[i][t];
        }
    if (a.cluster > 1) cg::this_cluster().sync();
    else __syncthreads();
    // Results: pairs of stored rows, spread over the cluster; the ranks' parts are added in their order.
    const cg::cluster_group cluster = cg::this_cluster();
    for (int i = rank * FR_THREADS + tid; i < NT * MX_TILE_ROWS / 2; i += a.cluster * FR_THREADS) {
        const int t = i / (MX_TILE_ROWS / 2), p = i - t * (MX_TILE_ROWS / 2);
        float2 v = make_float2(0.f, 0.f);
        for (int k = 0; k < a.cluster; k++) {
            const float2 o = *(const float2*)((a.cluster > 1 ? cluster.map_shared_rank(part, k) : part) + t * MX_TILE_ROWS + 2 * p);
            v.x += o.x;
            v.y += o.y;
        }
        const int row = tile * MX_TILE_ROWS + 2 * p;
        if (t >= n || row >= a.w.stored_rows) continue;
        const size_t o = (size_t)(row0 + t) * a.c.y_stride;
        if (a.w.activation) {
            store_float(a.c.y, a.c.y_type, o + (row >> 1), gate_act(a.w.activation, v.x) * v.y);
        } else {
            store_float(a.c.y, a.c.y_type, o + row, v.x);
            if (row + 1 < a.w.stored_rows) store_float(a.c.y, a.c.y_type, o + row + 1, v.y);
        }
    }
    if (tid == 0 && *fail) {                             // bounded, too: no copy may land after the block has left
        int none = 0;
        for (int k = max(0, requested - a.stages); k < requested; k++) (void)mbar_wait(&bar_full[k % a.stages], (k / a.stages) & 1, &none);
        atomicOr(a.w.status, SB_ERR_TIMEOUT);
    }
    if (a.cluster > 1) cg::this_cluster().sync();        // a block's parts are read by the others until here
}

template <int NT> cudaError_t launch(FewRowsArgs a, cudaStream_t stream) {
    const int sms = device_sms();
    const int passes = a.c.offsets ? a.c.rows : (a.c.rows + NT - 1) / NT;
    // blocks that have work: of a grouped call, at most a pass per row and per expert and NT rows
    const long long busy = (long long)a.w.row_tiles * (a.c.offsets ? std::min<long long>(a.c.rows, a.w.experts + a.c.rows / NT) : passes);
    a.cluster = 1;
    while (a.cluster < FR_MAX_CLUSTER && a.cluster * 2 <= a.w.chunks && busy * a.cluster < 2 * sms) a.cluster *= 2;
    // The widest rows need a cluster for their bytes alone: 131072 columns of eight rows, 64 chunks each of eight blocks, 147 KB
    while (true) {
        a.share = (a.w.chunks + a.cluster - 1) / a.cluster;
        a.stages = std::min(a.share, 6);
        while (a.stages > 2 && few_rows_smem<NT>(a.share, a.stages) > FR_MAX_SMEM) a.stages--;
        if (few_rows_smem<NT>(a.share, a.stages) <= FR_MAX_SMEM || a.cluster == FR_MAX_CLUSTER) break;
        a.cluster *= 2;
    }
    const size_t smem = few_rows_smem<NT>(a.share, a.stages);
    const void* kernel = (const void*)mxfp4_few_rows_kernel<NT>;
    cudaError_t e;
    if (smem > PLAIN_DYNAMIC_SMEM && (e = ensure_dynamic_smem(kernel, smem)) != cudaSuccess) return e;
    // a launch has at most 65535 blocks along y; the passes beyond follow in launches of their own
    for (int first = 0; first < passes; first += 65535) {
        a.first_pass = first;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.w.row_tiles * a.cluster, std::min(65535, passes - first));
        cfg.blockDim = dim3(FR_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        if ((e = cudaLaunchKernelEx(&cfg, mxfp4_few_rows_kernel<NT>, a)) != cudaSuccess) return e;
        count_launches(1);
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_mxfp4_few_rows(const Mxfp4Weights& w, const Mxfp4Call& c, cudaStream_t stream) {
    FewRowsArgs a = {};
    a.w = w;
    a.c = c;
    // rows of a pass: as many as there are, or as an expert has on average, rounded up
    const int want = c.offsets ? (c.rows + w.experts - 1) / w.experts : c.rows;
    if (want > 4) return launch<8>(a, stream);
    if (want > 2) return launch<4>(a, stream);
    if (want > 1) return launch<2>(a, stream);
    return launch<1>(a, stream);
}

}  // namespace sb
