// MXFP4 products on the tensor cores: block-scaled tcgen05.mma.kind::mxf4 (E2M1 codes in both operands, one E8M0 scale per 32
// columns of each, 32-bit accumulation in TMEM), dense or by expert groups.
//
// A unit = 128 stored weight rows (M) times one pass of a group's rows (N, a multiple of 16), K in chunks of 256 columns = one
// 128-byte row of packed codes = four MMAs of K = 64.  Persistent blocks; unit u of the launch goes to block u mod grid, a
// group's row tiles next to one another, so the blocks that work at the same time read the same activations.  Which group a
// unit belongs to is found in a prefix table over the groups' passes, made by every block from the device offsets.
// Four launch forms, by a rule at the launch:
//   passes of up to 96 rows: two blocks per SM, half of TMEM each; what bounds them is HBM (64 experts of 1536 x 5120, gate | up, 16 /
//     31 / 63 rows in each of the 64, 541 to 558 MB: 85 / 89 / 92 us, 6.4 to 6.0 TB/s of 6.5 measured; by passes of up to 128 rows
//     87 / 88 / 91);
//   few units: a cluster of 2 to 8 blocks shares each, K split, and the partial sums meet in distributed shared memory; latency (one
//     row of 4096 x 4096: 7.2 us);
//   longer passes: a pair of SMs (cta_group::2) takes two row tiles of a pass and each loads half of its rows.  Loads from L2
//     bounded one SM per unit (11 TB/s in all: 4096 x 5120 x 5120 55 us, 46.7 in pairs); now the tensor pipe is busy 60 % of the
//     cycles, the rest is the scale copies before each chunk's MMAs, six rounds of units where 5.1 would do, first loads and last stores;
//   the same with one SM per unit, where there is a single row tile.
// Warp roles:
//   warp 9      producer: one bulk copy of the weight tile, codes and scales, which lies in memory as the tensor core reads it, and
//               TMA copies of the rows' codes (boxes of 32 rows, 128-byte swizzle)
//   warps 0-3   scales of the rows: a chunk each in turn, loaded a turn ahead, written to shared memory in the order of a scale tile
//   warp 8      issuer: tcgen05.cp of the chunk's scale tiles to TMEM, then its four MMAs; both run in issue order
//   warps 4-7   epilogue: lane = weight row, column = row of the result; a gated pair's two rows are neighbouring lanes
// Every mbarrier wait is bounded; on expiry the block raises its failure flag, sets SB_ERR_TIMEOUT, waits (bounded) for copies
// and MMAs in flight, frees its TMEM and returns.  The block's and the cluster's barriers have no limit of their own: every warp comes
// to them, those that have given up as well.  Nor has the allocation of TMEM: what holds it does not wait for this block (see the
// launch).
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "mxfp4.h"
#include "mxfp4_passes.h"
#include "pdl.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace sb {
namespace {

constexpr int MT_THREADS = 320;          // warps 0-3 scales, 4-7 epilogue, 8 issuer, 9 producer
constexpr uint32_t MT_SF_STRIDE = 32, MT_SFB = 8;
constexpr int MT_SFB_BYTES = 2048;
constexpr int MT_MAX_STAGES = 8;
constexpr int MT_SMEM = 217 * 1024, MT_SMALL_SMEM = 103 * 1024;

struct MxTensorArgs {
    Mxfp4Weights w;
    Mxfp4Call c;
    int cap;                             // most rows of a pass, a multiple of 16
    int stages, stage_bytes;
    uint32_t tmem_cols, acc_cols;        // columns of TMEM, and of one of the two accumulators at its start
    int staged;                          // results go through shared memory behind the ring
    int split, share;                    // blocks of a cluster that share a unit, and most of its chunks that one takes
};

// kind::mxf4 instruction descriptor: A = B = E2M1, K-major, E8M0 scales, `half` = which two bytes of a scale word the MMA reads.
__device__ __forceinline__ uint32_t mx_idesc(int M, int N, uint32_t half) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | (half << 5) | (half << 30);
}

// PAIR: the instruction works on both SMs of a pair; all tcgen05 instructions of a kernel are of one kind.
template <bool PAIR>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// 32 rows of 16 bytes, unswizzled (8-row groups 128 bytes apart), to four TMEM columns of all four lane quarters; of a pair, each
// SM from its own shared memory.
template <bool PAIR> __device__ __forceinline__ void scale_copy(uint32_t taddr, uint32_t smem) {
    const uint64_t desc = make_desc((smem & 0x3ffffu) >> 4, (128u >> 4) | (1u << 14));
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Arrival at a barrier once everything issued so far is complete; of a pair, at the barriers of both blocks.
template <bool PAIR> __device__ __forceinline__ void mx_commit(uint64_t* bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else umma_commit(bar);
}

// Arrival at the same barrier of another block of the cluster.
__device__ __forceinline__ void remote_arrive(uint64_t* bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %0, %1;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [r];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}
// One lane of a converged warp.  The instructions for copies and MMAs take their operands from the warp's uniform registers: inside
// this election, with operands that are the same in all lanes, they are issued at once; under `lane == 0` the compiler has to
// go through the lanes, and a chunk's four MMAs, six scale copies and commit took 1100 cycles.
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}
// Barrier 1 among the four epilogue warps.
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Unit { int expert, tile, row0, n, N; };   // n rows of the pass, N = n up to a multiple of 16

struct Groups {
    const int *first, *begin;            // [experts + 1] passes before a group and its first row (shared memory); null for one dense matrix
    int experts, rows, cap, tiles;

    __device__ __forceinline__ bool unit(int u, Unit* out) const {
        const int pass = u / tiles;
        out->tile = u - pass * tiles;
        int b = 0, t = rows, e = 0, p = pass;
        if (first) {
            if (pass >= first[experts]) return false;
            int lo = 0, hi = experts;    // first[lo] <= pass < first[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= pass) lo = mid;
                else hi = mid;
            }
            e = lo;
            p = pass - first[e];
            b = begin[e];
            t = min(begin[e + 1], rows);
        }
        const int size = pass_rows(t - b, cap);
        out->expert = e;
        out->row0 = b + p * size;
        out->n = min(size, t - out->row0);
        out->N = (out->n + 15) & ~15;
        return out->n > 0;
    }
    __device__ __forceinline__ bool unit_uniform(int u, Unit* out) const {   // by a whole warp
        const bool ok = uniform(unit(u, out));
        out->expert = uniform(out->expert); out->tile = uniform(out->tile); out->row0 = uniform(out->row0);
        out->n = uniform(out->n); out->N = uniform(out->N);
        return ok;
    }
};

template <int FT, bool GATED, bool PAIR>
__global__ void __launch_bounds__(MT_THREADS, 2) mxfp4_tensor_kernel(const MxTensorArgs a, const __grid_constant__ CUtensorMap xmap) {
    using T = typename FloatType<FT>::T;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_free[MT_MAX_STAGES], bar_full[MT_MAX_STAGES], bar_sf[MT_MAX_STAGES], bar_peer[MT_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_done[2], bar_accfree[2], bar_drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ int s_first[1025], s_begin[1025];         // passes before a group, where it begins
    __shared__ int s_part[MT_THREADS / 32];

    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    uint8_t* stage_base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    volatile int* fail = &s_fail;
    if (tid == 0) {
        for (int s = 0; s < a.stages; s++) {
            mbar_init(&bar_free[s], 1);
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_sf[s], 1);
            mbar_init(&bar_peer[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&bar_done[b], 1);
            mbar_init(&bar_accfree[b], PAIR ? 8 : 4);
        }
        mbar_init(&bar_drain, 1);
        s_fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(a.tmem_cols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(a.tmem_cols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    // A dense product's weights do not wait for the launch before: the producer asks for them first.
    if (a.c.offsets) {
        pdl_wait();
        pdl_launch_dependents();
        // passes before every group: a thread sums a run of groups, then the threads' sums are scanned
        const int run = (a.w.experts + MT_THREADS - 1) / MT_THREADS;
        int sum = 0;
        for (int j = 0; j < run; j++) {
            const int e = tid * run + j;
            if (e >= a.w.experts) break;
            const int b = max(a.c.offsets[e], 0), t = a.c.offsets[e + 1], n = min(t, a.c.rows) - b;
            s_begin[e] = b;
            if (e == a.w.experts - 1) s_begin[e + 1] = t;
            s_first[e] = sum;
            if (n > 0) {
                const int size = pass_rows(n, a.cap);
                sum += (n + size - 1) / size;
            }
        }
        int scan = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= d) scan += o;
        }
        if (lane == 31) s_part[warp] = scan;
        __syncthreads();
        int front = scan - sum;
        for (int i = 0; i < warp; i++) front += s_part[i];
        for (int j = 0; j < run; j++) {
            const int e = tid * run + j;
            if (e >= a.w.experts) break;
            s_first[e] += front;
        }
        if (tid == MT_THREADS - 1) s_first[a.w.experts] = front + sum;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) cg::this_cluster().sync();                 // the other block's barriers and TMEM are there
    else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = (uint32_t)uniform((int)s_tmem);
    Groups groups;
    groups.first = a.c.offsets ? s_first : nullptr;
    groups.begin = s_begin; groups.experts = a.w.experts; groups.rows = a.c.rows; groups.cap = a.cap;
    groups.tiles = PAIR ? (a.w.row_tiles + 1) / 2 : a.w.row_tiles;   // of a pair, a unit is two tiles
    const int size = pass_rows(a.c.rows, a.cap);
    const int units = (a.c.offsets ? s_first[a.w.experts] : (a.c.rows + size - 1) / size) * groups.tiles;
    const int cluster_size = PAIR ? 2 : a.split;
    const int rank = (int)(blockIdx.x % cluster_size), first_unit = (int)blockIdx.x / cluster_size, unit_step = (int)gridDim.x / cluster_size;
    const int kc0 = PAIR ? 0 : rank * a.share, kc1 = PAIR ? a.w.chunks : min(a.w.chunks, kc0 + a.share);
    const int sfb_off = a.stage_bytes - MT_SFB_BYTES;    // a stage: weight tile, rows' codes, rows' scales

    const uint32_t stage0 = (uint32_t)uniform((int)smem_u32(stage_base));
    uint32_t produced = 0;
    if (warp == 9) {
        // ================= producer =================
        uint32_t s = 0, ph = 1;                          // a fresh barrier's previous phase counts as complete
        bool ok = true, waited = a.c.offsets != nullptr;
        for (int u = first_unit; u < units && ok; u += unit_step) {
            Unit un;
            if (!groups.unit_uniform(u, &un)) continue;
            // of a pair, each block brings its own tile (the last one twice where they are odd) and half of the rows
            const int half = PAIR ? un.N / 2 : un.N, row0 = un.row0 + (PAIR ? rank * half : 0);
            const int boxes = (half + MT_BOX - 1) / MT_BOX;
            const uint32_t tx = MX_TILE_BYTES + boxes * (MT_BOX * MT_CHUNK);
            const int tile_at = PAIR ? min(2 * un.tile + rank, a.w.row_tiles - 1) : un.tile;
            const uint8_t* tile = a.w.tiles + ((size_t)un.expert * a.w.row_tiles + tile_at) * a.w.chunks * MX_TILE_BYTES;
            int early = kc0;                             // weights of the chunks below have been asked for
            if (!waited) {
                early = min(kc1, kc0 + a.stages);
                if (elected())
                    for (int k = 0; k < early - kc0; k++) {
                        mbar_expect_tx(&bar_full[k], tx);
                        bulk_load(stage0 + k * a.stage_bytes, tile + (size_t)(kc0 + k) * MX_TILE_BYTES, MX_TILE_BYTES, smem_u32(&bar_full[k]));
                    }
                __syncwarp();
                pdl_wait();
                pdl_launch_dependents();
                waited = true;
            }
            for (int kc = kc0; kc < kc1; kc++, produced++) {
                ok = mbar_wait(&bar_free[s], ph, fail);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (elected()) {
                    const uint32_t dst = stage0 + s * a.stage_bytes;
                    if (kc >= early) {
                        mbar_expect_tx(&bar_full[s], tx);
                        bulk_load(dst, tile + (size_t)kc * MX_TILE_BYTES, MX_TILE_BYTES, smem_u32(&bar_full[s]));
                    }
                    for (int b = 0; b < boxes; b++)
                        tma_load_2d(dst + MX_TILE_BYTES + b * (MT_BOX * MT_CHUNK), &xmap, kc * MT_CHUNK, row0 + b * MT_BOX, &bar_full[s]);
                }
                __syncwarp();
                if (++s == (uint32_t)a.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (PAIR && warp == 8 && rank == 1) {
        // ================= second block of a pair: its stages, reported to the first =================
        uint32_t s = 0, ph = 0;
        bool ok = true;
        if (!a.c.offsets) {
            pdl_wait();
            pdl_launch_dependents();
        }
        for (int u = first_unit; u < units && ok; u += unit_step) {
            Unit un;
            if (!groups.unit_uniform(u, &un)) continue;
            for (int kc = kc0; kc < kc1 && ok; kc++) {
                ok = __all_sync(0xffffffffu, mbar_wait2(&bar_full[s], ph, &bar_sf[s], ph, fail));
                if (ok && lane == 0) remote_arrive(&bar_peer[s], 0);
                __syncwarp();
                if (++s == (uint32_t)a.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 8) {
        // ================= issuer =================
        uint32_t s = 0, ph = 0, done = 0, par = 0, ready = 0;
        bool ok = true;
        if (!a.c.offsets) {
            pdl_wait();
            pdl_launch_dependents();
        }
        for (int u = first_unit; u < units && ok; u += unit_step) {
            Unit un;
            if (!groups.unit_uniform(u, &un)) continue;
            const uint32_t buf = done & 1u;
            if (done >= 2u)
                ok = __all_sync(0xffffffffu, mbar_wait(&bar_accfree[buf], ((done >> 1) - 1) & 1, fail));
            const uint32_t id0 = mx_idesc(PAIR ? 256 : 128, un.N, 0), id1 = mx_idesc(PAIR ? 256 : 128, un.N, 1);
            const uint32_t d = tmem + buf * a.acc_cols;
            for (int kc = kc0; kc < kc1 && ok; kc++) {
                if (!ready) ok = __all_sync(0xffffffffu, mbar_wait2(&bar_full[s], ph, &bar_sf[s], ph, fail));
                if (PAIR && !ready && ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar_peer[s], ph, fail));
                if (!ok) break;
                // The next stage's barriers are asked before this stage's MMAs go out: an answer takes some 130 cycles.  (Asking two
                // stages ahead, to copy the next chunk's scales before this chunk's MMAs, cost more than it hid: 46.7 -> 49.8 us.)
                const uint32_t ns = s + 1 == (uint32_t)a.stages ? 0 : s + 1, nph = ns ? ph : ph ^ 1u;
                const uint32_t r_full = mbar_test(&bar_full[ns], nph), r_sf = mbar_test(&bar_sf[ns], nph), r_peer = PAIR ? mbar_test(&bar_peer[ns], nph) : 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t st = stage0 + s * a.stage_bytes;
                const uint32_t sf = tmem + 2 * a.acc_cols + par * MT_SF_STRIDE;
                par ^= 1u;
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        scale_copy<PAIR>(sf + 4 * k, st + MX_CODE_BYTES + k * 512);
                        scale_copy<PAIR>(sf + MT_SFB + 8 * k, st + sfb_off + k * 1024);
                        if (un.N > 128) scale_copy<PAIR>(sf + MT_SFB + 8 * k + 4, st + sfb_off + k * 1024 + 512);
                    }
                    const uint32_t alo = DESC_B_LO | ((st & 0x3ffffu) >> 4), blo = alo + (MX_TILE_BYTES >> 4);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mx_mma<PAIR>(d, make_desc(alo + j * 2, DESC_B_HI), make_desc(blo + j * 2, DESC_B_HI), (j & 1) ? id1 : id0,
                               sf + 4 * (j >> 1), sf + MT_SFB + 8 * (j >> 1), (kc > kc0 || j > 0) ? 1u : 0u);
                    mx_commit<PAIR>(&bar_free[s]);
                    if (kc == kc1 - 1) mx_commit<PAIR>(&bar_done[buf]);
                }
                __syncwarp();
                ready = __all_sync(0xffffffffu, r_full & r_sf & r_peer);
                s = ns;
                ph = nph;
            }
            done++;
        }
    } else if (warp < 4) {
        // ================= scales of the rows =================
        if (!a.c.offsets) {
            pdl_wait();
            pdl_launch_dependents();
        }
        // Warp w takes every fourth chunk (of fewer stages than four, as many warps as stages take turns: a barrier's parity tells
        // only the last two rounds of a stage apart, and a warp must not look further ahead); lane l holds the scales of rows l,
        // l + 32, ...: eight bytes of each per chunk, which lie in a scale tile as the words of one 16-byte store.  (All four warps on every chunk, a row or two a thread, took 670 cycles
        // a chunk and were what the issuer waited for.)
        constexpr int GROUPS = MT_MAX_N / 32;
        const int blocks = a.w.cols / 32;
        const size_t pitch = ((size_t)blocks + 15) / 16 * 16;
        const int step = min(4, a.stages);
        uint32_t position = 0, s = 0, ph = 1;            // position: chunks of the units before
        bool ok = warp < step;
        for (int u = first_unit; u < units && ok; u += unit_step) {
            Unit un;
            if (!groups.unit_uniform(u, &un)) continue;
            const uint8_t* base = a.c.scales + (size_t)(un.row0 + lane) * pitch;
            uint2 next[GROUPS];
            int kc = kc0 + (warp + step - (int)(position % step)) % step;    // this warp's first chunk of the unit
#pragma unroll
            for (int j = 0; j < GROUPS; j++)
                if (lane + 32 * j < un.n && kc < kc1) next[j] = *(const uint2*)(base + (size_t)(32 * j) * pitch + kc * 8);
                else next[j] = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
            s += (uint32_t)(kc - kc0);
            while (s >= (uint32_t)a.stages) { s -= a.stages; ph ^= 1u; }
            for (; kc < kc1 && ok; kc += step) {
                uint32_t lo[8], hi[8];                   // blocks 0..3 and 4..7 of the lane's rows; row group 7 does not exist
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    lo[j] = j < GROUPS ? next[j < GROUPS ? j : 0].x : 0u;
                    hi[j] = j < GROUPS ? next[j < GROUPS ? j : 0].y : 0u;
                }
                if (kc * 8 + 8 > blocks) {               // blocks behind the last column read as 2^0
                    const int left = blocks - kc * 8;
                    const uint32_t keep0 = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
                    const uint32_t keep1 = left > 4 ? (1u << (8 * (left - 4))) - 1u : 0u;
#pragma unroll
                    for (int j = 0; j < GROUPS; j++) {
                        lo[j] = (lo[j] & keep0) | (0x7f7f7f7fu & ~keep0);
                        hi[j] = (hi[j] & keep1) | (0x7f7f7f7fu & ~keep1);
                    }
                }
#pragma unroll
                for (int j = 0; j < GROUPS; j++)
                    if (lane + 32 * j < un.n && kc + step < kc1) next[j] = *(const uint2*)(base + (size_t)(32 * j) * pitch + (kc + step) * 8);
                ok = __all_sync(0xffffffffu, mbar_wait(&bar_free[s], ph, fail));
                if (ok) {
                    uint4* sfb = (uint4*)(stage_base + s * a.stage_bytes + sfb_off) + lane;
                    sfb[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    sfb[64] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (un.N > 128) {
                        sfb[32] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                        sfb[96] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_sf[s]);  // always: the issuer never waits for a warp that gave up
                s += step;
                while (s >= (uint32_t)a.stages) { s -= a.stages; ph ^= 1u; }
            }
            // on to the stage of the next unit's first chunk
            position += kc1 > kc0 ? (uint32_t)(kc1 - kc0) : 0u;
            s = position % a.stages;
            ph = 1u ^ ((position / a.stages) & 1u);
        }
    } else {
        // ================= epilogue (TMEM lane quarter warp - 4) =================
        constexpr int WIDTH = MX_TILE_ROWS / (GATED ? 2 : 1);        // results of a tile per row
        const int q = warp - 4;
        const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16);
        uint32_t done = 0;
        bool ok = true;
        if (!a.c.offsets) {
            pdl_wait();
            pdl_launch_dependents();
        }
        int u = first_unit;
        for (; u < units && ok; u += unit_step) {
            Unit un;
            if (!groups.unit(u, &un)) continue;
            if (kc0 >= kc1) continue;                    // this block of the cluster has no chunks
            const int m = (PAIR ? 2 * un.tile + rank : un.tile) * 128 + q * 32 + lane;
            const bool live = m < a.w.stored_rows;
            // A store per row of the result writes 64 bytes a warp and takes some nine cycles of the SM; 16 bytes a lane, of rows that
            // lie together in shared memory, are four times less of them.
            const bool stage_out = PAIR && a.staged && m - q * 32 - lane + MX_TILE_ROWS <= a.w.stored_rows;
            const uint32_t buf = done & 1u;
            ok = mbar_wait(&bar_done[buf], (done >> 1) & 1, fail);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int n0 = 0; n0 < un.N; n0 += 32) {
                uint32_t acc[32];
                tmem_ld32(trow + buf * a.acc_cols + n0, acc);
                if (!PAIR && a.split > 1) {
                    // the ring is idle after a cluster's only unit: partial sums [row of the result][128] go there
                    float* part = (float*)stage_base + n0 * MX_TILE_ROWS + q * 32 + lane;
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (n0 + k < un.N) part[k * MX_TILE_ROWS] = __uint_as_float(acc[k]);
                } else {
                    T out[32];                           // of a gated pair 16
                    const bool odd = lane & 1;
                    if (GATED) {
                        // lanes 2 i and 2 i + 1 hold gate and up of the same result: the even lane takes even rows, the odd lane odd ones
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const float mine = __uint_as_float(odd ? acc[2 * k + 1] : acc[2 * k]);
                            const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(odd ? acc[2 * k] : acc[2 * k + 1]), 1);
                            out[k] = FloatType<FT>::down(gate_act(a.w.activation, odd ? other : mine) * (odd ? mine : other));
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k++) out[k] = FloatType<FT>::down(__uint_as_float(acc[k]));
                    }
                    if (stage_out) {
                        T* slab = (T*)(stage_base + a.stages * a.stage_bytes);
                        epilogue_sync();                 // the slab before this one has been stored
#pragma unroll
                        for (int k = 0; k < (GATED ? 16 : 32); k++)
                            if (GATED) slab[(2 * k + odd) * WIDTH + (q * 32 + lane) / 2] = out[k];
                            else slab[k * WIDTH + q * 32 + lane] = out[k];
                        epilogue_sync();
                        constexpr int PIECES = WIDTH * (int)sizeof(T) / 16;
                        T* y = (T*)a.c.y + (size_t)(un.row0 + n0) * a.c.y_stride + (m - q * 32 - lane) / (GATED ? 2 : 1);
                        const int pieces = min(32, un.n - n0) * PIECES;
                        for (int i = q * 32 + lane; i < pieces; i += 128) {
                            const int r = i / PIECES, c = i % PIECES;
                            ((uint4*)(y + (size_t)r * a.c.y_stride))[c] = ((const uint4*)(slab + r * WIDTH))[c];
                        }
                        __syncwarp();
                    } else {
                        T* y = (T*)a.c.y + (size_t)(un.row0 + n0 + (GATED && odd)) * a.c.y_stride + (GATED ? m >> 1 : m);
                        const int left = live ? un.n - n0 - (GATED && odd) : 0;      // rows below it exist
                        constexpr int STEP = GATED ? 2 : 1;
                        if (left > 32 - STEP) {          // all of them: no branch between the stores
#pragma unroll
                            for (int k = 0; k < 32 / STEP; k++) y[(size_t)(STEP * k) * a.c.y_stride] = out[k];
                        } else {
#pragma unroll
                            for (int k = 0; k < 32 / STEP; k++)
                                if (STEP * k < left) y[(size_t)(STEP * k) * a.c.y_stride] = out[k];
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (PAIR) remote_arrive(&bar_accfree[buf], 0);       // the first block's own as well
                else mbar_arrive(&bar_accfree[buf]);
            }
            done++;
        }
        // Where results meet in shared memory a warp that has given up still comes to every barrier that the others may wait at, from
        // the unit that it broke off.  (Four warps that agree at a barrier with a reduction cost 2 us of 63.)
        if (PAIR && !ok && a.staged)
            for (; u < units; u += unit_step) {
                Unit un;
                if (!groups.unit(u, &un) || (2 * un.tile + rank + 1) * MX_TILE_ROWS > a.w.stored_rows) continue;
                for (int n0 = 0; n0 < un.N; n0 += 32) {
                    epilogue_sync();
                    epilogue_sync();
                }
            }
    }

    if (!PAIR && a.split > 1) {
        // The cluster's partial sums, added in rank order; the rows of the result are dealt out to its blocks.
        const cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        Unit un;
        if (first_unit < units && groups.unit(first_unit, &un)) {
            const int live = (a.w.chunks + a.share - 1) / a.share;
            constexpr int PIECES = MX_TILE_ROWS / 4;     // four stored rows at a time; all blocks' parts are asked for at once
            for (int i = rank * MT_THREADS + tid; i < un.n * PIECES; i += a.split * MT_THREADS) {
                const int n = i / PIECES, p = i - n * PIECES, m = un.tile * MX_TILE_ROWS + 4 * p;
                float4 o[MT_MAX_SPLIT];
#pragma unroll
                for (int k = 0; k < MT_MAX_SPLIT; k++)
                    if (k < live) o[k] = *(const float4*)(cluster.map_shared_rank((float*)stage_base, k) + n * MX_TILE_ROWS + 4 * p);
                float v[4] = {o[0].x, o[0].y, o[0].z, o[0].w};
#pragma unroll
                for (int k = 1; k < MT_MAX_SPLIT; k++)
                    if (k < live) { v[0] += o[k].x; v[1] += o[k].y; v[2] += o[k].z; v[3] += o[k].w; }
                T* y = (T*)a.c.y + (size_t)(un.row0 + n) * a.c.y_stride;
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    if (GATED) {
                        if (m + j < a.w.stored_rows) y[(m + j) >> 1] = FloatType<FT>::down(gate_act(a.w.activation, v[j]) * v[j + 1]);
                    } else {
                        if (m + j < a.w.stored_rows) y[m + j] = FloatType<FT>::down(v[j]);
                        if (m + j + 1 < a.w.stored_rows) y[m + j + 1] = FloatType<FT>::down(v[j + 1]);
                    }
                }
            }
        }
        cluster.sync();                                  // a block's sums are read by the others until here
    }
    __syncthreads();
    if (*fail) {
        if (tid == 0) atomicOr(a.w.status, SB_ERR_TIMEOUT);
        // wait (bounded, no early exit) for the copies requested and the MMAs issued before TMEM and shared memory are released
        if (warp == 9 && lane == 0) {
            int none = 0;
            const uint32_t n = (uint32_t)a.stages;
            for (uint32_t t = produced > n ? produced - n : 0; t < produced; t++) (void)mbar_wait(&bar_full[t % n], (t / n) & 1, &none);
        }
        __syncthreads();
        if (warp == 8 && (!PAIR || rank == 0) && elected()) {        // the lane that issued the MMAs: a commit covers its own only
            int none = 0;
            if (PAIR)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&bar_drain)) : "memory");
            else umma_commit(&bar_drain);
            (void)mbar_wait(&bar_drain, 0, &none);
        }
        __syncthreads();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) cg::this_cluster().sync();                 // neither block leaves while the other's MMAs read its shared memory
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
    }
}

using Kernel = void (*)(const MxTensorArgs, const CUtensorMap);
template <bool GATED, bool PAIR> Kernel pick_kernel(int type) {
    return type == FT_F32 ? mxfp4_tensor_kernel<FT_F32, GATED, PAIR> : type == FT_BF16 ? mxfp4_tensor_kernel<FT_BF16, GATED, PAIR>
                                                                                       : mxfp4_tensor_kernel<FT_F16, GATED, PAIR>;
}
Kernel pick_kernel(bool gated, int type, bool pair) {
    return gated ? (pair ? pick_kernel<true, true>(type) : pick_kernel<true, false>(type))
                 : (pair ? pick_kernel<false, true>(type) : pick_kernel<false, false>(type));
}

}  // namespace

cudaError_t launch_mxfp4_product(const Mxfp4Weights& w, const Mxfp4Call& c, cudaStream_t stream) {
    TensorMapEncodeFn encode = nullptr;
    cudaError_t e = tensor_map_encoder(&encode);
    if (e != cudaSuccess) return e;
    CUtensorMap xmap;
    cuuint64_t dims[2] = {(cuuint64_t)w.cols / 2, (cuuint64_t)c.rows}, strides[1] = {(cuuint64_t)w.cols / 2};
    cuuint32_t box[2] = {(cuuint32_t)MT_CHUNK, (cuuint32_t)MT_BOX}, estr[2] = {1, 1};
    if (encode(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(c.codes), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    MxTensorArgs a;
    a.w = w;
    a.c = c;
    const int sms = device_sms();
    a.cap = choose_cap(c.offsets ? (int)std::min(1.25 * c.rows / w.experts + 8, 1e9) : c.rows, c.offsets ? std::min(c.rows, w.experts) : 1, w.row_tiles,
                       w.chunks, sms);
    a.stage_bytes = MX_TILE_BYTES + a.cap * MT_CHUNK + MT_SFB_BYTES;
    const bool small = a.cap <= MT_SMALL_N;
    a.acc_cols = small ? MT_SMALL_N : MT_MAX_N;
    a.tmem_cols = small ? 256 : 512;
    const long long passes = c.offsets ? std::min<long long>(c.rows, c.rows / a.cap + w.experts) : (c.rows + a.cap - 1) / a.cap;
    const long long units = passes * w.row_tiles;
    if (units > INT32_MAX / 2) return cudaErrorInvalidValue;
    const int half = std::min(MT_MAX_STAGES, (MT_SMALL_SMEM - 1024) / a.stage_bytes);
    a.split = choose_split(units, w.chunks, small ? half : 0, sms);
    a.share = (w.chunks + a.split - 1) / a.split;
    // Two blocks per SM where there is work for them or where half the stages hold all chunks; otherwise one with twice the stages
    const bool pairs = small && (units * a.split > sms || a.share <= half);
    const bool pair = !small && a.split == 1 && w.row_tiles > 1;
    const size_t y_size = float_type_size(c.y_type);
    // Results of pairs of SMs go through shared memory (4096 rows of 5120 x 5120: 48.5 -> 46.7 us); of short passes it costs what it
    // saves (4096 of 5000 x 256: 17.6 and 19.0 us), and of single SMs too (18889 rows of 128 x 1408: 8.1 and 8.5).
    a.staged = pair && (uintptr_t)c.y % 16 == 0 && c.y_stride * y_size % 16 == 0;
    const int slab = a.staged ? MT_BOX * MX_TILE_ROWS / (w.activation ? 2 : 1) * (int)y_size : 0;
    long long turns = 1;                                 // units of a block
    int grid = (int)units * a.split;
    if (pair) {
        const long long two = passes * ((w.row_tiles + 1) / 2);
        a.stage_bytes = MX_TILE_BYTES + (a.cap / 2 + MT_BOX - 1) / MT_BOX * MT_BOX * MT_CHUNK + MT_SFB_BYTES;
        grid = 2 * (int)std::min<long long>(sms / 2, two);
        turns = (two + grid / 2 - 1) / (grid / 2);
    } else if (a.split == 1) {
        grid = (int)std::min<long long>(pairs ? 2 * sms : sms, units);
        turns = (units + grid - 1) / grid;
    }
    // as many stages as fit, but no more than a block has chunks
    const int fit = std::min(MT_MAX_STAGES, ((pairs ? MT_SMALL_SMEM : MT_SMEM) - 1024 - slab) / a.stage_bytes);
    a.stages = (int)std::min<long long>(fit, turns * a.share);
    if (a.split > 1) a.stages = std::max(a.stages, (a.cap * MX_TILE_ROWS * 4 + a.stage_bytes - 1) / a.stage_bytes);    // partial sums
    // Blocks that wait for one another hold TMEM while they do, and one that finds none left waits for it without a limit; of two such
    // groups on the same SMs, each could hold what the other waits for.  None can be: a block of a pair, or of a cluster that takes all
    // of TMEM, comes with long rows only and asks for 167 KB and more of an SM's 228, one of a cluster that takes half of it for 47 and
    // more, and each has 10 KB beside that (the least that the rules above give, over 1.3 million sizes).  A rule that changes this must
    // ask for more here.
    const size_t smem = (size_t)a.stages * a.stage_bytes + slab + 1024;
    const auto kernel = pick_kernel(w.activation != 0, c.y_type, pair);
    if ((e = ensure_dynamic_smem((const void*)kernel, smem)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(MT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pair ? 2 : a.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    if ((e = cudaLaunchKernelEx(&cfg, kernel, a, xmap)) == cudaSuccess) count_launches(1);
    return e;
}

}  // namespace sb
