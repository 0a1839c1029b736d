// Routing to experts outside a stack: scores of a row of logits, a bias that balances the experts' load, experts limited to
// the best groups, top-k, weights, and the grouping of the selections by expert.
//
//   s_e = exp(l_e - m) / sum exp(l - m)  or  1 / (1 + exp(-l_e));   key_e = s_e + b_e, or l_e itself where there is no bias
//   (both scores rise with the logit, so the logits order the experts exactly);
//   a group's score is the sum of its best one or two keys; the best groups stay; the best k keys of their experts win,
//   the lowest index among equals; w_e = scale * s_e, divided by the sum over the selected ones on request.
//
// A selection is a whole number, so it may not depend on how a sum was rounded.  Everything is computed in 32 bits first; where
// the key that just won and the one that just lost, or the scores of a group that stays and of one that goes, are closer than the
// rounding errors of both, and where a selected score is too small for 32 bits, the row is done again in 64 bits by the same code (of
// rows of 256 experts one in 8500 with a bias, one in 1100 by groups of two keys without one).  Other weights are quotients of scores in
// 32 bits: 5e-8 off on average, where rounding alone leaves 2e-8 to 3e-8.
//
// One warp per token: lane l holds experts l, l + 32, ...; the running maximum of the top-k is a warp-wide integer reduction of
// order-preserving bit patterns.  Bound by the chain of reductions (two per selected expert), not by memory: 4099 tokens of 256
// experts 8.0 us (plain softmax) and 14.1 us (sigmoid, bias, eight groups; 1.2 of them a row done again); grouping their 32 792 selections
// 7.5 us more, a dozen synchronised phases of one cluster.  One token of 128 experts, routed and grouped in one launch: 4 us.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <float.h>
#include <limits.h>

#include <algorithm>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "pdl.cuh"

namespace cg = cooperative_groups;

namespace sb {
bool cuda_ok(cudaError_t e, const char* what);

namespace {

constexpr int RT_WARPS = 4;              // tokens of a block of the routing kernel
constexpr int RT_FUSED_TOKENS = 16;      // up to here one block routes and groups
constexpr int GR_WARPS = 32;
constexpr int GR_HELD = 8;               // selections of a lane that stay in registers between the two passes
constexpr int GR_CLUSTER = 8;
constexpr int GR_FEW = 512;              // RT_FUSED_TOKENS times the largest top-k
constexpr size_t GR_MAX_SMEM = 200 * 1024;
constexpr int GR_ONE_BLOCK = 2048;       // selections that one block groups by itself
constexpr unsigned FULL = 0xffffffffu;

struct RouteArgs {
    const void* logits;
    int type;
    size_t stride;
    int rows, E, topk, sigmoid, groups, topk_groups, group_top, renormalize;
    float scale;
    const float* bias;
    int32_t* selected;
    float* weights;
};

struct GroupArgs {
    const int32_t* selected;
    int n, E;
    int32_t *offsets, *g2c, *c2g;
    int ordered;                         // a block's selections fit into shared memory in the order of their groups
};

// Bit patterns that order like the values, -0 like +0; 0 is below every finite one and stands for "none".
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Keys as they are compared, by integer reductions over the warp: the largest key and its lowest index.
template <typename S> struct Keys;
template <> struct Keys<float> {
    using K = uint32_t;
    static __device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }     // 2 units
    static __device__ __forceinline__ K of(float v) { return v > -CUDART_INF_F ? ordered(v) : 0u; }     // false for NaN
    static __device__ __forceinline__ float value(K k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
    static __device__ __forceinline__ K best(K k, int e, int& at) {
        const K m = __reduce_max_sync(FULL, k);
        at = (int)__reduce_min_sync(FULL, k == m ? (unsigned)e : 0x7fffffffu);
        return m;
    }
};
template <> struct Keys<double> {
    using K = unsigned long long;
    static __device__ __forceinline__ double quotient(double a, double b) { return a / b; }
    static __device__ __forceinline__ K of(double v) {
        if (!(v > -CUDART_INF)) return 0ull;
        const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
        return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
    }
    static __device__ __forceinline__ double value(K k) {
        return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
    }
    static __device__ __forceinline__ K best(K k, int e, int& at) {
        const unsigned hi = __reduce_max_sync(FULL, (unsigned)(k >> 32));
        const unsigned lo = __reduce_max_sync(FULL, (unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
        const K m = ((K)hi << 32) | lo;
        at = (int)__reduce_min_sync(FULL, k == m ? (unsigned)e : 0x7fffffffu);
        return m;
    }
};

template <typename S> __device__ __forceinline__ S warp_sum(S v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
    return v;
}

// One token by one warp.  False where 32 bits do not decide; the caller then comes again with S = double.
// sh: E keys of this warp's own, used with groups only.
template <int VPT, typename S>
__device__ bool route_token(const RouteArgs& a, const float (&l)[VPT], int token, int lane, void* sh) {
    using Q = Keys<S>;
    using K = typename Q::K;
    constexpr bool wide = sizeof(S) == 8;
    S score[VPT];
    S top_score = 1;                                     // no score is larger
    float m = 0.f;                                       // a score is about exp(l - m) where it is small
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const S x = (S)l[i];
            const S t = exp(x < (S)0 ? x : -x);          // at most 1
            score[i] = Q::quotient(x < (S)0 ? t : (S)1, (S)1 + t);
        }
    } else {
        m = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < VPT; i++) m = fmaxf(m, l[i]);            // fmaxf passes over NaN
        m = Keys<float>::value(__reduce_max_sync(FULL, max(Keys<float>::of(m), 1u)));
        S sum = 0;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            // an infinite logit takes part as the limit would: the infinite ones share the whole
            score[i] = l[i] == m ? (S)1 : (l[i] > -CUDART_INF_F ? exp((S)l[i] - (S)m) : (S)0);
            sum += score[i];
        }
        sum = warp_sum(sum);
        if (sum > (S)0) {
            top_score = (S)1 / sum;
#pragma unroll
            for (int i = 0; i < VPT; i++) score[i] = wide ? score[i] / sum : score[i] * top_score;
        }
    }
    K key[VPT];                                          // 0: this expert cannot be chosen
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int e = lane + 32 * i;
        const bool live = e < a.E && l[i] > -CUDART_INF_F;
        if (a.bias) key[i] = live ? Q::of(score[i] + (S)a.bias[min(e, a.E - 1)]) : 0;
        else key[i] = live ? Q::of((S)l[i]) : 0;
    }
    // Rounding errors of two keys together.  Softmax: a score is off by less than 2e-6 of the largest (its exponential by two units
    // of the last place, the difference before it by |l - m| / 2 units, the sum by 37 additions).  Sigmoid: by 4.2e-7 (exponential
    // and quotient two units each, the sum half a unit).  The bias adds one rounding, below.
    const S slack = wide ? (S)0 : a.sigmoid ? (S)1e-6 : (S)4e-6 * top_score;
    if (a.groups > 1) {
        K* keys = (K*)sh;
        const int per = a.E / a.groups;
        const bool by_logit = !a.bias && a.group_top == 1;           // one key, and the logit orders those
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int e = lane + 32 * i;
            if (e < a.E) keys[e] = (a.bias || by_logit || !key[i]) ? key[i] : Q::of(score[i]);
        }
        __syncwarp();
        // lanes of a group: as many as a power of two allows; each keeps the best two of its share
        int share = 1;
        while (share * 2 * a.groups <= 32) share *= 2;
        const int g = lane / share, sub = lane - g * share;
        K k1 = 0, k2 = 0;
        if (g < a.groups) {
            int at = (g * share) % per + sub;            // each group from another place: groups of 32 would meet in the same banks
            for (int j = sub; j < per; j += share) {
                if (at >= per) at -= per;
                const K k = keys[g * per + at];
                at += share;
                k2 = max(k2, min(k1, k));
                k1 = max(k1, k);
            }
        }
        for (int d = 1; d < share; d <<= 1) {
            const K o1 = __shfl_xor_sync(FULL, k1, d), o2 = __shfl_xor_sync(FULL, k2, d);
            k2 = max(max(k2, o2), min(k1, o1));
            k1 = max(k1, o1);
        }
        __syncwarp();
        K mine = k1;
        S far = 0;                                       // how far the sum may be from that of the exact keys; each is rounded in units
        if (g >= a.groups || sub != 0) mine = 0;         // of its own size, which the sum does not show where two of them cancel
        if (mine) {
            const S x = Q::value(k1);
            far = (S)2 * slack + (S)4e-7 * fabs(x);
            if (a.group_top == 2 && k2) {
                const S y = Q::value(k2);
                far += (S)4e-7 * fabs(y);
                mine = Q::of(x + y);
                mine = max(mine, (K)1);                  // two of the lowest value: no sum in 32 bits, but a group that can stay
            }
        }
        uint32_t stay = 0;                               // bit g: the group stays
        K left = mine;
        for (int r = 0; r < a.topk_groups; r++) {
            int at;
            if (!Q::best(left, g, at)) break;
            stay |= 1u << at;
            if (g == at) left = 0;
        }
        if (!wide && !by_logit) {
            // decided if the least that a staying group can be worth is above the most that any other can
            const float v = mine > 1 ? (float)Q::value(mine) : -FLT_MAX, low = mine > 1 ? v - (float)far : -CUDART_INF_F;
            const bool stays = mine != left;
            const uint32_t l = !stays ? 0xffffffffu : ordered(low > -CUDART_INF_F ? low : -CUDART_INF_F);       // false for NaN
            const float least = Keys<float>::value(__reduce_min_sync(FULL, l));
            if (__any_sync(FULL, left && !(v + (float)far < least))) return false;
        }
        const uint32_t inverse = ((1u << 20) + per - 1) / per;       // e / per for e * per below 2^20
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int e = lane + 32 * i;
            if (e < a.E && !((stay >> (((uint32_t)e * inverse) >> 20)) & 1u)) key[i] = 0;
        }
    }
    uint32_t taken = 0;                                  // bit i: expert lane + 32 i is selected
    K mine = 0, last = 0;
    int at_i = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++)
        if (key[i] > mine) { mine = key[i]; at_i = i; }
    int found = 0;
    for (int r = 0; r <= a.topk; r++) {
        int e;
        const K m = Q::best(mine, lane + 32 * at_i, e);
        if (!m) break;
        if (r == a.topk) {                               // the best expert that was not selected
            if (!wide && a.bias) {
                const S x = Q::value(last), y = Q::value(m);
                if (!(x - y > slack + (S)4e-7 * (fabs(x) + fabs(y)))) return false;
            }
            break;
        }
        last = m;
        found++;
        if ((e & 31) == lane) {
            taken |= 1u << (e >> 5);
            mine = 0;
#pragma unroll
            for (int i = 0; i < VPT; i++)
                if (!((taken >> i) & 1u) && key[i] > mine) { mine = key[i]; at_i = i; }
        }
    }
    if (!wide && (a.bias || (float)Q::value(last) - m < -60.f)) {       // without a bias the last one has the lowest logit
        // A score that 32 bits hold with few bits or not at all can become an ordinary weight, by the sum of the selected ones or by
        // the scale.  Below exp(-800) it is zero in 64 bits, too.
        bool faint = false;
#pragma unroll
        for (int i = 0; i < VPT; i++) faint |= ((taken >> i) & 1u) && score[i] < (S)1e-30 && l[i] - m > -800.f;
        if (__any_sync(FULL, faint)) return false;
    }
    S div = 1;
    if (a.renormalize) {
        S sum = 0;
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if ((taken >> i) & 1u) sum += score[i];
        sum = warp_sum(sum);
        div = sum > (S)0 ? sum : (S)1;
    }
    int32_t* ids = a.selected + (size_t)token * a.topk;
    float* w = a.weights + (size_t)token * a.topk;
    int before = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const uint32_t here = __ballot_sync(FULL, (taken >> i) & 1u);
        if ((taken >> i) & 1u) {
            const int p = before + __popc(here & ((1u << lane) - 1u));
            ids[p] = lane + 32 * i;
            w[p] = (float)((S)a.scale * (score[i] / div));
        }
        before += __popc(here);
    }
    for (int p = found + lane; p < a.topk; p += 32) {
        ids[p] = -1;
        w[p] = 0.0f;
    }
    return true;
}

template <int VPT> __device__ __forceinline__ void route_row(const RouteArgs& a, int token, int lane, void* sh) {
    float l[VPT];
    const size_t row = (size_t)token * a.stride;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int e = lane + 32 * i;
        l[i] = e < a.E ? load_float(a.logits, a.type, row + e) : -CUDART_INF_F;
    }
    if (!route_token<VPT, float>(a, l, token, lane, sh)) {
        __syncwarp();
        route_token<VPT, double>(a, l, token, lane, sh);
    }
}

// Stable counting sort of the selections by expert.  A warp owns a contiguous piece of them and a histogram; the pieces of a
// block's warps, and of a cluster's blocks, follow one another, so positions keep the canonical order inside an expert.
// Selections outside [0, E) belong to no group: their place is -1, and so are the entries behind the last group.
// The lanes of a warp that hold the same expert find one another by setting their bits in a word per expert (the instruction that
// compares all lanes takes 270 cycles a warp where the experts differ: 16.5 us for 32792 selections).
__device__ __forceinline__ uint32_t same_expert(uint32_t* bits, int e, bool ok, int lane) {
    if (ok) atomicOr(bits + e, 1u << lane);
    __syncwarp();
    const uint32_t same = ok ? bits[e] : 0u;
    __syncwarp();
    if (ok) bits[e] = 0;
    return same;                                         // the caller's next __syncwarp lets the words be set again
}

__device__ void group_selections(const GroupArgs& a, uint32_t* hist, int rank, int blocks, bool cluster) {
    using Sums = unsigned long long;                     // low word: of the whole grouping, high word: of this block's part
    __shared__ Sums s_part[32], s_live;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    uint32_t* bits = hist + (warps + warp) * a.E;        // this warp's words
    uint32_t* total = hist + 2 * warps * a.E;            // this block's selections of every expert
    uint32_t* base = total + a.E;                        // where this block's part of the group begins
    uint32_t* local = base + a.E;                        // where it begins among the block's selections
    uint32_t* order = local + a.E;                       // the block's selections in that order: expert << 16 | number in the block
    const int piece = ((a.n + warps * blocks - 1) / (warps * blocks) + 31) & ~31;
    const int w_all = rank * warps + warp;
    const int begin = (int)min((long long)w_all * piece, (long long)a.n);
    const int end = (int)min((long long)begin + piece, (long long)a.n);
    const bool keep = piece <= 32 * GR_HELD;
    const int block_begin = rank * warps * piece;        // read only where the pieces are short
    int held[GR_HELD];
    uint32_t same[GR_HELD];
    for (int i = tid; i < 2 * warps * a.E; i += blockDim.x) hist[i] = 0;
    pdl_wait();                                          // the selections come from the launch before
    pdl_launch_dependents();
#pragma unroll
    for (int j = 0; j < GR_HELD; j++) {
        const int i = begin + 32 * j + lane;
        held[j] = i < end ? a.selected[i] : -1;
        same[j] = 0;
    }
    __syncthreads();
    uint32_t* mine = hist + warp * a.E;
    for (int i0 = begin; i0 < end; i0 += 32 * GR_HELD) {
        if (i0 > begin) {
#pragma unroll
            for (int j = 0; j < GR_HELD; j++) {
                const int i = i0 + 32 * j + lane;
                held[j] = i < end ? a.selected[i] : -1;
            }
        }
#pragma unroll
        for (int j = 0; j < GR_HELD; j++) {
            if (i0 + 32 * j >= end) break;
            const int e = held[j];
            const bool ok = e >= 0 && e < a.E;
            same[j] = same_expert(bits, e, ok, lane);
            if (ok && lane == __ffs(same[j]) - 1) mine[e] += __popc(same[j]);
            __syncwarp();
        }
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += blockDim.x) {        // prefix over the warps
        uint32_t t = 0;
        for (int w0 = 0; w0 < warps; w0 += 8) {
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] = hist[(w0 + j) * a.E + e];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                hist[(w0 + j) * a.E + e] = t;
                t += c[j];
            }
        }
        total[e] = t;
    }
    if (cluster) cg::this_cluster().sync();
    else __syncthreads();
    // offsets of the groups: a thread sums a run of experts, then the threads' sums are scanned
    const int run = (a.E + (int)blockDim.x - 1) / (int)blockDim.x;
    Sums sum = 0;
    for (int j = 0; j < run; j++) {
        const int e = tid * run + j;
        if (e >= a.E) break;
        uint32_t all = 0, before = 0;
        if (cluster) {
#pragma unroll
            for (int b = 0; b < GR_CLUSTER; b++) {
                const uint32_t c = *cg::this_cluster().map_shared_rank(total + e, b);
                if (b < rank) before += c;
                all += c;
            }
        } else {
            all = total[e];
        }
        base[e] = (uint32_t)sum + before;                // still without the experts of the threads before
        local[e] = (uint32_t)(sum >> 32);
        sum += (Sums)total[e] << 32 | all;
    }
    // this block has read the others' totals; it leaves when all have (the wait at the end)
    if (cluster) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    Sums scan = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const Sums o = __shfl_up_sync(FULL, scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 31) s_part[warp] = scan;
    __syncthreads();
    if (warp == 0) {
        Sums p = lane < warps ? s_part[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const Sums o = __shfl_up_sync(FULL, p, d);
            if (lane >= d) p += o;
        }
        if (lane < warps) s_part[lane] = p;
        if (lane == 31) s_live = p;
    }
    __syncthreads();
    const Sums front = scan - sum + (warp ? s_part[warp - 1] : 0ull);
    for (int j = 0; j < run; j++) {
        const int e = tid * run + j;
        if (e >= a.E) break;
        base[e] += (uint32_t)front;
        local[e] += (uint32_t)(front >> 32);
    }
    __syncthreads();
    const uint32_t live = (uint32_t)s_live;
    if (rank == 0) {                                     // block 0: nothing before its part, so base is the offset
        for (int e = tid; e < a.E; e += blockDim.x) a.offsets[e] = (int32_t)base[e];
        if (tid == 0) a.offsets[a.E] = (int32_t)live;
    }
    for (int i0 = begin; i0 < end; i0 += 32 * GR_HELD) {
        if (!keep) {
#pragma unroll
            for (int j = 0; j < GR_HELD; j++) {
                const int i = i0 + 32 * j + lane;
                held[j] = i < end ? a.selected[i] : -1;
            }
        }
#pragma unroll
        for (int j = 0; j < GR_HELD; j++) {
            if (i0 + 32 * j >= end) break;
            const int i = i0 + 32 * j + lane, e = held[j];
            const bool ok = e >= 0 && e < a.E;
            const uint32_t lanes = keep ? same[j] : same_expert(bits, e, ok, lane);
            uint32_t p = 0;
            if (ok) p = mine[e] + __popc(lanes & ((1u << lane) - 1u));       // among the block's selections of this expert
            __syncwarp();
            if (ok) {
                if (a.ordered) order[local[e] + p] = (uint32_t)e << 16 | (uint32_t)(i - block_begin);
                else a.g2c[base[e] + p] = i;
                a.c2g[i] = (int32_t)(base[e] + p);
                if (lane == __ffs(lanes) - 1) mine[e] += __popc(lanes);
            } else if (i < end) {
                a.c2g[i] = -1;
            }
            __syncwarp();
        }
    }
    if (a.ordered) {                                     // out group by group: runs of neighbours instead of single words
        __syncthreads();
        const uint32_t mine_all = (uint32_t)(s_live >> 32);
        for (uint32_t p = tid; p < mine_all; p += blockDim.x) {
            const uint32_t v = order[p], e = v >> 16;
            a.g2c[base[e] + p - local[e]] = block_begin + (int)(v & 0xffffu);
        }
    }
    for (long long p = (long long)live + (long long)rank * blockDim.x + tid; p < a.n; p += (long long)blocks * blockDim.x)
        a.g2c[p] = -1;
    if (cluster) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

__host__ __device__ inline size_t group_smem(int E, int warps) { return (size_t)(2 * warps + 3) * E * sizeof(uint32_t); }
__host__ __device__ inline size_t route_smem(int E, int groups, int warps) {
    return groups > 1 ? (size_t)warps * E * sizeof(unsigned long long) : 0;
}

template <int VPT> __global__ void __launch_bounds__(RT_WARPS * 32) route_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int token = blockIdx.x * RT_WARPS + warp;
    pdl_wait();
    pdl_launch_dependents();
    if (token < a.rows) route_row<VPT>(a, token, lane, smem + route_smem(a.E, a.groups, warp));
}

__global__ void __launch_bounds__(GR_WARPS * 32) group_kernel(const GroupArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const bool cluster = gridDim.x > 1;
    group_selections(a, (uint32_t*)smem, (int)blockIdx.x, (int)gridDim.x, cluster);
}

// Up to 512 selections: a thread per selection, and per expert, counts the selections that come before it.
__device__ void group_few(const GroupArgs& a) {
    __shared__ int s_sel[GR_FEW];
    const int tid = threadIdx.x;
    for (int i = tid; i < a.n; i += blockDim.x) {
        const int e = a.selected[i];
        s_sel[i] = e >= 0 && e < a.E ? e : INT_MAX;      // behind every group
    }
    __syncthreads();
    for (int i = tid; i < a.n; i += blockDim.x) {
        const int e = s_sel[i];
        int p = 0;
        for (int j = 0; j < a.n; j++) p += s_sel[j] < e || (s_sel[j] == e && j < i);
        a.c2g[i] = e == INT_MAX ? -1 : p;
        a.g2c[p] = e == INT_MAX ? -1 : i;
    }
    for (int e = tid; e <= a.E; e += blockDim.x) {
        int p = 0;
        for (int j = 0; j < a.n; j++) p += s_sel[j] < e;
        a.offsets[e] = p;
    }
}

// Few tokens: one block routes them, a warp each, and groups what they selected.
template <int VPT> __global__ void __launch_bounds__(RT_FUSED_TOKENS * 32) route_group_kernel(const RouteArgs a, const GroupArgs g) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (warp < a.rows) route_row<VPT>(a, warp, lane, smem + route_smem(a.E, a.groups, warp));
    __syncthreads();
    group_few(g);
}

template <int VPT> cudaError_t launch_route(const RouteArgs& a, const GroupArgs* g, cudaStream_t stream) {
    cudaError_t e;
    if (g && a.rows <= RT_FUSED_TOKENS && a.rows > 0) {
        const int warps = std::max(a.rows, 4);           // a warp per token; four at least, for the counting
        const size_t smem = route_smem(a.E, a.groups, a.rows);
        if (smem > PLAIN_DYNAMIC_SMEM && (e = ensure_dynamic_smem((const void*)route_group_kernel<VPT>, smem)) != cudaSuccess) return e;
        return launch_pdl(route_group_kernel<VPT>, dim3(1), dim3(warps * 32), smem, stream, a, *g);
    }
    if (a.rows > 0) {
        const size_t smem = route_smem(a.E, a.groups, RT_WARPS);
        e = launch_pdl(route_kernel<VPT>, dim3((a.rows + RT_WARPS - 1) / RT_WARPS), dim3(RT_WARPS * 32), smem, stream, a);
        if (e != cudaSuccess) return e;
    }
    if (!g) return cudaSuccess;
    const int warps = a.E <= 512 ? GR_WARPS : GR_WARPS / 2;          // two words per expert and warp and three tables: at most 140 KB
    GroupArgs ga = *g;
    const int blocks = ga.n > GR_ONE_BLOCK ? GR_CLUSTER : 1;
    const long long held = (ga.n + (long long)warps * blocks - 1) / (warps * blocks);      // of a warp
    const long long part = (held + 31) / 32 * 32 * warps;           // of a block
    size_t smem = group_smem(a.E, warps);
    ga.ordered = part <= 0xffff && smem + part * 4 <= GR_MAX_SMEM;
    if (ga.ordered) smem += part * 4;
    if (smem > PLAIN_DYNAMIC_SMEM && (e = ensure_dynamic_smem((const void*)group_kernel, smem)) != cudaSuccess) return e;
    if (blocks > 1) return launch_pdl_cluster(group_kernel, GR_CLUSTER, dim3(warps * 32), smem, stream, ga);
    return launch_pdl(group_kernel, dim3(1), dim3(warps * 32), smem, stream, ga);
}

}  // namespace
}  // namespace sb

extern "C" int salt_b200_route_experts(const SaltB200RouteSpec* spec, const void* d_logits, int dtype, size_t row_stride, int rows,
                                       const float* d_bias, int32_t* d_selected, float* d_weights, int32_t* d_group_offsets,
                                       int32_t* d_grouped_to_canonical, int32_t* d_canonical_to_grouped, void* stream) {
    using namespace sb;
    if (!spec || !float_type_ok(dtype) || rows < 0) return -1;
    const SaltB200RouteSpec& s = *spec;
    if (s.n_experts < 1 || s.n_experts > 1024 || s.topk < 1 || s.topk > 32 || s.topk > s.n_experts || s.n_groups < 1 ||
        s.n_groups > 32 || s.n_experts % s.n_groups || s.topk_groups < 1 || s.topk_groups > s.n_groups ||
        (s.group_top != 1 && s.group_top != 2) || (s.scoring != SALT_B200_SCORE_SOFTMAX && s.scoring != SALT_B200_SCORE_SIGMOID) ||
        s.topk > s.topk_groups * (s.n_experts / s.n_groups) || !(s.scale >= -3.4e38f && s.scale <= 3.4e38f))
        return -1;
    if ((int64_t)rows * s.topk > (int64_t)1 << 24) return -1;
    const bool group = d_group_offsets || d_grouped_to_canonical || d_canonical_to_grouped;
    if (group && !d_group_offsets) return -1;
    if (rows > 0 && (!d_logits || !d_selected || !d_weights || row_stride < (size_t)s.n_experts ||
                     (uintptr_t)d_logits % float_type_size(dtype) || (group && (!d_grouped_to_canonical || !d_canonical_to_grouped))))
        return -1;
    if (row_stride > (size_t)1 << 40 || ((uintptr_t)d_bias | (uintptr_t)d_selected | (uintptr_t)d_weights | (uintptr_t)d_group_offsets |
                                         (uintptr_t)d_grouped_to_canonical | (uintptr_t)d_canonical_to_grouped) % 4)
        return -1;
    if (rows == 0 && !group) return 0;
    RouteArgs a;
    a.logits = d_logits; a.type = dtype; a.stride = row_stride; a.rows = rows; a.E = s.n_experts; a.topk = s.topk;
    a.sigmoid = s.scoring == SALT_B200_SCORE_SIGMOID; a.groups = s.n_groups; a.topk_groups = s.topk_groups; a.group_top = s.group_top;
    a.renormalize = s.renormalize != 0; a.scale = s.scale; a.bias = d_bias; a.selected = d_selected; a.weights = d_weights;
    if (a.groups == a.topk_groups) a.groups = a.topk_groups = 1;     // every group stays
    GroupArgs g = {d_selected, rows * s.topk, s.n_experts, d_group_offsets, d_grouped_to_canonical, d_canonical_to_grouped, 0};
    const cudaStream_t st = (cudaStream_t)stream;
    const GroupArgs* gp = group ? &g : nullptr;
    cudaError_t e;
    if (a.E <= 32) e = launch_route<1>(a, gp, st);
    else if (a.E <= 64) e = launch_route<2>(a, gp, st);
    else if (a.E <= 128) e = launch_route<4>(a, gp, st);
    else if (a.E <= 256) e = launch_route<8>(a, gp, st);
    else if (a.E <= 512) e = launch_route<16>(a, gp, st);
    else e = launch_route<32>(a, gp, st);
    return cuda_ok(e, "route experts") ? 0 : -1;
}
