// The three floating-point types of the device-pointer operators (SALT_B200_F32 / _BF16 / _F16), eight elements at a time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sb {

enum : int { FT_F32 = 0, FT_BF16 = 1, FT_F16 = 2 };
inline bool float_type_ok(int t) { return t >= FT_F32 && t <= FT_F16; }
__host__ __device__ __forceinline__ size_t float_type_size(int t) { return t == FT_F32 ? 4 : 2; }

template <int FT> struct FloatType;
template <> struct FloatType<FT_F32> {
    using T = float;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct FloatType<FT_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float up(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T down(float v) { return __float2bfloat16_rn(v); }
};
template <> struct FloatType<FT_F16> {
    using T = __half;
    static __device__ __forceinline__ float up(T v) { return __half2float(v); }
    static __device__ __forceinline__ T down(float v) { return __float2half_rn(v); }
};

// Eight consecutive elements; p is 16-byte aligned.
template <int FT> __device__ __forceinline__ void load8(const typename FloatType<FT>::T* p, float (&v)[8]) {
    if constexpr (FT == FT_F32) {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 q = *(const uint4*)p;
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (FT == FT_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*(const __half2*)&w[i]);
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
        }
    }
}

template <int FT> __device__ __forceinline__ void store8(typename FloatType<FT>::T* p, const float (&v)[8]) {
    if constexpr (FT == FT_F32) {
        ((float4*)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4*)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (FT == FT_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *(const uint32_t*)&h;
            } else {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *(const uint32_t*)&h;
            }
        }
        *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One element of a type known at run time (the branch is uniform).
__device__ __forceinline__ float load_float(const void* p, int type, size_t i) {
    if (type == FT_F32) return ((const float*)p)[i];
    if (type == FT_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_float(void* p, int type, size_t i, float v) {
    if (type == FT_F32) ((float*)p)[i] = v;
    else if (type == FT_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
    else ((__half*)p)[i] = __float2half_rn(v);
}

}  // namespace sb
