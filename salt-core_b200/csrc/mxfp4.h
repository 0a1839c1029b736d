// MXFP4 weights on the device and the launches of their products.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "mxfp4_passes.h"

namespace sb {

// Layout made once at creation: per 128 stored rows and 256 columns one tile of 17 KB that a single bulk copy brings into shared
// memory as the tensor core reads it, tiles of a row block next to one another.  (Rows of codes side by side, as they come, are 128 separate lines
// of 128 bytes per tile and two kinds of copies.)
//   16384 bytes of codes: row r at r * 128, its 16-byte piece c (one block of 32 columns) at place c ^ (r % 8);
//   1024 bytes of scales: block c of row r at (c / 4) * 512 + (r % 32) * 16 + (r / 32) * 4 + c % 4.
// A gated pair is stored with its rows alternating (gate row i at 2 i, up row i at 2 i + 1), so that the two values an activation
// needs lie side by side in every kernel.  Rows and columns that fill a tile up have codes 0 and scales 127 = 2^0.
// (The sizes are in mxfp4_passes.h.)
struct Mxfp4Weights {
    int device;
    int rows, cols, experts;     // rows of the result; cols = K
    int stored_rows;             // rows, or 2 rows of a gated pair
    int row_tiles, chunks;       // tiles of an expert along rows and columns
    int activation;              // SALT_B200_ACT_*
    uint8_t* tiles;              // [experts][row_tiles][chunks][MX_TILE_BYTES]
    int* status;
};

struct Mxfp4Call {
    const uint8_t* codes;        // [rows][cols / 2]
    const uint8_t* scales;       // [rows][pitch]
    const int32_t* offsets;      // [experts + 1] or null: one matrix, all rows
    int rows;
    void* y;
    int y_type;
    size_t y_stride;
};

// mxfp4_tensor.cu: any number of rows
cudaError_t launch_mxfp4_product(const Mxfp4Weights& w, const Mxfp4Call& c, cudaStream_t stream);

// y = act(gate) * up.  Both activations are g / (1 + exp(-z)): z = g is SiLU, z = 2 sqrt(2 / pi) (g + 0.044715 g^3) the tanh form of GELU.
// With t = exp(-|z|) that is g / (1 + t) above zero and g t / (1 + t) below it: the quotient's divisor lies between 1 and 2, and a gate far
// below zero keeps its bits until the result is too small for 32.  (exp(-z) as it stands grows past 2^126 there, where the fast
// quotient is zero, and the fast exponential is off by |z| units; both together were 0.3 to 1.1 us faster: 64 experts of 1536 x 5120 for
// 1999 tokens 104.9 -> 105.3, 4096 rows of 2560 x 5120 53.1 -> 53.9.)
__device__ __forceinline__ float gate_act(int activation, float g) {
    const float z = activation == 2 ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
    const float t = expf(-fabsf(z));
    float r;                                             // of a number from 1 to 2: one unit off at most, nothing to flush
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + t));
    return (z < 0.f ? g * t : g) * r;
}

// Bulk copy of a tile (both addresses on 16 bytes, a multiple of 16 bytes) into this block's own shared memory.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(bar)
                 : "memory");
}

}  // namespace sb
