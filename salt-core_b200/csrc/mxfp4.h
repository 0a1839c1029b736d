// MXFP4 weights on the device and the launches of their products.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sb {

// Layout made once at creation.  Codes: [experts][stored rows][cols / 2]; a gated pair is stored with its rows alternating (gate
// row i at 2 i, up row i at 2 i + 1), so that the two values an activation needs lie side by side in every kernel.  Scales: per
// 128 stored rows and 128 columns one tile of 512 bytes, the byte of row r and 32-column block k at (r % 32) * 16 + (r / 32) * 4 + k
// (the order in which the tensor core reads them); tiles beyond the last row or column hold 127 = 2^0.
struct Mxfp4Weights {
    int device;
    int rows, cols, experts;     // rows of the result; cols = K
    int stored_rows;             // rows, or 2 rows of a gated pair
    int row_tiles, col_tiles;    // scale tiles of an expert; col_tiles is even
    int activation;              // SALT_B200_ACT_*
    uint8_t* codes;
    uint8_t* scales;
    int* status;
};
struct Mxfp4Handle : Mxfp4Weights { CUtensorMap map; };

struct Mxfp4Call {
    const uint8_t* codes;        // [rows][cols / 2]
    const uint8_t* scales;       // [rows][pitch]
    const int32_t* offsets;      // [experts + 1] or null: one matrix, all rows
    int rows;
    void* y;
    int y_type;
    size_t y_stride;
};

// mxfp4_few_rows.cu: passes of up to eight rows, exact integer sums per block
cudaError_t launch_mxfp4_few_rows(const Mxfp4Weights& w, const Mxfp4Call& c, cudaStream_t stream);

// mxfp4_tensor.cu: block-scaled tensor-core products
cudaError_t make_mxfp4_weight_map(CUtensorMap* out, const Mxfp4Weights& w);
cudaError_t launch_mxfp4_tensor(const Mxfp4Weights& w, const CUtensorMap& weight_map, const Mxfp4Call& c, cudaStream_t stream);

// y = act(gate) * up
__device__ __forceinline__ float gate_act(int activation, float g) {
    if (activation == 2) return g / (1.0f + expf(-g));                                                  // SiLU
    const float t = tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g));                          // GELU, tanh form
    return 0.5f * g * (1.0f + t);
}

}  // namespace sb
