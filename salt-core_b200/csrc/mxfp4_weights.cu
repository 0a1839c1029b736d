// MXFP4 weight handles and the entry points of their products.
#include <string.h>

#include <new>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "mxfp4.h"

namespace sb {
bool cuda_ok(cudaError_t e, const char* what);

namespace {

// One expert's matrix (or gated pair) from dense rows of codes and scale bytes into tiles (see Mxfp4Weights).  One thread per 16
// bytes of a tile.
struct TileSource {
    const uint8_t *codes[2], *scales[2];                 // gate and up, or one matrix
    int rows, blocks, parts;                             // blocks = columns / 32
};
__global__ void mxfp4_tiles_kernel(const TileSource s, uint4* tiles, int row_tiles, int chunks) {
    constexpr int PIECES = MX_TILE_BYTES / 16, CODE_PIECES = MX_CODE_BYTES / 16;
    const size_t n = (size_t)row_tiles * chunks * PIECES;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
        const size_t tile = i / PIECES;
        const int piece = (int)(i - tile * PIECES), rt = (int)(tile / chunks), kc = (int)(tile - (size_t)rt * chunks);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (piece < CODE_PIECES) {
            const int r = piece >> 3, k = kc * 8 + ((piece & 7) ^ (r & 7)), row = rt * MX_TILE_ROWS + r;
            const int which = s.parts == 2 ? row & 1 : 0, src = s.parts == 2 ? row >> 1 : row;
            if (src < s.rows && k < s.blocks) v = ((const uint4*)s.codes[which])[(size_t)src * s.blocks + k];
        } else {
            const int at = (piece - CODE_PIECES) * 16;   // four rows 32 apart, four blocks each
            uint8_t b[16];
            for (int j = 0; j < 16; j++) {
                const int r = ((at & 511) >> 4) + 32 * (j >> 2), k = kc * 8 + (at >> 9) * 4 + (j & 3), row = rt * MX_TILE_ROWS + r;
                const int which = s.parts == 2 ? row & 1 : 0, src = s.parts == 2 ? row >> 1 : row;
                b[j] = src < s.rows && k < s.blocks ? s.scales[which][(size_t)src * s.blocks + k] : 127;
            }
            memcpy(&v, b, 16);
        }
        tiles[i] = v;
    }
}

bool on_device(const Mxfp4Weights* w) {
    int dev = -1;
    return cuda_ok(cudaGetDevice(&dev), "device") && dev == w->device;
}

void free_weights(Mxfp4Weights* w) {
    if (w->tiles) cudaFree(w->tiles);
    if (w->status) cudaFree(w->status);
    delete w;
}

bool upload(const SaltB200Mxfp4Spec& s, Mxfp4Weights* w, uint8_t* staged, cudaStream_t stream) {
    const size_t row_bytes = (size_t)s.cols / 2, blocks = (size_t)s.cols / 32;
    const bool gated = s.up_codes != nullptr;
    const size_t pitch = s.scale_row_stride ? s.scale_row_stride : blocks;
    const size_t code_stride = s.expert_code_stride ? s.expert_code_stride : (size_t)s.rows * row_bytes;
    const size_t scale_stride = s.expert_scale_stride ? s.expert_scale_stride : (size_t)s.rows * pitch;
    const size_t code_bytes = (size_t)s.rows * row_bytes, scale_bytes = (size_t)s.rows * blocks;
    TileSource src;
    src.rows = s.rows; src.blocks = (int)blocks; src.parts = gated ? 2 : 1;
    for (int e = 0; e < s.n_experts; e++) {
        for (int which = 0; which < src.parts; which++) {
            uint8_t* codes = staged + which * code_bytes;
            uint8_t* scales = staged + src.parts * code_bytes + which * scale_bytes;
            if (!cuda_ok(cudaMemcpyAsync(codes, (const uint8_t*)(which ? s.up_codes : s.codes) + e * code_stride, code_bytes, cudaMemcpyDefault,
                                         stream),
                         "mxfp4 codes") ||
                !cuda_ok(cudaMemcpy2DAsync(scales, blocks, (const uint8_t*)(which ? s.up_scales : s.scales) + e * scale_stride, pitch, blocks,
                                           s.rows, cudaMemcpyDefault, stream),
                         "mxfp4 scales"))
                return false;
            src.codes[which] = codes;
            src.scales[which] = scales;
        }
        const size_t n = (size_t)w->row_tiles * w->chunks * (MX_TILE_BYTES / 16);
        const unsigned grid = (unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096);
        mxfp4_tiles_kernel<<<grid, 256, 0, stream>>>(src, (uint4*)w->tiles + e * n, w->row_tiles, w->chunks);
        if (!cuda_ok(launched(), "mxfp4 tiles")) return false;
    }
    return cuda_ok(cudaStreamSynchronize(stream), "mxfp4 upload");
}

int product(Mxfp4Weights* w, const uint8_t* codes, const uint8_t* scales, const int32_t* offsets, int rows, void* y, int y_type,
            size_t y_stride, cudaStream_t stream) {
    if (!w || !on_device(w) || rows < 0 || rows > 1 << 30 || !float_type_ok(y_type) || y_stride < (size_t)w->rows || y_stride > (size_t)1 << 40) return -1;
    if (rows == 0) return 0;
    if (!codes || !scales || !y || (uintptr_t)offsets % 4 || (uintptr_t)codes % 16 || (uintptr_t)scales % 16 || (uintptr_t)y % float_type_size(y_type)) return -1;
    Mxfp4Call c;
    c.codes = codes; c.scales = scales; c.offsets = offsets; c.rows = rows; c.y = y; c.y_type = y_type; c.y_stride = y_stride;
    return cuda_ok(launch_mxfp4_product(*w, c, stream), "mxfp4 product") ? 0 : -1;
}

}  // namespace
}  // namespace sb

extern "C" {

int salt_b200_mxfp4_weights_create(const SaltB200Mxfp4Spec* spec, void* stream, void** weights_out) {
    using namespace sb;
    if (!spec || !weights_out) return -1;
    const SaltB200Mxfp4Spec& s = *spec;
    const bool gated = s.up_codes != nullptr;
    if (s.rows < 1 || s.rows > 1 << 24 || s.cols < 32 || s.cols % 32 || s.cols > SALT_B200_MXFP4_MAX_COLS || s.n_experts < 1 ||
        s.n_experts > 1024 || !s.codes || !s.scales || gated != (s.up_scales != nullptr) ||
        (gated ? s.activation != SALT_B200_ACT_GELU_TANH && s.activation != SALT_B200_ACT_SILU : s.activation != SALT_B200_ACT_NONE) ||
        (s.scale_row_stride && s.scale_row_stride < (size_t)s.cols / 32) || s.scale_row_stride > (size_t)1 << 31)
        return -1;
    const size_t pitch = s.scale_row_stride ? s.scale_row_stride : (size_t)s.cols / 32;
    if (s.n_experts > 1 && ((s.expert_code_stride && s.expert_code_stride < (size_t)s.rows * (s.cols / 2)) ||
                            (s.expert_scale_stride && s.expert_scale_stride < (size_t)(s.rows - 1) * pitch + s.cols / 32)))
        return -1;
    int ndev = 0, dev = 0, major = 0;
    if (!cuda_ok(cudaGetDeviceCount(&ndev), "device count") || ndev < 1 || !cuda_ok(cudaGetDevice(&dev), "device") ||
        !cuda_ok(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev), "capability") || major != 10)
        return -1;
    Mxfp4Weights* w = new (std::nothrow) Mxfp4Weights();
    if (!w) return -1;
    w->device = dev; w->rows = s.rows; w->cols = s.cols; w->experts = s.n_experts;
    w->stored_rows = gated ? 2 * s.rows : s.rows;
    w->row_tiles = (w->stored_rows + MX_TILE_ROWS - 1) / MX_TILE_ROWS;
    w->chunks = (s.cols + MX_TILE_COLS - 1) / MX_TILE_COLS;
    w->activation = s.activation;
    uint8_t* staged = nullptr;
    const size_t bytes = (size_t)s.n_experts * w->row_tiles * w->chunks * MX_TILE_BYTES;
    bool ok = cuda_ok(cudaMalloc((void**)&w->tiles, bytes), "mxfp4 tiles") && cuda_ok(cudaMalloc((void**)&w->status, sizeof(int)), "mxfp4 status") &&
              cuda_ok(cudaMalloc((void**)&staged, (size_t)w->stored_rows * (s.cols / 2 + s.cols / 32)), "mxfp4 staging") &&
              cuda_ok(cudaMemsetAsync(w->status, 0, sizeof(int), (cudaStream_t)stream), "mxfp4 status") &&
              upload(s, w, staged, (cudaStream_t)stream);
    if (staged) cudaFree(staged);
    if (!ok) {
        free_weights(w);
        return -1;
    }
    *weights_out = w;
    return 0;
}

int salt_b200_mxfp4_weights_destroy(void* weights) {
    if (!weights) return -1;
    sb::free_weights((sb::Mxfp4Weights*)weights);
    return 0;
}

int salt_b200_mxfp4_matmul(void* weights, const uint8_t* d_codes, const uint8_t* d_scales, int rows, void* d_y, int y_dtype,
                           size_t y_row_stride, void* stream) {
    sb::Mxfp4Weights* w = (sb::Mxfp4Weights*)weights;
    if (!w || w->experts != 1) return -1;
    return sb::product(w, d_codes, d_scales, nullptr, rows, d_y, y_dtype, y_row_stride, (cudaStream_t)stream);
}

int salt_b200_mxfp4_experts(void* weights, const uint8_t* d_codes, const uint8_t* d_scales, const int32_t* d_group_offsets, int rows,
                            void* d_y, int y_dtype, size_t y_row_stride, void* stream) {
    if (!d_group_offsets) return -1;
    return sb::product((sb::Mxfp4Weights*)weights, d_codes, d_scales, d_group_offsets, rows, d_y, y_dtype, y_row_stride,
                       (cudaStream_t)stream);
}

int salt_b200_mxfp4_status(void* weights, void* stream) {
    using namespace sb;
    Mxfp4Weights* w = (Mxfp4Weights*)weights;
    if (!w || !on_device(w)) return -1;
    int status = 0;
    if (!cuda_ok(cudaMemcpyAsync(&status, w->status, sizeof status, cudaMemcpyDeviceToHost, (cudaStream_t)stream), "mxfp4 status") ||
        !cuda_ok(cudaMemsetAsync(w->status, 0, sizeof(int), (cudaStream_t)stream), "mxfp4 status") ||
        !cuda_ok(cudaStreamSynchronize((cudaStream_t)stream), "mxfp4 status"))
        return -1;
    return status ? -1 : 0;
}

}  // extern "C"
