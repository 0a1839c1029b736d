// MXFP4 weight handles and the entry points of their products.
#include <new>

#include "../../include/salt_gpu_b200.h"
#include "float_types.cuh"
#include "internal.h"
#include "mxfp4.h"

namespace sb {
bool cuda_ok(cudaError_t e, const char* what);

namespace {

// Stored rows' scale bytes from row-major order into tiles (see Mxfp4Weights).  One thread per byte of the result.
__global__ void mxfp4_scale_tiles_kernel(const uint8_t* gate, const uint8_t* up, uint8_t* tiles, int rows, int blocks, int row_tiles,
                                         int col_tiles) {
    const size_t n = (size_t)row_tiles * col_tiles * 512;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
        const int in = (int)(i & 511);
        const size_t t = i >> 9;
        const int rt = (int)(t / col_tiles), ct = (int)(t - (size_t)rt * col_tiles);
        const int r = rt * 128 + ((in >> 2) & 3) * 32 + (in >> 4), k = ct * 4 + (in & 3);
        const int src = up ? r >> 1 : r;
        uint8_t s = 127;
        if (src < rows && k < blocks) s = (up && (r & 1) ? up : gate)[(size_t)src * blocks + k];
        tiles[i] = s;
    }
}

bool on_device(const Mxfp4Weights* w) {
    int dev = -1;
    return cuda_ok(cudaGetDevice(&dev), "device") && dev == w->device;
}

void free_weights(Mxfp4Handle* w) {
    if (w->codes) cudaFree(w->codes);
    if (w->scales) cudaFree(w->scales);
    if (w->status) cudaFree(w->status);
    delete w;
}

bool upload(const SaltB200Mxfp4Spec& s, Mxfp4Weights* w, uint8_t* staged, cudaStream_t stream) {
    const size_t row_bytes = (size_t)s.cols / 2, blocks = (size_t)s.cols / 32;
    const bool gated = s.up_codes != nullptr;
    const size_t pitch = s.scale_row_stride ? s.scale_row_stride : blocks;
    const size_t code_stride = s.expert_code_stride ? s.expert_code_stride : (size_t)s.rows * row_bytes;
    const size_t scale_stride = s.expert_scale_stride ? s.expert_scale_stride : (size_t)s.rows * pitch;
    for (int e = 0; e < s.n_experts; e++) {
        for (int which = 0; which < (gated ? 2 : 1); which++) {
            const uint8_t* codes = (const uint8_t*)(which ? s.up_codes : s.codes) + e * code_stride;
            const uint8_t* scales = (const uint8_t*)(which ? s.up_scales : s.scales) + e * scale_stride;
            uint8_t* dst = w->codes + (size_t)e * w->stored_rows * row_bytes + which * row_bytes;
            if (!cuda_ok(cudaMemcpy2DAsync(dst, (gated ? 2 : 1) * row_bytes, codes, row_bytes, row_bytes, s.rows, cudaMemcpyDefault,
                                           stream),
                         "mxfp4 codes") ||
                !cuda_ok(cudaMemcpy2DAsync(staged + which * (size_t)s.rows * blocks, blocks, scales, pitch, blocks, s.rows,
                                           cudaMemcpyDefault, stream),
                         "mxfp4 scales"))
                return false;
        }
        const size_t n = (size_t)w->row_tiles * w->col_tiles * 512;
        const unsigned grid = (unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096);
        mxfp4_scale_tiles_kernel<<<grid, 256, 0, stream>>>(staged, gated ? staged + (size_t)s.rows * blocks : nullptr,
                                                           w->scales + e * n, s.rows, (int)blocks, w->row_tiles, w->col_tiles);
        if (!cuda_ok(launched(), "mxfp4 scale tiles")) return false;
    }
    return cuda_ok(cudaStreamSynchronize(stream), "mxfp4 upload");
}

int product(Mxfp4Handle* w, const uint8_t* codes, const uint8_t* scales, const int32_t* offsets, int rows, void* y, int y_type,
            size_t y_stride, cudaStream_t stream) {
    if (!w || !on_device(w) || rows < 0 || !float_type_ok(y_type) || y_stride < (size_t)w->rows || y_stride > (size_t)1 << 40) return -1;
    if (rows == 0) return 0;
    if (!codes || !scales || !y || (uintptr_t)codes % 16 || (uintptr_t)scales % 16 || (uintptr_t)y % float_type_size(y_type)) return -1;
    Mxfp4Call c;
    c.codes = codes; c.scales = scales; c.offsets = offsets; c.rows = rows; c.y = y; c.y_type = y_type; c.y_stride = y_stride;
    const bool few = rows <= (offsets ? 2 * w->experts : 8);
    return cuda_ok(few ? launch_mxfp4_few_rows(*w, c, stream) : launch_mxfp4_tensor(*w, w->map, c, stream), "mxfp4 product") ? 0 : -1;
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
    Mxfp4Handle* w = new (std::nothrow) Mxfp4Handle();
    if (!w) return -1;
    w->device = dev; w->rows = s.rows; w->cols = s.cols; w->experts = s.n_experts;
    w->stored_rows = gated ? 2 * s.rows : s.rows;
    w->row_tiles = (w->stored_rows + 127) / 128;
    w->col_tiles = (s.cols + 255) / 256 * 2;
    w->activation = s.activation;
    uint8_t* staged = nullptr;
    const size_t codes = (size_t)s.n_experts * w->stored_rows * (s.cols / 2);
    const size_t scales = (size_t)s.n_experts * w->row_tiles * w->col_tiles * 512;
    bool ok = cuda_ok(cudaMalloc((void**)&w->codes, codes), "mxfp4 codes") && cuda_ok(cudaMalloc((void**)&w->scales, scales), "mxfp4 scales") &&
              cuda_ok(cudaMalloc((void**)&w->status, sizeof(int)), "mxfp4 status") &&
              cuda_ok(cudaMalloc((void**)&staged, (size_t)w->stored_rows * (s.cols / 32)), "mxfp4 staging") &&
              cuda_ok(cudaMemsetAsync(w->status, 0, sizeof(int), (cudaStream_t)stream), "mxfp4 status") &&
              upload(s, w, staged, (cudaStream_t)stream) && cuda_ok(make_mxfp4_weight_map(&w->map, *w), "mxfp4 map");
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
    sb::free_weights((sb::Mxfp4Handle*)weights);
    return 0;
}

int salt_b200_mxfp4_matmul(void* weights, const uint8_t* d_codes, const uint8_t* d_scales, int rows, void* d_y, int y_dtype,
                           size_t y_row_stride, void* stream) {
    sb::Mxfp4Handle* w = (sb::Mxfp4Handle*)weights;
    if (!w || w->experts != 1) return -1;
    return sb::product(w, d_codes, d_scales, nullptr, rows, d_y, y_dtype, y_row_stride, (cudaStream_t)stream);
}

int salt_b200_mxfp4_experts(void* weights, const uint8_t* d_codes, const uint8_t* d_scales, const int32_t* d_group_offsets, int rows,
                            void* d_y, int y_dtype, size_t y_row_stride, void* stream) {
    if (!d_group_offsets) return -1;
    return sb::product((sb::Mxfp4Handle*)weights, d_codes, d_scales, d_group_offsets, rows, d_y, y_dtype, y_row_stride,
                       (cudaStream_t)stream);
}

int salt_b200_mxfp4_status(void* weights, void* stream) {
    using namespace sb;
    Mxfp4Handle* w = (Mxfp4Handle*)weights;
    if (!w || !on_device(w)) return -1;
    int status = 0;
    if (!cuda_ok(cudaMemcpyAsync(&status, w->status, sizeof status, cudaMemcpyDeviceToHost, (cudaStream_t)stream), "mxfp4 status") ||
        !cuda_ok(cudaMemsetAsync(w->status, 0, sizeof(int), (cudaStream_t)stream), "mxfp4 status") ||
        !cuda_ok(cudaStreamSynchronize((cudaStream_t)stream), "mxfp4 status"))
        return -1;
    return status;
}

}  // extern "C"
