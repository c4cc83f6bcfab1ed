// Dropout whose mask is drawn from counters and stored nowhere: the backward pass draws the same one again.
#include "typed.h"
#include "rng.h"

namespace {

struct DropoutLaunch {
    const void* x; const void* residual; void* y;
    int ldx, ldr, ldy, cols;
    size_t count;                 // rows * cols
    uint32_t threshold;           // of 65536: an element stays where its 16 bits reach it
    float scale;
    uint64_t seed, stream;
    const uint64_t* stream_offset;
};

// A thread takes groups of eight elements, what one call of the generator decides: 16 bits an element resolve a rate to 1.5e-5, and the 40 quarter-rate multiplications of a
// call are shared by twice as many elements as with the words of rand_f32. VECTOR: groups lie in memory as they are counted (rows without a gap between them, or of a multiple of eight columns) on 16-byte
// boundaries; otherwise element by element.
template <typename T, bool VECTOR> __global__ __launch_bounds__(256) void dropout_kernel(DropoutLaunch a) {
    const T* x = (const T*)a.x; const T* residual = (const T*)a.residual; T* y = (T*)a.y;
    const uint64_t stream = a.stream + *a.stream_offset;
    const size_t groups = (a.count + 7) / 8;
    for (size_t g = (size_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += (size_t)gridDim.x * blockDim.x) {
        const size_t first = g * 8;
        const rlt_u32x4 w = rlt_philox(a.seed, stream, g);
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        const int n = a.count - first < 8 ? (int)(a.count - first) : 8;
        size_t row = first / a.cols; int col = (int)(first - row * a.cols);
        for (int i = 0; i < n; i++) {
            const uint32_t bits = (words[i >> 1] >> (16 * (i & 1))) & 0xffffu;
            float v = bits >= a.threshold ? (float)x[row * a.ldx + col] * a.scale : 0.0f;
            if (residual) v += (float)residual[row * a.ldr + col];
            y[row * a.ldy + col] = (T)v;
            if (++col == a.cols) { col = 0; row++; }
        }
    }
}

template <typename T> void launch(rlt_rocm_device* device, const DropoutLaunch& a) {
    const size_t groups = (a.count + 7) / 8, blocks = (groups + 255) / 256;
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, device->stream, a);
}

}  // namespace

extern "C" int rlt_rocm_dropout(rlt_rocm_device* device, int type, const void* x, int ldx, const void* residual, int ldr, void* y, int ldy, int rows, int cols, float rate,
                                uint64_t seed, uint64_t stream) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE((type == RLT_TYPE_F32 || type == RLT_TYPE_BF16) && x && y && rows > 0 && cols > 0 && ldx >= cols && ldy >= cols && (!residual || ldr >= cols));
    RLT_REQUIRE(rate >= 0.0f && rate <= 1.0f);      // not a NaN either
    DropoutLaunch a = {x, residual, y, ldx, ldr, ldy, cols, (size_t)rows * cols, (uint32_t)(rate * 65536.0f + 0.5f), 0.0f, seed, stream, device->stream_offset};
    a.scale = a.threshold < 65536u ? (float)(65536.0 / (65536.0 - a.threshold)) : 0.0f;
    if (type == RLT_TYPE_F32) launch<float>(device, a); else launch<rlt_bf16>(device, a);
    return rlt_launch_status(device);
}
