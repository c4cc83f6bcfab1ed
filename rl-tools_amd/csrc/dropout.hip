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

enum Layout { DENSE, ROWS, ELEMENTS };      // groups lie side by side on 16-byte boundaries; within rows of whole groups on such boundaries; anything else
constexpr int UNROLL = 4;

// A group of eight elements is what one call of the generator decides: 16 bits an element resolve a rate to 1.5e-5, and the call's twenty 32 x 32 multiplications are shared by twice as many
// elements as with the words of rand_f32. A thread takes UNROLL groups, the workgroup's thread count apart, all of whose loads are asked for before the first draw. Memory
// bounds it: 32,768 x 4,096 bfloat16 95 us, 5.6 TB/s; 4,001 x 1,023 fp32 with a residual 10.2 us; a launch at 256 x 256, 3.9 us. Rows that neither follow each other
// nor are whole groups go element by element: 4,001 x 1,023 fp32 without a residual, rows 1,040 apart, 16.9 us, where rows of 1,024 take 7.6; bfloat16 14.4.
template <typename T, int LAYOUT> __global__ __launch_bounds__(256) void dropout_kernel(DropoutLaunch a) {
    constexpr int V = 16 / sizeof(T);
    const T* x = (const T*)a.x; const T* residual = (const T*)a.residual; T* y = (T*)a.y;
    const uint64_t stream = a.stream + *a.stream_offset;
    const size_t groups = (a.count + 7) / 8, whole = a.count / 8, first = (size_t)blockIdx.x * (256 * UNROLL) + threadIdx.x;
    if constexpr (LAYOUT != ELEMENTS) {
        float v[UNROLL][8], r[UNROLL][8];
        size_t ax[UNROLL], ar[UNROLL], ay[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; j++) {
            const size_t g = first + j * 256;
            if constexpr (LAYOUT == DENSE) ax[j] = ar[j] = ay[j] = g * 8;
            else {
                const uint32_t per_row = (uint32_t)a.cols / 8, row = (uint32_t)g / per_row, col = ((uint32_t)g - row * per_row) * 8;
                ax[j] = (size_t)row * a.ldx + col; ar[j] = (size_t)row * a.ldr + col; ay[j] = (size_t)row * a.ldy + col;
            }
            if (g < whole) {
#pragma unroll
                for (int i = 0; i < 8; i += V) rlt_load<V>(x + ax[j] + i, v[j] + i);
                if (residual) {
#pragma unroll
                    for (int i = 0; i < 8; i += V) rlt_load<V>(residual + ar[j] + i, r[j] + i);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < UNROLL; j++) {
            const size_t g = first + j * 256;
            const rlt_u32x4 w = rlt_philox(a.seed, stream, g);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            if (g < whole) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t bits = (i & 1) ? words[i >> 1] >> 16 : words[i >> 1] & 0xffffu;
                    v[j][i] = bits >= a.threshold ? v[j][i] * a.scale : 0.0f;
                    if (residual) v[j][i] += r[j][i];
                }
#pragma unroll
                for (int i = 0; i < 8; i += V) rlt_store<V>(y + ay[j] + i, v[j] + i);
            } else if (g < groups) {      // the last group of a dense tensor
                for (int i = 0; g * 8 + i < a.count; i++) {
                    const uint32_t bits = (words[i >> 1] >> (16 * (i & 1))) & 0xffffu;
                    float e = bits >= a.threshold ? (float)x[g * 8 + i] * a.scale : 0.0f;
                    if (residual) e += (float)residual[g * 8 + i];
                    y[g * 8 + i] = (T)e;
                }
            }
        }
    } else {
        for (int j = 0; j < UNROLL; j++) {
            const size_t g = first + j * 256;
            if (g >= groups) break;
            const rlt_u32x4 w = rlt_philox(a.seed, stream, g);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            size_t row = g * 8 / a.cols; int col = (int)(g * 8 - row * a.cols);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (g * 8 + i >= a.count) break;
                const uint32_t bits = (i & 1) ? words[i >> 1] >> 16 : words[i >> 1] & 0xffffu;
                float e = bits >= a.threshold ? (float)x[row * a.ldx + col] * a.scale : 0.0f;
                if (residual) e += (float)residual[row * a.ldr + col];
                y[row * a.ldy + col] = (T)e;
                if (++col == a.cols) { col = 0; row++; }
            }
        }
    }
}

template <typename T> int launch(rlt_rocm_device* device, const DropoutLaunch& a) {
    const size_t blocks = ((a.count + 7) / 8 + 256 * UNROLL - 1) / (256 * UNROLL);
    if (blocks > UINT32_MAX / 256) return RLT_E_UNSUPPORTED;      // 2^32 threads are more than a dimension of a grid holds
    const bool aligned = rlt_vectors<T>(a.x, 0) && rlt_vectors<T>(a.y, 0) && (!a.residual || rlt_vectors<T>(a.residual, 0));
    const bool dense = a.ldx == a.cols && a.ldy == a.cols && (!a.residual || a.ldr == a.cols);
    const bool rows = a.cols % 8 == 0 && rlt_vectors<T>(a.x, a.ldx) && rlt_vectors<T>(a.y, a.ldy) && (!a.residual || rlt_vectors<T>(a.residual, a.ldr)) && a.count / 8 <= UINT32_MAX;
    if (aligned && dense) hipLaunchKernelGGL((dropout_kernel<T, DENSE>), dim3((unsigned)blocks), dim3(256), 0, device->stream, a);
    else if (rows) hipLaunchKernelGGL((dropout_kernel<T, ROWS>), dim3((unsigned)blocks), dim3(256), 0, device->stream, a);
    else hipLaunchKernelGGL((dropout_kernel<T, ELEMENTS>), dim3((unsigned)blocks), dim3(256), 0, device->stream, a);
    return rlt_launch_status(device);
}

}  // namespace

extern "C" int rlt_rocm_dropout(rlt_rocm_device* device, int type, const void* x, int ldx, const void* residual, int ldr, void* y, int ldy, int rows, int cols, float rate,
                                uint64_t seed, uint64_t stream) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE((type == RLT_TYPE_F32 || type == RLT_TYPE_BF16) && x && y && rows > 0 && cols > 0 && ldx >= cols && ldy >= cols && (!residual || ldr >= cols));
    RLT_REQUIRE(rate >= 0.0f && rate <= 1.0f);      // not a NaN either
    DropoutLaunch a = {x, residual, y, ldx, ldr, ldy, cols, (size_t)rows * cols, (uint32_t)(rate * 65536.0f + 0.5f), 0.0f, seed, stream, device->stream_offset};
    a.scale = a.threshold < 65536u ? (float)(65536.0 / (65536.0 - a.threshold)) : 0.0f;
    return type == RLT_TYPE_F32 ? launch<float>(device, a) : launch<rlt_bf16>(device, a);
}
