// The norm after a block, its gate and residual scale, and the norm before the next block: one pass over the rows forward, one backward.
#include "typed.h"

namespace {

constexpr int MAX_DIM = 8192;
enum { BRANCH_W = 0, BRANCH_B, OUTPUT_W, OUTPUT_B, SCALE, SUMS };      // column sums of the backward pass

struct NormForward {
    rlt_residual_norm p;
    const void* x; const void* branch; const void* gate; void* y; void* h;
    int ldx, ldb, ldg, ldy, ldh, rows;
};
struct NormBackward {
    rlt_residual_norm p;
    const void* branch; const void* gate; const void* y; const void* d_y; const void* d_h; void* d_x; void* d_branch; void* d_gate;
    int ldb, ldg, ldy, lddy, lddh, lddx, lddb, lddg, rows;
    float* partial;               // [workgroups][SUMS][dim]
};

// Sums over the THREADS that share a row, every one of which receives them. Consecutive calls take turns with two halves of `lds`: a wavefront that writes one has passed the barrier
// behind which everybody had read it.
template <int THREADS, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* lds, int& turn) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = rlt_wave_sum(v[i]);
    if constexpr (THREADS > 64) {
        constexpr int WAVES = THREADS / 64;
        float* half = lds + turn * WAVES * 4;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) half[(threadIdx.x >> 6) * 4 + i] = v[i];
        }
        rlt_lds_barrier();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) s += half[w * 4 + i];
            v[i] = s;
        }
    }
}

// Thread t of a row's THREADS has vectors t, t + THREADS, ... of V elements, K of them.
template <int V, int K, int THREADS, typename T> __device__ __forceinline__ void load_row(const T* src, int dim, float (&v)[V * K]) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V;
        if (c < dim) rlt_load<V>(src + c, v + k * V);
        else {
#pragma unroll
            for (int i = 0; i < V; i++) v[k * V + i] = 0.0f;
        }
    }
}
template <int V, int K, int THREADS, typename T> __device__ __forceinline__ void store_row(T* dst, int dim, const float (&v)[V * K]) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V;
        if (c < dim) rlt_store<V>(dst + c, v + k * V);
    }
}
// parameters of this thread's columns; `otherwise` where there are none
template <int V, int K, int THREADS> __device__ __forceinline__ void load_parameters(const float* src, float otherwise, int dim, float (&v)[V * K]) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V + i;
            v[k * V + i] = src && c < dim ? src[c] : otherwise;
        }
}
// subtracts a row's mean; columns beyond dim stay zero
template <int V, int K, int THREADS> __device__ __forceinline__ void subtract(float (&v)[V * K], float mean, int dim) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V;
        if (c < dim) {
#pragma unroll
            for (int i = 0; i < V; i++) v[k * V + i] -= mean;
        }
    }
}

// a row's values less their mean (RLT_NORM_LAYER), and 1 / deviation
template <int V, int K, int THREADS> __device__ __forceinline__ float normalise(float (&v)[V * K], int kind, float epsilon, int dim, float* lds, int& turn) {
    constexpr int N = V * K;
    if (kind == RLT_NORM_NONE) return 1.0f;
    const float inverse_dim = 1.0f / dim;
    float s[1];
    if (kind == RLT_NORM_LAYER) {
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += v[i];
        row_sums<THREADS>(s, lds, turn);
        subtract<V, K, THREADS>(v, s[0] * inverse_dim, dim);
    }
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) s[0] = fmaf(v[i], v[i], s[0]);
    row_sums<THREADS>(s, lds, turn);
    return 1.0f / sqrtf(s[0] * inverse_dim + epsilon);
}

// The gate's activation and its derivative. Functions as rlt_act has them; GELU as x / (1 + e^(-2 z)), which keeps its relative accuracy where 1 + tanh(z) cancels.
__device__ __forceinline__ float gate_of(float x, int kind, float& slope) {
    if (kind == RLT_ACT_SIGMOID || kind == RLT_ACT_GELU) {
        const float a = 0.3989422804014327f, b = 0.044715f, z = kind == RLT_ACT_GELU ? 2.0f * a * fmaf(b * x * x, x, x) : x;
        const float e = expf(-fabsf(z)), large = 1.0f / (1.0f + e), small = e * large, p = z >= 0.0f ? large : small, q = z >= 0.0f ? small : large;      // p + q = 1
        if (kind == RLT_ACT_SIGMOID) { slope = p * q; return p; }
        slope = p * fmaf(2.0f * x * q, a * fmaf(3.0f * b * x, x, 1.0f), 1.0f);
        return x * p;
    }
    slope = rlt_dact(x, kind);
    return rlt_act(x, kind);
}

template <typename T, int V, int K, int THREADS> __global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_forward_kernel(NormForward a) {
    constexpr int N = V * K, ROWS = THREADS < 256 ? 256 / THREADS : 1;
    __shared__ float lds[THREADS > 64 ? 2 * (THREADS / 64) * 4 : 1];
    int turn = 0;
    const int dim = a.p.dim;
    float bw[N], bb[N], ow[N], ob[N], scale[N];
    load_parameters<V, K, THREADS>(a.p.branch_weights, 1.0f, dim, bw); load_parameters<V, K, THREADS>(a.p.branch_biases, 0.0f, dim, bb);
    load_parameters<V, K, THREADS>(a.p.output_weights, 1.0f, dim, ow); load_parameters<V, K, THREADS>(a.p.output_biases, 0.0f, dim, ob);
    load_parameters<V, K, THREADS>(a.p.residual_scale, 1.0f, dim, scale);
    for (int row = blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows; row += gridDim.x * ROWS) {
        float y[N];
        load_row<V, K, THREADS>((const T*)a.x + (size_t)row * a.ldx, dim, y);
        if (a.branch) {
            float u[N], g[N];
            load_row<V, K, THREADS>((const T*)a.branch + (size_t)row * a.ldb, dim, u);
            if (a.gate) load_row<V, K, THREADS>((const T*)a.gate + (size_t)row * a.ldg, dim, g);
            const float inverse = normalise<V, K, THREADS>(u, a.p.branch_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float n = fmaf(u[i] * inverse, bw[i], bb[i]);
                float slope;
                y[i] = fmaf(a.gate ? scale[i] * gate_of(g[i], a.p.gate_activation, slope) : scale[i], n, y[i]);
            }
            // columns beyond dim: u, g and y are zero, a bias is too
        }
        if (a.y) store_row<V, K, THREADS>((T*)a.y + (size_t)row * a.ldy, dim, y);
        if (a.h) {
            const float inverse = normalise<V, K, THREADS>(y, a.p.output_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = fmaf(y[i] * inverse, ow[i], ob[i]);
            store_row<V, K, THREADS>((T*)a.h + (size_t)row * a.ldh, dim, y);
        }
    }
}

// d: gradient with respect to the normalised row; becomes the one with respect to the row
template <int V, int K, int THREADS> __device__ __forceinline__ void norm_gradient(float (&d)[V * K], const float (&normalised)[V * K], float inverse, int kind, int dim, float* lds, int& turn) {
    constexpr int N = V * K;
    if (kind == RLT_NORM_NONE) return;
    const float inverse_dim = 1.0f / dim;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; i++) { s[0] = fmaf(d[i], normalised[i], s[0]); s[1] += d[i]; }
    row_sums<THREADS>(s, lds, turn);
    const float along = s[0] * inverse_dim, mean = kind == RLT_NORM_LAYER ? s[1] * inverse_dim : 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V;
#pragma unroll
        for (int i = k * V; i < k * V + V; i++) d[i] = c < dim ? inverse * (d[i] - normalised[i] * along - mean) : 0.0f;      // the sums that follow take no column beyond dim
    }
}

template <typename T, int V, int K, int THREADS> __global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_backward_kernel(NormBackward a) {
    constexpr int N = V * K, ROWS = THREADS < 256 ? 256 / THREADS : 1;
    __shared__ float lds[THREADS > 64 ? 2 * (THREADS / 64) * 4 : 1];
    int turn = 0;
    const int dim = a.p.dim;
    float bw[N], bb[N], ow[N], scale[N];
    load_parameters<V, K, THREADS>(a.p.branch_weights, 1.0f, dim, bw); load_parameters<V, K, THREADS>(a.p.branch_biases, 0.0f, dim, bb);
    load_parameters<V, K, THREADS>(a.p.output_weights, 1.0f, dim, ow); load_parameters<V, K, THREADS>(a.p.residual_scale, 1.0f, dim, scale);
    float sums[SUMS][N];
#pragma unroll
    for (int j = 0; j < SUMS; j++)
#pragma unroll
        for (int i = 0; i < N; i++) sums[j][i] = 0.0f;
    for (int row = blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows; row += gridDim.x * ROWS) {
        float d[N];      // the gradient that reaches the residual stream
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = 0.0f;
        if (a.d_y) load_row<V, K, THREADS>((const T*)a.d_y + (size_t)row * a.lddy, dim, d);
        if (a.d_h) {
            float e[N], y[N];
            load_row<V, K, THREADS>((const T*)a.d_h + (size_t)row * a.lddh, dim, e);
            load_row<V, K, THREADS>((const T*)a.y + (size_t)row * a.ldy, dim, y);
            const float inverse = normalise<V, K, THREADS>(y, a.p.output_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) {
                y[i] *= inverse;
                sums[OUTPUT_W][i] = fmaf(e[i], y[i], sums[OUTPUT_W][i]); sums[OUTPUT_B][i] += e[i];
                e[i] *= ow[i];
            }
            norm_gradient<V, K, THREADS>(e, y, inverse, a.p.output_norm, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) d[i] += e[i];
        }
        if (a.d_x) store_row<V, K, THREADS>((T*)a.d_x + (size_t)row * a.lddx, dim, d);
        if (a.branch) {
            float u[N], g[N], e[N];
            load_row<V, K, THREADS>((const T*)a.branch + (size_t)row * a.ldb, dim, u);
            if (a.gate) load_row<V, K, THREADS>((const T*)a.gate + (size_t)row * a.ldg, dim, g);
            const float inverse = normalise<V, K, THREADS>(u, a.p.branch_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) {
                u[i] *= inverse;
                float slope;
                const float n = fmaf(u[i], bw[i], bb[i]), m = a.gate ? gate_of(g[i], a.p.gate_activation, slope) : 1.0f, dn = d[i] * scale[i] * m;
                sums[SCALE][i] = fmaf(d[i] * m, n, sums[SCALE][i]);
                sums[BRANCH_W][i] = fmaf(dn, u[i], sums[BRANCH_W][i]); sums[BRANCH_B][i] += dn;
                if (a.gate) g[i] = d[i] * scale[i] * n * slope;
                e[i] = dn * bw[i];
            }
            if (a.d_gate) store_row<V, K, THREADS>((T*)a.d_gate + (size_t)row * a.lddg, dim, g);
            if (a.d_branch) {
                norm_gradient<V, K, THREADS>(e, u, inverse, a.p.branch_norm, dim, lds, turn);
                store_row<V, K, THREADS>((T*)a.d_branch + (size_t)row * a.lddb, dim, e);
            }
        }
    }
    float* out = a.partial + ((size_t)blockIdx.x * ROWS + threadIdx.x / THREADS) * SUMS * dim;
    float* const wanted[SUMS] = {a.p.d_branch_weights, a.p.d_branch_biases, a.p.d_output_weights, a.p.d_output_biases, a.p.d_residual_scale};
#pragma unroll
    for (int j = 0; j < SUMS; j++)
        if (wanted[j]) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int c = (k * THREADS + (int)(threadIdx.x % THREADS)) * V + i;
                    if (c < dim) out[(size_t)j * dim + c] = sums[j][k * V + i];
                }
        }
}

// adds up the workgroups' column sums, in their order: 64 columns to a workgroup, whose wavefronts take every fourth block each
__global__ __launch_bounds__(256) void norm_sum_kernel(const float* __restrict__ partial, int blocks, int dim, rlt_residual_norm p, int accumulate) {
    __shared__ float part[4][64];
    float* const to[SUMS] = {p.d_branch_weights, p.d_branch_biases, p.d_output_weights, p.d_output_biases, p.d_residual_scale};
    float* dst = to[blockIdx.y];
    if (!dst) return;
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < dim)
        for (int b = wave; b < blocks; b += 4) s += partial[((size_t)b * SUMS + blockIdx.y) * dim + c];
    part[wave][threadIdx.x & 63] = s;
    __syncthreads();
    if (wave == 0 && c < dim) {
        s = ((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x];
        dst[c] = accumulate ? dst[c] + s : s;
    }
}

int backward_blocks(const rlt_residual_norm*, int rows) { return rows < 256 ? rows : 256; }

bool described(const rlt_residual_norm* p) {
    return p && (p->type == RLT_TYPE_F32 || p->type == RLT_TYPE_BF16) && p->dim > 0 && p->branch_norm >= RLT_NORM_NONE && p->branch_norm <= RLT_NORM_LAYER && p->output_norm >= RLT_NORM_NONE &&
           p->output_norm <= RLT_NORM_LAYER && p->gate_activation >= RLT_ACT_IDENTITY && p->gate_activation <= RLT_ACT_SIGMOID && p->epsilon > 0.0f;
}

}  // namespace

extern "C" {

int rlt_rocm_residual_norm_forward(rlt_rocm_device* device, const rlt_residual_norm* layer, const void* x, int ldx, const void* branch, int ldb, const void* gate, int ldg,
                                   void* y, int ldy, void* h, int ldh, int rows) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && rows > 0);
    const int dim = layer->dim;
    RLT_REQUIRE(x && ldx >= dim && (!branch || ldb >= dim) && (!gate || ldg >= dim) && (!y || ldy >= dim) && (!h || ldh >= dim) && (y || h));
    if (dim > MAX_DIM) return RLT_E_UNSUPPORTED;
    const NormForward a = {*layer, x, branch, gate, y, h, ldx, ldb, ldg, ldy, ldh, rows};
    if (layer->type == RLT_TYPE_F32) hipLaunchKernelGGL((norm_forward_kernel<float, 1, 8, 1024>), dim3(rows < 1024 ? rows : 1024), dim3(1024), 0, device->stream, a);
    else hipLaunchKernelGGL((norm_forward_kernel<rlt_bf16, 1, 8, 1024>), dim3(rows < 1024 ? rows : 1024), dim3(1024), 0, device->stream, a);
    return rlt_launch_status(device);
}

size_t rlt_rocm_residual_norm_workspace_bytes(const rlt_residual_norm* layer, int rows) {
    if (!described(layer) || rows <= 0) return 0;
    return (size_t)backward_blocks(layer, rows) * SUMS * layer->dim * sizeof(float);
}

int rlt_rocm_residual_norm_backward(rlt_rocm_device* device, const rlt_residual_norm* layer, const void* branch, int ldb, const void* gate, int ldg, const void* y, int ldy,
                                    const void* d_y, int lddy, const void* d_h, int lddh, void* d_x, int lddx, void* d_branch, int lddb, void* d_gate, int lddg, int rows,
                                    int accumulate, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && rows > 0);
    const int dim = layer->dim;
    RLT_REQUIRE((d_y || d_h) && (!d_y || lddy >= dim) && (!d_h || (lddh >= dim && y && ldy >= dim)) && (!branch || ldb >= dim) && (!gate || ldg >= dim));
    RLT_REQUIRE((!d_x || lddx >= dim) && (!d_branch || (branch && lddb >= dim)) && (!d_gate || (branch && gate && lddg >= dim)));
    // gradients of parameters that nothing reaches
    RLT_REQUIRE((branch || !(layer->d_branch_weights || layer->d_branch_biases || layer->d_residual_scale)) && (d_h || !(layer->d_output_weights || layer->d_output_biases)));
    if (dim > MAX_DIM) return RLT_E_UNSUPPORTED;
    const bool sums = layer->d_branch_weights || layer->d_branch_biases || layer->d_output_weights || layer->d_output_biases || layer->d_residual_scale;
    RLT_REQUIRE(!sums || (workspace && workspace_bytes >= rlt_rocm_residual_norm_workspace_bytes(layer, rows)));
    const NormBackward a = {*layer, branch, gate, y, d_y, d_h, d_x, d_branch, d_gate, ldb, ldg, ldy, lddy, lddh, lddx, lddb, lddg, rows, (float*)workspace};
    const int blocks = backward_blocks(layer, rows);
    if (layer->type == RLT_TYPE_F32) hipLaunchKernelGGL((norm_backward_kernel<float, 1, 8, 1024>), dim3(blocks), dim3(1024), 0, device->stream, a);
    else hipLaunchKernelGGL((norm_backward_kernel<rlt_bf16, 1, 8, 1024>), dim3(blocks), dim3(1024), 0, device->stream, a);
    int rc = rlt_launch_status(device);
    if (rc || !sums) return rc;
    hipLaunchKernelGGL(norm_sum_kernel, dim3((dim + 63) / 64, SUMS), dim3(256), 0, device->stream, (const float*)workspace, blocks, dim, *layer, accumulate);
    return rlt_launch_status(device);
}

}  // extern "C"
