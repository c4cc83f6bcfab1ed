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

// THREADS share a row: a part of a wavefront, a wavefront (several rows to a workgroup of 256 then, whose wavefronts do not wait for each other) or a workgroup.
template <int THREADS> constexpr int WORKGROUP = THREADS <= 64 ? 256 : THREADS;

// Sums over the threads that share a row, every one of which receives them. Consecutive calls take turns with two halves of `lds`: a wavefront that writes one has passed the barrier
// behind which everybody had read it.
template <int THREADS, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* lds, int& turn) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        asm volatile("" : "+v"(v[i]));      // no contraction into the first exchange: both sides of an exchange round alike (rlt_wave_sum)
#pragma unroll
        for (int off = (THREADS < 64 ? THREADS : 64) / 2; off > 0; off >>= 1) v[i] += __shfl_xor(v[i], off, 64);
    }
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

// The gates' activations, in place, and their derivatives. One loop over a thread's gates for each function, not a choice for each gate. Functions as rlt_act has them; sigmoid and GELU, as x / (1 + e^(-2 z)),
// keep their relative accuracy where 1 + tanh(z) cancels.
template <int N, bool SLOPES> __device__ __forceinline__ void gates_of(float (&g)[N], float (&slope)[N], int kind) {
    if (kind == RLT_ACT_SIGMOID) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float e = __expf(-fabsf(g[i])), large = __fdividef(1.0f, 1.0f + e), small = e * large;      // e in (0, 1]: both to two units
            if (SLOPES) slope[i] = small * large;
            g[i] = g[i] >= 0.0f ? large : small;
        }
    } else if (kind == RLT_ACT_IDENTITY) {
#pragma unroll
        for (int i = 0; i < N; i++) slope[i] = 1.0f;
    } else if (kind == RLT_ACT_GELU) {
        const float a = 0.3989422804014327f, b = 0.044715f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = g[i], z = 2.0f * a * fmaf(b * x * x, x, x), e = expf(-fabsf(z)), large = 1.0f / (1.0f + e), small = e * large, p = z >= 0.0f ? large : small, q = z >= 0.0f ? small : large;
            if (SLOPES) slope[i] = p * fmaf(2.0f * x * q, a * fmaf(3.0f * b * x, x, 1.0f), 1.0f);
            g[i] = x * p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) { if (SLOPES) slope[i] = rlt_dact(g[i], kind); g[i] = rlt_act(g[i], kind); }
    }
}

template <typename T, int V, int K, int THREADS> __global__ __launch_bounds__(WORKGROUP<THREADS>) void norm_forward_kernel(NormForward a) {
    constexpr int N = V * K, ROWS = WORKGROUP<THREADS> / THREADS;
    __shared__ float lds[THREADS > 64 ? 2 * (THREADS / 64) * 4 : 1];
    int turn = 0;
    const int dim = a.p.dim;
    float bw[N], bb[N], ow[N], ob[N], scale[N];
    load_parameters<V, K, THREADS>(a.p.branch_weights, 1.0f, dim, bw); load_parameters<V, K, THREADS>(a.p.branch_biases, 0.0f, dim, bb);
    load_parameters<V, K, THREADS>(a.p.output_weights, 1.0f, dim, ow); load_parameters<V, K, THREADS>(a.p.output_biases, 0.0f, dim, ob);
    load_parameters<V, K, THREADS>(a.p.residual_scale, 1.0f, dim, scale);
    for (int row = blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows; row += gridDim.x * ROWS) {
        float y[N], u[N], g[N];
        if (a.branch) load_row<V, K, THREADS>((const T*)a.branch + (size_t)row * a.ldb, dim, u);
        load_row<V, K, THREADS>((const T*)a.x + (size_t)row * a.ldx, dim, y);
        if (a.branch && a.gate) load_row<V, K, THREADS>((const T*)a.gate + (size_t)row * a.ldg, dim, g);
        if (a.branch) {
            const float inverse = normalise<V, K, THREADS>(u, a.p.branch_norm, a.p.epsilon, dim, lds, turn);
            float slope[N];
            if (a.gate) gates_of<N, false>(g, slope, a.p.gate_activation);
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = fmaf(a.gate ? scale[i] * g[i] : scale[i], fmaf(u[i] * inverse, bw[i], bb[i]), y[i]);
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

template <typename T, int V, int K, int THREADS, bool BIASES> __global__ __launch_bounds__(WORKGROUP<THREADS>) void norm_backward_kernel(NormBackward a) {
    constexpr int N = V * K, ROWS = WORKGROUP<THREADS> / THREADS;
    __shared__ float lds[THREADS > 64 ? 2 * (THREADS / 64) * 4 : ROWS * THREADS * N];
    int turn = 0;
    const int dim = a.p.dim;
    float bw[N], bb[N], ow[N], scale[N];
    load_parameters<V, K, THREADS>(a.p.branch_weights, 1.0f, dim, bw);
    load_parameters<V, K, THREADS>(BIASES ? a.p.branch_biases : nullptr, 0.0f, dim, bb);
    load_parameters<V, K, THREADS>(a.p.output_weights, 1.0f, dim, ow); load_parameters<V, K, THREADS>(a.p.residual_scale, 1.0f, dim, scale);
    float sums[SUMS][N];
#pragma unroll
    for (int j = 0; j < SUMS; j++)
#pragma unroll
        for (int i = 0; i < N; i++) sums[j][i] = 0.0f;
    for (int row = blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows; row += gridDim.x * ROWS) {
        float d[N], e[N], y[N], u[N], g[N];      // d: the gradient that reaches the residual stream
        if (a.d_h) {
            load_row<V, K, THREADS>((const T*)a.d_h + (size_t)row * a.lddh, dim, e);
            load_row<V, K, THREADS>((const T*)a.y + (size_t)row * a.ldy, dim, y);
        }
        if (a.d_y) load_row<V, K, THREADS>((const T*)a.d_y + (size_t)row * a.lddy, dim, d);
        else {
#pragma unroll
            for (int i = 0; i < N; i++) d[i] = 0.0f;
        }
        if (a.branch) load_row<V, K, THREADS>((const T*)a.branch + (size_t)row * a.ldb, dim, u);
        if (a.branch && a.gate) load_row<V, K, THREADS>((const T*)a.gate + (size_t)row * a.ldg, dim, g);
        if (a.d_h) {
            const float inverse = normalise<V, K, THREADS>(y, a.p.output_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) {
                y[i] *= inverse;
                sums[OUTPUT_W][i] = fmaf(e[i], y[i], sums[OUTPUT_W][i]);
                if (BIASES) sums[OUTPUT_B][i] += e[i];
                e[i] *= ow[i];
            }
            norm_gradient<V, K, THREADS>(e, y, inverse, a.p.output_norm, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) d[i] += e[i];
        }
        if (a.d_x) store_row<V, K, THREADS>((T*)a.d_x + (size_t)row * a.lddx, dim, d);
        if (a.branch) {
            const float inverse = normalise<V, K, THREADS>(u, a.p.branch_norm, a.p.epsilon, dim, lds, turn);
            float slope[N];
            if (a.gate) gates_of<N, true>(g, slope, a.p.gate_activation);
#pragma unroll
            for (int i = 0; i < N; i++) {
                u[i] *= inverse;
                const float n = BIASES ? fmaf(u[i], bw[i], bb[i]) : u[i] * bw[i], m = a.gate ? g[i] : 1.0f, dn = d[i] * scale[i] * m;
                sums[SCALE][i] = fmaf(d[i] * m, n, sums[SCALE][i]);
                sums[BRANCH_W][i] = fmaf(dn, u[i], sums[BRANCH_W][i]);
                if (BIASES) sums[BRANCH_B][i] += dn;
                if (a.gate) slope[i] *= d[i] * scale[i] * n;
                e[i] = dn * bw[i];
            }
            if (a.d_gate) store_row<V, K, THREADS>((T*)a.d_gate + (size_t)row * a.lddg, dim, slope);
            if (a.d_branch) {
                norm_gradient<V, K, THREADS>(e, u, inverse, a.p.branch_norm, dim, lds, turn);
                store_row<V, K, THREADS>((T*)a.d_branch + (size_t)row * a.lddb, dim, e);
            }
        }
    }
    float* const wanted[SUMS] = {a.p.d_branch_weights, a.p.d_branch_biases, a.p.d_output_weights, a.p.d_output_biases, a.p.d_residual_scale};
    float* out = a.partial + (size_t)blockIdx.x * SUMS * dim;
#pragma unroll
    for (int j = 0; j < SUMS; j++) {
        if (!wanted[j]) continue;
        if constexpr (ROWS > 1) {      // the rows' threads side by side, then column by column in their order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) lds[(threadIdx.x / THREADS) * THREADS * N + (k * THREADS + threadIdx.x % THREADS) * V + i] = sums[j][k * V + i];
            __syncthreads();
            for (int c = threadIdx.x; c < dim; c += WORKGROUP<THREADS>) {
                float s = 0.0f;
#pragma unroll
                for (int r = 0; r < ROWS; r++) s += lds[r * THREADS * N + c];
                out[(size_t)j * dim + c] = s;
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int c = (k * THREADS + (int)threadIdx.x) * V + i;
                    if (c < dim) out[(size_t)j * dim + c] = sums[j][k * V + i];
                }
        }
    }
}

// adds up the workgroups' column sums, in a fixed order: 64 columns to a workgroup, whose wavefronts take every sixteenth block each
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float* __restrict__ partial, int blocks, int dim, rlt_residual_norm p, int accumulate) {
    __shared__ float part[16][64];
    float* const to[SUMS] = {p.d_branch_weights, p.d_branch_biases, p.d_output_weights, p.d_output_biases, p.d_residual_scale};
    float* dst = to[blockIdx.y];
    if (!dst) return;
    const int lane = threadIdx.x & 63, c = blockIdx.x * 64 + lane, wave = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < dim)
#pragma unroll 8
        for (int b = wave; b < blocks; b += 16) s += partial[((size_t)b * SUMS + blockIdx.y) * dim + c];
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < dim) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; w++) s += part[w][lane];
        dst[c] = accumulate ? dst[c] + s : s;
    }
}

// threads that share a row in the backward pass, eight columns each
int backward_threads(int dim) { return dim <= 128 ? 16 : dim <= 512 ? 64 : dim <= 1024 ? 128 : dim <= 2048 ? 256 : dim <= 4096 ? 512 : 1024; }
int backward_blocks(const rlt_residual_norm* p, int rows) {
    const int threads = backward_threads(p->dim), at_once = threads <= 64 ? 256 / threads : 1, blocks = (rows + at_once - 1) / at_once;
    return blocks < 512 ? blocks : 512;
}

template <typename T, int V> void launch_forward(rlt_rocm_device* device, const NormForward& a) {
    const int dim = a.p.dim;
    auto go = [&](auto kernel, int threads) {
        const int workgroup = threads <= 64 ? 256 : threads, at_once = workgroup / threads, blocks = (a.rows + at_once - 1) / at_once;
        hipLaunchKernelGGL(kernel, dim3(blocks < 2048 ? blocks : 2048), dim3(workgroup), 0, device->stream, a);
    };
    if (dim <= 128) go(norm_forward_kernel<T, V, 8 / V, 16>, 16);
    else if (dim <= 512) go(norm_forward_kernel<T, V, 8 / V, 64>, 64);
    else if (dim <= 1024) go(norm_forward_kernel<T, V, 8 / V, 128>, 128);
    else if (dim <= 2048) go(norm_forward_kernel<T, V, 8 / V, 256>, 256);
    else if (dim <= 4096) go(norm_forward_kernel<T, V, 8 / V, 512>, 512);
    else go(norm_forward_kernel<T, V, 8 / V, 1024>, 1024);
}
template <typename T, int V, bool BIASES> void launch_backward(rlt_rocm_device* device, const NormBackward& a) {
    const int threads = backward_threads(a.p.dim);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(backward_blocks(&a.p, a.rows)), dim3(threads <= 64 ? 256 : threads), 0, device->stream, a); };
    if (threads == 16) go(norm_backward_kernel<T, V, 8 / V, 16, BIASES>);
    else if (threads == 64) go(norm_backward_kernel<T, V, 8 / V, 64, BIASES>);
    else if (threads == 128) go(norm_backward_kernel<T, V, 8 / V, 128, BIASES>);
    else if (threads == 256) go(norm_backward_kernel<T, V, 8 / V, 256, BIASES>);
    else if (threads == 512) go(norm_backward_kernel<T, V, 8 / V, 512, BIASES>);
    else go(norm_backward_kernel<T, V, 8 / V, 1024, BIASES>);
}
// vectors of 16 bytes where every tensor's rows start on such boundaries and hold whole vectors
template <typename T> void forward(rlt_rocm_device* device, const NormForward& a) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = a.p.dim % V == 0 && rlt_vectors<T>(a.x, a.ldx) && rlt_vectors<T>(a.branch, a.branch ? a.ldb : 0) && rlt_vectors<T>(a.gate, a.gate ? a.ldg : 0) &&
                         rlt_vectors<T>(a.y, a.y ? a.ldy : 0) && rlt_vectors<T>(a.h, a.h ? a.ldh : 0);
    if (vectors) launch_forward<T, V>(device, a); else launch_forward<T, 1>(device, a);
}
template <typename T> void backward(rlt_rocm_device* device, const NormBackward& a) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = a.p.dim % V == 0 && rlt_vectors<T>(a.branch, a.branch ? a.ldb : 0) && rlt_vectors<T>(a.gate, a.gate ? a.ldg : 0) && rlt_vectors<T>(a.y, a.d_h ? a.ldy : 0) &&
                         rlt_vectors<T>(a.d_y, a.d_y ? a.lddy : 0) && rlt_vectors<T>(a.d_h, a.d_h ? a.lddh : 0) && rlt_vectors<T>(a.d_x, a.d_x ? a.lddx : 0) &&
                         rlt_vectors<T>(a.d_branch, a.d_branch ? a.lddb : 0) && rlt_vectors<T>(a.d_gate, a.d_gate ? a.lddg : 0);
    const bool biases = a.p.branch_biases || a.p.d_branch_biases || a.p.d_output_biases;
    if (vectors) { if (biases) launch_backward<T, V, true>(device, a); else launch_backward<T, V, false>(device, a); }
    else { if (biases) launch_backward<T, 1, true>(device, a); else launch_backward<T, 1, false>(device, a); }
}

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
    if (layer->type == RLT_TYPE_F32) forward<float>(device, a); else forward<rlt_bf16>(device, a);
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
    if (layer->type == RLT_TYPE_F32) backward<float>(device, a); else backward<rlt_bf16>(device, a);
    int rc = rlt_launch_status(device);
    if (rc || !sums) return rc;
    hipLaunchKernelGGL(norm_sum_kernel, dim3((dim + 63) / 64, SUMS), dim3(1024), 0, device->stream, (const float*)workspace, backward_blocks(layer, rows), dim, *layer, accumulate);
    return rlt_launch_status(device);
}

}  // extern "C"
