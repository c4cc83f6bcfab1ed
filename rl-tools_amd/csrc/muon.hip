// Optimiser step for matrices whose updates are orthogonalised by products: A = X X^T, X <- a X + (b A + c A A) X, a few times.
#include "typed.h"

namespace {

// Factors are held as two numbers of 16 bits, the value's nearest and what it leaves: 22 bits and a sign, whose products in the matrix instructions (high x high, high x low, low x high, summed up in fp32) are as good as fp32's own:
// what is dropped, low x low and the rounding of the low part, is 2^-24.6 of a product in the mean (fp32's own rounding of a factor: 2^-25.3), at a third of the 16-bit rate, where fp32 instructions have a sixteenth.
// Values are held times SCALE. Singular values stay below 1.21, those of A below 1.47, those of b A + c A A above -2.81 and below 0, so that no element leaves the range of 16 bits.
typedef _Float16 f16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr float SCALE = 16384.0f, UNSCALE = 1.0f / 16384.0f, QA = 3.4445f, QB = -4.775f, QC = 2.0315f;
constexpr int GROUP = 24, MAX_SIDE = 1 << 16, MAX_ITERATIONS = 32, PARTS = 256;      // matrices of a launch; partial sums of a norm

struct Matrix {
    const float* w; const float* g; const float* m; float* next_w; float* next_m;
    double* sums;                 // PARTS partial sums of u^2
    f16* x; f16* t[2]; f16* a; f16* b;      // X [M x N], its transpose [N x M] (one that is read, one that is written), A and b A + c A A [M x M]; the low parts behind the high ones
    int rows, cols, M, N;         // M <= N: rows and columns, or columns and rows where there are more rows, filled up to whole tiles
    float factor;                 // alpha * sqrt(max(1, rows / cols))
    int first;                    // workgroups of a launch before this matrix's
};
struct Matrices {
    Matrix m[GROUP];
    int n, from;                  // from: which transpose is read
    float momentum, epsilon, keep;      // keep: 1 - alpha * weight_decay
    int nesterov;
};
__device__ __forceinline__ const Matrix& matrix_of(const Matrices& all, int& block) {
    int i = 0;
    while (i + 1 < all.n && block >= all.m[i + 1].first) i++;
    block -= all.m[i].first;
    return all.m[i];
}
__device__ __forceinline__ void split(float v, f16& high, f16& low) { high = (f16)v; low = (f16)(v - (float)high); }

// The momentum, and the sum of the update's squares in 64 bits (no square of an fp32 number leaves their range).
__global__ __launch_bounds__(256) void momentum_kernel(Matrices all) {
    __shared__ double sums[4];
    int block = blockIdx.x;
    const Matrix& a = matrix_of(all, block);
    const size_t size = (size_t)a.rows * a.cols;
    double s = 0.0;
    for (size_t i = (size_t)block * 256 + threadIdx.x; i < size; i += PARTS * 256) {
        const float g = a.g[i], m = fmaf(all.momentum, a.m[i], g), u = all.nesterov ? fmaf(all.momentum, m, g) : m;
        a.next_m[i] = m;
        s = fma((double)u, (double)u, s);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.sums[block] = ((sums[0] + sums[1]) + sums[2]) + sums[3];
}

// X and its transpose, tiles of 64 x 64, zeros beyond the matrix
__global__ __launch_bounds__(256) void normalise_kernel(Matrices all) {
    __shared__ float tile[64][65];
    __shared__ double norm;
    int block = blockIdx.x;
    const Matrix& a = matrix_of(all, block);
    const bool tall = a.rows > a.cols;
    const int wide = tall ? a.M : a.N, across = wide / 64, r0 = block / across * 64, c0 = block % across * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave == 0) {
        double s = 0.0;
        for (int i = lane; i < PARTS; i += 64) s += a.sums[i];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
        if (lane == 0) norm = sqrt(s) + (double)all.epsilon;
    }
    __syncthreads();
    const double inverse = (double)SCALE / norm;
    f16* const rows = tall ? a.t[0] : a.x; f16* const columns = tall ? a.x : a.t[0];
    const size_t plane = (size_t)a.M * a.N;
    const int high = tall ? a.N : a.M;
#pragma unroll 4
    for (int i = wave; i < 64; i += 4) {
        const int r = r0 + i, c = c0 + lane;
        float v = 0.0f;
        if (r < a.rows && c < a.cols) {
            const size_t e = (size_t)r * a.cols + c;
            const float g = a.g[e], m = a.next_m[e];
            v = (float)((double)(all.nesterov ? fmaf(all.momentum, m, g) : m) * inverse);
        }
        tile[i][lane] = v;
        f16 h, l;
        split(v, h, l);
        rows[(size_t)r * wide + c] = h; rows[plane + (size_t)r * wide + c] = l;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = wave; i < 64; i += 4) {
        f16 h, l;
        split(tile[lane][i], h, l);
        columns[(size_t)(c0 + i) * high + r0 + lane] = h; columns[plane + (size_t)(c0 + i) * high + r0 + lane] = l;
    }
}

// C[i][j] = sum over k of P[i][k] Q[j][k], both with k side by side. Four wavefronts share a tile of 64 W x 64 W, each has W x W tiles of 32 x 32. GRAM: A = X X^T; SQUARE: b A + c A A (both symmetric: tiles on and below the
// diagonal, written twice); UPDATE: a X + (b A + c A A) X; LAST: the same, straight into the parameters.
enum Phase { GRAM, SQUARE, UPDATE, LAST };
template <int W, int PHASE> __global__ __launch_bounds__(256) void product_kernel(Matrices all) {
    constexpr int T = 64 * W, BK = 32, ROWS = 4 * T, LOADS = ROWS * 4 / 256;      // rows of the tile in LDS: P high, P low, Q high, Q low
    extern __shared__ __attribute__((aligned(16))) f16 lds[];      // [2][ROWS][BK], chunks of eight changed about within a row so that the rows that are read together lie in different banks
    int block = blockIdx.x;
    const Matrix& a = matrix_of(all, block);
    const bool symmetric = PHASE == GRAM || PHASE == SQUARE;
    int ti, tj;
    if (symmetric) {
        ti = (int)((sqrtf(8.0f * block + 1.0f) - 1.0f) * 0.5f);
        while (ti * (ti + 1) / 2 > block) ti--;
        while ((ti + 1) * (ti + 2) / 2 <= block) ti++;
        tj = block - ti * (ti + 1) / 2;
    } else { const int down = a.M / T; tj = block / down; ti = block - tj * down; }
    const int depth = PHASE == GRAM ? a.N : a.M;
    const f16* const P = PHASE == GRAM ? a.x : PHASE == SQUARE ? a.a : a.b; const f16* const Q = PHASE == GRAM ? a.x : PHASE == SQUARE ? a.a : a.t[all.from];
    const size_t square = (size_t)a.M * a.M, plane = (size_t)a.M * a.N, p_plane = PHASE == GRAM ? plane : square, q_plane = PHASE == SQUARE ? square : plane;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    const int row = threadIdx.x >> 2, chunk = threadIdx.x & 3;
    const f16* const p0 = P + (size_t)(ti * T + row) * depth + chunk * 8; const f16* const q0 = Q + (size_t)(tj * T + row) * depth + chunk * 8;
    f16x8 held[LOADS];
    auto ask = [&](int k) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int part = i / W, down = i % W * 64;      // part: P high, P low, Q high, Q low
            const f16* const from = part < 2 ? p0 + (part & 1) * p_plane : q0 + (part & 1) * q_plane;
            held[i] = *reinterpret_cast<const f16x8*>(from + (size_t)down * depth + k);
        }
    };
    f32x16 sum[W][W];
#pragma unroll
    for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < W; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum[i][j][e] = 0.0f;
    ask(0);
    int turn = 0;
    for (int k = 0; k < depth; k += BK, turn ^= 1) {
        f16* const to = lds + turn * ROWS * BK;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int r = i * 64 + row;
            *reinterpret_cast<f16x8*>(to + r * BK + (chunk ^ (r >> 1 & 3)) * 8) = held[i];
        }
        if (k + BK < depth) ask(k + BK);
        rlt_lds_barrier();
#pragma unroll
        for (int kk = 0; kk < BK / 16; kk++) {
            auto fragment = [&](int part, int tile) {
                const int r = part * T + tile * 32 + (lane & 31);
                return *reinterpret_cast<const f16x8*>(to + r * BK + ((kk * 2 + (lane >> 5)) ^ (r >> 1 & 3)) * 8);
            };
            f16x8 ph[W], pl[W], qh[W], ql[W];
#pragma unroll
            for (int i = 0; i < W; i++) {
                ph[i] = fragment(0, wi * W + i); pl[i] = fragment(1, wi * W + i);
                qh[i] = fragment(2, wj * W + i); ql[i] = fragment(3, wj * W + i);
            }
#pragma unroll
            for (int i = 0; i < W; i++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[i], qh[j], sum[i][j], 0, 0, 0);
                    sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], ql[j], sum[i][j], 0, 0, 0);
                    sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], qh[j], sum[i][j], 0, 0, 0);
                }
        }
    }
    // a lane has column lane % 32 and, four by four, rows of its tiles
#pragma unroll
    for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int c = tj * T + (wj * W + j) * 32 + (lane & 31);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int r = ti * T + (wi * W + i) * 32 + g * 8 + (lane >> 5) * 4;
                f16x4 high, low;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[e] = sum[i][j][g * 4 + e] * UNSCALE;
                    if (PHASE == SQUARE) v[e] = fmaf(QC, v[e], QB * ((float)a.a[(size_t)(r + e) * a.M + c] + (float)a.a[square + (size_t)(r + e) * a.M + c]));
                    if (PHASE == UPDATE || PHASE == LAST) v[e] = fmaf(QA, (float)a.x[(size_t)(r + e) * a.N + c] + (float)a.x[plane + (size_t)(r + e) * a.N + c], v[e]);
                    f16 h, l;
                    split(v[e], h, l);
                    high[e] = h; low[e] = l;
                }
                if (PHASE == LAST) {
                    const bool tall = a.rows > a.cols;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int wr = tall ? c : r + e, wc = tall ? r + e : c;
                        if (wr < a.rows && wc < a.cols) a.next_w[(size_t)wr * a.cols + wc] = fmaf(-a.factor, v[e] * UNSCALE, all.keep * a.w[(size_t)wr * a.cols + wc]);
                    }
                } else if (PHASE == UPDATE) {
#pragma unroll
                    for (int e = 0; e < 4; e++) { a.x[(size_t)(r + e) * a.N + c] = high[e]; a.x[plane + (size_t)(r + e) * a.N + c] = low[e]; }
                    f16* const t = a.t[all.from ^ 1] + (size_t)c * a.M + r;
                    *reinterpret_cast<f16x4*>(t) = high; *reinterpret_cast<f16x4*>(t + plane) = low;
                } else {
                    f16* const out = PHASE == GRAM ? a.a : a.b;
#pragma unroll
                    for (int e = 0; e < 4; e++) { out[(size_t)(r + e) * a.M + c] = high[e]; out[square + (size_t)(r + e) * a.M + c] = low[e]; }
                    if (ti != tj) { *reinterpret_cast<f16x4*>(out + (size_t)c * a.M + r) = high; *reinterpret_cast<f16x4*>(out + square + (size_t)c * a.M + r) = low; }
                }
            }
        }
}

bool described(const rlt_muon_tensor* t, int n) {
    if (!t || n <= 0) return false;
    for (int i = 0; i < n; i++) if (t[i].rows <= 0 || t[i].cols <= 0) return false;
    return true;
}
bool supported(const rlt_muon_tensor* t, int n) {
    for (int i = 0; i < n; i++) if (t[i].rows > MAX_SIDE || t[i].cols > MAX_SIDE || (int64_t)t[i].rows * t[i].cols > 1 << 30) return false;
    return true;
}
// tiles of 128 x 128 from there on
int width_of(const rlt_muon_tensor& t) { return (t.rows < t.cols ? t.rows : t.cols) >= 512 ? 2 : 1; }
int filled(int n, int tile) { return (n + tile - 1) / tile * tile; }
size_t bytes_of(const rlt_muon_tensor& t) {
    const int tile = 64 * width_of(t);
    const size_t M = filled(t.rows < t.cols ? t.rows : t.cols, tile), N = filled(t.rows < t.cols ? t.cols : t.rows, tile);
    return PARTS * sizeof(double) + (6 * M * N + 4 * M * M) * sizeof(f16);
}
template <int W, int PHASE> int launch(rlt_rocm_device* device, Matrices& all) {
    size_t blocks = 0;
    for (int i = 0; i < all.n; i++) {
        all.m[i].first = (int)blocks;
        const size_t down = all.m[i].M / (64 * W), across = all.m[i].N / (64 * W);
        blocks += PHASE == GRAM || PHASE == SQUARE ? down * (down + 1) / 2 : down * across;
    }
    const auto kernel = product_kernel<W, PHASE>;
    const int bytes = 2 * 4 * 64 * W * 32 * (int)sizeof(f16);
    RLT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), bytes, device->stream, all);
    return rlt_launch_status(device);
}
template <int W> int run(rlt_rocm_device* device, Matrices& all, int iterations) {
    size_t tiles = 0;
    for (int i = 0; i < all.n; i++) all.m[i].first = i * PARTS;
    hipLaunchKernelGGL(momentum_kernel, dim3(all.n * PARTS), dim3(256), 0, device->stream, all);
    int rc = rlt_launch_status(device);
    if (rc) return rc;
    for (int i = 0; i < all.n; i++) { all.m[i].first = (int)tiles; tiles += (size_t)all.m[i].M / 64 * (all.m[i].N / 64); }
    hipLaunchKernelGGL(normalise_kernel, dim3((unsigned)tiles), dim3(256), 0, device->stream, all);
    if ((rc = rlt_launch_status(device))) return rc;
    all.from = 0;
    for (int k = 0; k < iterations; k++, all.from ^= 1) {
        if ((rc = launch<W, GRAM>(device, all)) || (rc = launch<W, SQUARE>(device, all))) return rc;
        if ((rc = k + 1 < iterations ? launch<W, UPDATE>(device, all) : launch<W, LAST>(device, all))) return rc;
    }
    return 0;
}

}  // namespace

extern "C" {

size_t rlt_rocm_muon_workspace_bytes(const rlt_muon_tensor* tensors, int n) {
    if (!described(tensors, n) || !supported(tensors, n)) return 0;
    size_t bytes = 0;
    for (int i = 0; i < n; i++) bytes += bytes_of(tensors[i]);
    return bytes;
}

int rlt_rocm_muon_step(rlt_rocm_device* device, const rlt_muon_tensor* tensors, int n, const rlt_muon_parameters* parameters, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(tensors, n) && parameters && parameters->iterations > 0 && parameters->iterations <= MAX_ITERATIONS && parameters->epsilon >= 0.0f);
    for (int i = 0; i < n; i++) {
        const rlt_muon_tensor& t = tensors[i];
        RLT_REQUIRE(t.parameters && t.gradient && t.momentum && t.next_parameters && t.next_momentum && t.next_momentum != t.gradient && t.next_parameters != t.gradient && t.next_parameters != t.next_momentum &&
                    t.next_parameters != t.momentum && t.next_momentum != t.parameters);
        for (int j = 0; j < i; j++) RLT_REQUIRE(t.next_parameters != tensors[j].next_parameters && t.next_momentum != tensors[j].next_momentum);      // a matrix twice
    }
    if (!supported(tensors, n)) return RLT_E_UNSUPPORTED;
    RLT_REQUIRE(workspace && workspace_bytes >= rlt_rocm_muon_workspace_bytes(tensors, n) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
    char* at = (char*)workspace;
    for (int width = 1; width <= 2; width++) {
        Matrices all{};
        all.momentum = parameters->momentum; all.epsilon = parameters->epsilon; all.keep = 1.0f - parameters->alpha * parameters->weight_decay; all.nesterov = parameters->nesterov;
        for (int i = 0; i < n; i++) {
            const rlt_muon_tensor& t = tensors[i];
            if (width_of(t) == width) {
                Matrix& m = all.m[all.n++];
                const int tile = 64 * width, low = t.rows < t.cols ? t.rows : t.cols, high = t.rows < t.cols ? t.cols : t.rows;
                m.w = t.parameters; m.g = t.gradient; m.m = t.momentum; m.next_w = t.next_parameters; m.next_m = t.next_momentum;
                m.rows = t.rows; m.cols = t.cols; m.M = filled(low, tile); m.N = filled(high, tile);
                m.factor = parameters->alpha * sqrtf(t.rows > t.cols ? (float)t.rows / t.cols : 1.0f);
                const size_t plane = (size_t)m.M * m.N, square = (size_t)m.M * m.M;
                m.sums = (double*)at; at += PARTS * sizeof(double);
                f16* p = (f16*)at;
                m.x = p; m.t[0] = p + 2 * plane; m.t[1] = p + 4 * plane; m.a = p + 6 * plane; m.b = m.a + 2 * square;
                at = (char*)(m.b + 2 * square);
            }
            if (all.n == GROUP || (i == n - 1 && all.n)) {
                const int rc = width == 2 ? run<2>(device, all, parameters->iterations) : run<1>(device, all, parameters->iterations);
                if (rc) return rc;
                all.n = 0;
            }
        }
    }
    return 0;
}

}  // extern "C"
