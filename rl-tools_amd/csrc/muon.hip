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
};
struct Matrices {
    Matrix m[GROUP];
    int first[GROUP];             // workgroups of a launch before each matrix's
    int n, from;                  // from: which transpose is read
    int blocks;
    float momentum, epsilon, keep;      // keep: 1 - alpha * weight_decay
    int nesterov;
};
__device__ __forceinline__ const Matrix& matrix_of(const Matrices& all, int& block) {
    const int lane = threadIdx.x & 63, i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < all.n && all.first[lane < GROUP ? lane : 0] <= block)) - 1);
    block -= all.first[i];
    return all.m[i];
}
// consecutive workgroups go round the XCDs: those that read the same rows to one XCD, whose L2 they share. Beyond the last: -1
__device__ __forceinline__ int block_of(const Matrices& all) {
    const int per = (all.blocks + 7) / 8, block = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    return block < all.blocks ? block : -1;
}
__device__ __forceinline__ void split(float v, f16& high, f16& low) { high = (f16)v; low = (f16)(v - (float)high); }

// The momentum, and the sum of the update's squares in 64 bits (no square of an fp32 number leaves their range). VECTORS: four elements at a time, where all buffers start on 16-byte boundaries.
template <bool VECTORS> __device__ __forceinline__ double momentum(const Matrices& all, const Matrix& a, int part) {
    constexpr int V = VECTORS ? 4 : 1, AHEAD = 4;
    typedef float vector __attribute__((ext_vector_type(V)));
    const size_t size = (size_t)a.rows * a.cols / V, step = (size_t)PARTS * 256;
    double s = 0.0;
    auto one = [&](vector g, vector m, size_t i) {
        vector next;
#pragma unroll
        for (int e = 0; e < V; e++) {
            next[e] = fmaf(all.momentum, m[e], g[e]);
            const double u = all.nesterov ? fmaf(all.momentum, next[e], g[e]) : next[e];
            s = fma(u, u, s);
        }
        reinterpret_cast<vector*>(a.next_m)[i] = next;
    };
    size_t i = (size_t)part * 256 + threadIdx.x;
    for (; i + (AHEAD - 1) * step < size; i += AHEAD * step) {
        vector g[AHEAD], m[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) { g[j] = reinterpret_cast<const vector*>(a.g)[i + j * step]; m[j] = reinterpret_cast<const vector*>(a.m)[i + j * step]; }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) one(g[j], m[j], i + j * step);
    }
    for (; i < size; i += step) one(reinterpret_cast<const vector*>(a.g)[i], reinterpret_cast<const vector*>(a.m)[i], i);
    return s;
}
__global__ __launch_bounds__(256) void momentum_kernel(Matrices all) {
    __shared__ double sums[4];
    int block = blockIdx.x;
    const Matrix& a = matrix_of(all, block);
    const bool vectors = ((reinterpret_cast<uintptr_t>(a.g) | reinterpret_cast<uintptr_t>(a.m) | reinterpret_cast<uintptr_t>(a.next_m)) & 15) == 0 && (size_t)a.rows * a.cols % 4 == 0;
    double s = vectors ? momentum<true>(all, a, block) : momentum<false>(all, a, block);
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
// diagonal, written twice); UPDATE: a X + (b A + c A A) X; LAST: the same, straight into the parameters. What comes from memory waits in registers for DEPTH stages of 32 k.
enum Phase { GRAM, SQUARE, UPDATE, LAST };
template <int W> constexpr int DEPTH = W == 1 ? 4 : W == 2 ? 2 : 1;
template <int W, int PHASE> __global__ __launch_bounds__(256, W < 3 ? 2 : 1) void product_kernel(Matrices all) {
    constexpr int T = 64 * W, BK = 32, ROWS = 4 * T, LOADS = ROWS * 4 / 256;      // rows of the tile in LDS: P high, P low, Q high, Q low
    extern __shared__ __attribute__((aligned(16))) f16 lds[];      // [2][ROWS][BK], chunks of eight changed about within a row so that the rows that are read together lie in different banks
    int block = block_of(all);
    if (block < 0) return;
    const Matrix& a = matrix_of(all, block);
    const bool symmetric = PHASE == GRAM || PHASE == SQUARE;
    int ti, tj;
    if (symmetric) {
        ti = (int)((sqrtf(8.0f * block + 1.0f) - 1.0f) * 0.5f);
        while (ti * (ti + 1) / 2 > block) ti--;
        while ((ti + 1) * (ti + 2) / 2 <= block) ti++;
        tj = block - ti * (ti + 1) / 2;
    } else {      // eight rows of tiles at a time, column by column
        const int down = (a.M + T - 1) / T, across = (a.N + T - 1) / T, band = block / (8 * across), rows = min(8, down - band * 8), within = block - band * 8 * across;
        tj = within / rows; ti = band * 8 + within - tj * rows;
    }
    const int depth = PHASE == GRAM ? a.N : a.M;
    const f16* const P = PHASE == GRAM ? a.x : PHASE == SQUARE ? a.a : a.b; const f16* const Q = PHASE == GRAM ? a.x : PHASE == SQUARE ? a.a : a.t[all.from];
    const size_t square = (size_t)a.M * a.M, plane = (size_t)a.M * a.N, p_plane = PHASE == GRAM ? plane : square, q_plane = PHASE == SQUARE ? square : plane;
    const int q_rows = symmetric ? a.M : a.N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    const int row = threadIdx.x >> 2, chunk = threadIdx.x & 3;
    const unsigned own = (unsigned)row * depth + chunk * 8;
    f16x8 held[DEPTH<W>][LOADS];
    auto ask = [&](int k, f16x8 (&to)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int part = i / W, down = (part < 2 ? ti : tj) * T + i % W * 64, at_row = down < (part < 2 ? a.M : q_rows) ? down : 0;      // rows beyond the matrix: any that are there, nobody reads their sums
            const f16* const from = (part < 2 ? P + (part & 1) * p_plane : Q + (part & 1) * q_plane) + (size_t)at_row * depth + k;
            to[i] = *reinterpret_cast<const f16x8*>(from + own);
        }
    };
    f32x16 sum[W][W];
#pragma unroll
    for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < W; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum[i][j][e] = 0.0f;
    auto multiply = [&](const f16* from) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; kk++) {
            auto fragment = [&](int part, int tile) {
                const int r = part * T + tile * 32 + (lane & 31);
                return *reinterpret_cast<const f16x8*>(from + r * BK + ((kk * 2 + (lane >> 5)) ^ (r >> 1 & 3)) * 8);
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
    };
#pragma unroll
    for (int d = 0; d < DEPTH<W>; d++) if (d * BK < depth) ask(d * BK, held[d]);
    int turn = 0;
    for (int k0 = 0; k0 < depth; k0 += DEPTH<W> * BK) {
#pragma unroll
        for (int d = 0; d < DEPTH<W>; d++) {
            const int k = k0 + d * BK;
            if (k >= depth) break;
            f16* const to = lds + turn * ROWS * BK;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int r = i * 64 + row;
                *reinterpret_cast<f16x8*>(to + r * BK + (chunk ^ (r >> 1 & 3)) * 8) = held[d][i];
            }
            if (k + DEPTH<W> * BK < depth) ask(k + DEPTH<W> * BK, held[d]);
            rlt_lds_barrier();
            multiply(to);
            turn ^= 1;
        }
    }
    // a lane has column lane % 32 and, four by four, rows of its tiles
#pragma unroll
    for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            const int c = tj * T + (wj * W + j) * 32 + (lane & 31);
            if (ti * T + (wi * W + i) * 32 >= a.M || tj * T + (wj * W + j) * 32 >= q_rows) continue;
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
int filled(int n) { return (n + 63) / 64 * 64; }
size_t bytes_of(const rlt_muon_tensor& t) {
    const size_t M = filled(t.rows < t.cols ? t.rows : t.cols), N = filled(t.rows < t.cols ? t.cols : t.rows);
    return PARTS * sizeof(double) + (6 * M * N + 4 * M * M) * sizeof(f16);
}
template <int W, int PHASE> size_t tiles_of(const Matrix& m) {
    const size_t down = (m.M + 64 * W - 1) / (64 * W), across = (m.N + 64 * W - 1) / (64 * W);
    return PHASE == GRAM || PHASE == SQUARE ? down * (down + 1) / 2 : down * across;
}
template <int W, int PHASE> size_t tiles_of(const Matrices& all) {
    size_t n = 0;
    for (int i = 0; i < all.n; i++) n += tiles_of<W, PHASE>(all.m[i]);
    return n;
}
template <int W, int PHASE> int launch_width(rlt_rocm_device* device, Matrices& all) {
    size_t blocks = 0;
    for (int i = 0; i < all.n; i++) { all.first[i] = (int)blocks; blocks += tiles_of<W, PHASE>(all.m[i]); }
    all.blocks = (int)blocks;
    const auto kernel = product_kernel<W, PHASE>;
    const int bytes = 2 * 4 * 64 * W * 32 * (int)sizeof(f16);
    RLT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks + 7) / 8 * 8), dim3(256), bytes, device->stream, all);
    return rlt_launch_status(device);
}
// Tiles as wide as leave the fewest rounds over the compute units, a round's time as measured per tile.
template <int PHASE> int launch(rlt_rocm_device* device, Matrices& all) {
    const size_t units = device->compute_units > 0 ? device->compute_units : 256;
    auto rounds = [&](size_t tiles) { return (double)((tiles + units - 1) / units); };
    const double cost[4] = {rounds(tiles_of<1, PHASE>(all)) * 2.5, rounds(tiles_of<2, PHASE>(all)) * 6.2, rounds(tiles_of<3, PHASE>(all)) * 11.3, rounds(tiles_of<4, PHASE>(all)) * 18.8};
    int best = 0;
    for (int i = 1; i < 4; i++) if (cost[i] < cost[best]) best = i;
    return best == 0 ? launch_width<1, PHASE>(device, all) : best == 1 ? launch_width<2, PHASE>(device, all) : best == 2 ? launch_width<3, PHASE>(device, all) : launch_width<4, PHASE>(device, all);
}
int run(rlt_rocm_device* device, Matrices& all, int iterations) {
    size_t tiles = 0;
    for (int i = 0; i < all.n; i++) all.first[i] = i * PARTS;
    hipLaunchKernelGGL(momentum_kernel, dim3(all.n * PARTS), dim3(256), 0, device->stream, all);
    int rc = rlt_launch_status(device);
    if (rc) return rc;
    for (int i = 0; i < all.n; i++) { all.first[i] = (int)tiles; tiles += (size_t)all.m[i].M / 64 * (all.m[i].N / 64); }
    hipLaunchKernelGGL(normalise_kernel, dim3((unsigned)tiles), dim3(256), 0, device->stream, all);
    if ((rc = rlt_launch_status(device))) return rc;
    all.from = 0;
    for (int k = 0; k < iterations; k++, all.from ^= 1) {
        if ((rc = launch<GRAM>(device, all)) || (rc = launch<SQUARE>(device, all))) return rc;
        if ((rc = k + 1 < iterations ? launch<UPDATE>(device, all) : launch<LAST>(device, all))) return rc;
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
    Matrices all{};
    all.momentum = parameters->momentum; all.epsilon = parameters->epsilon; all.keep = 1.0f - parameters->alpha * parameters->weight_decay; all.nesterov = parameters->nesterov;
    for (int i = 0; i < n; i++) {
        const rlt_muon_tensor& t = tensors[i];
        Matrix& m = all.m[all.n++];
        m.w = t.parameters; m.g = t.gradient; m.m = t.momentum; m.next_w = t.next_parameters; m.next_m = t.next_momentum;
        m.rows = t.rows; m.cols = t.cols; m.M = filled(t.rows < t.cols ? t.rows : t.cols); m.N = filled(t.rows < t.cols ? t.cols : t.rows);
        m.factor = parameters->alpha * sqrtf(t.rows > t.cols ? (float)t.rows / t.cols : 1.0f);
        const size_t plane = (size_t)m.M * m.N, square = (size_t)m.M * m.M;
        m.sums = (double*)at; at += PARTS * sizeof(double);
        f16* const p = (f16*)at;
        m.x = p; m.t[0] = p + 2 * plane; m.t[1] = p + 4 * plane; m.a = p + 6 * plane; m.b = m.a + 2 * square;
        at = (char*)(m.b + 2 * square);
        if (all.n == GROUP || i == n - 1) {
            const int rc = run(device, all, parameters->iterations);
            if (rc) return rc;
            all.n = 0;
        }
    }
    return 0;
}

}  // extern "C"
