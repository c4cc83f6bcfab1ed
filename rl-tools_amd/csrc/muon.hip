// Optimiser step for matrices whose updates are orthogonalised by products: A = X X^T, X <- a X + (b A + c A A) X, a few times.
#include "typed.h"
#include <algorithm>

namespace {

// Factors are held as two numbers of 16 bits, the value's nearest and LOW times what it leaves: 22 bits and a sign, where fp32 has 24, for a third of the 16-bit rate in the matrix instructions; fp32 instructions have a sixteenth. Products are
// high x high, high x low and low x high, summed up in fp32; what is dropped, low x low and the rounding of the low part, is 2^-24.6 of a product in the mean (fp32's own rounding of a factor: 2^-25.3). Over the whole update the error is fp32's, most of
// it from the sums (512 x 1,024: 1.3e-6 of it, 2.0e-6 with fp32 products).
// Values are held times SCALE. Singular values stay below 1.21, those of A below 1.47, those of b A + c A A above -2.81 and below 0, so that no element leaves the range of 16 bits. At its lower end the two parts do: elements keep their 22 bits down to
// 2^-25 of the update's norm and lose one for each factor of two below. LOW moves that end: 2^9 is where rows and columns far below the others are best (as they are, 2^0, 2^-16 of the norm; half of the rows of 512 x 1,024 times 1e-6 of the others: 5.6e-4 of
// theirs then, 1.1e-6 now, 4e-7 with fp32 products; times 1e-8: 5.6e-2 and 1.1e-4). Tiles whose registers hold one sum alone take the high parts times 2^-9 to the low ones, which costs such a product bits below 2^-20 of the factor's norm; more than 2^9
// loses more there than the low parts gain. With sums apart 2^11 would be better still, in a second walk over k, as the registers do not hold both: two matrices of 4,096 columns 21.0 ms, 17.2 with the factors (16.8 without).
typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef rlt_f32x4 f32x4;
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr float LOW = 512.0f, UNLOW = 1.0f / LOW;
constexpr float SCALE = 16384.0f, UNSCALE = 1.0f / 16384.0f, QA = 3.4445f, QB = -4.775f, QC = 2.0315f;
constexpr int GROUP = 24, MAX_SIDE = 1 << 16, MAX_ITERATIONS = 32, PARTS = 256;      // matrices of a launch; partial sums of a norm
constexpr int JOBS = 768;         // workgroups of a launch whose tiles are shared, at the most

// What a launch is told: 16 bytes for each of its matrices, which a wavefront reads in one trip to where the launch left them (a row of longer entries, found and then read, was two trips).
struct Entry {
    char* scratch;                // its part of the workspace, see Matrix
    uint16_t M, N;                // in 64s: M <= N, rows and columns, or columns and rows where there are more rows, filled up
    int first;                    // workgroups of the launch before this matrix's
};
static_assert(sizeof(Entry) == 16, "");
struct Tensor {
    const float* w; const float* g; const float* m; float* next_w; float* next_m;
    int rows, cols;
    float factor;                 // alpha * sqrt(max(1, rows / cols))
};
struct Entries {
    Entry e[GROUP];
    int n, from;                  // from: which transpose is read
    int length;                   // symmetric products: k that a workgroup adds up, a tile's others go to others
    float* parts;                 // their sums, by workgroups
};
struct Tensors { Tensor t[GROUP]; float momentum, epsilon, keep; int nesterov; };      // keep: 1 - alpha * weight_decay
struct Phases { Entries entries; };
struct Last { Entries entries; Tensors tensors; int iterations; };

// X [M x N], its transpose [N x M] (one that is read, one that is written), A and b A + c A A [M x M], the low parts behind the high ones; PARTS partial sums of u^2 ahead of them
#define GLOBAL __attribute__((address_space(1)))
struct Matrix {
    GLOBAL char* scratch; int M, N, index;
    __device__ __forceinline__ size_t plane() const { return (size_t)M * N; }
    __device__ __forceinline__ size_t square() const { return (size_t)M * M; }
    __device__ __forceinline__ const GLOBAL double* sums() const { return (const GLOBAL double*)scratch; }
    __device__ __forceinline__ GLOBAL f16* x() const { return (GLOBAL f16*)(scratch + PARTS * sizeof(double)); }
    __device__ __forceinline__ GLOBAL f16* t(int which) const { return x() + (which ? 4 : 2) * plane(); }
    __device__ __forceinline__ GLOBAL f16* a() const { return x() + 6 * plane(); }
    __device__ __forceinline__ GLOBAL f16* b() const { return a() + 2 * square(); }
};
__device__ __forceinline__ Matrix matrix_of(const Entries& all, int& block) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63;
    const i32x4 mine = *reinterpret_cast<const i32x4*>(&all.e[lane < GROUP ? lane : 0]);
    const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < all.n && mine[3] <= block)) - 1);
    const unsigned low = __builtin_amdgcn_readlane(mine[0], i), high = __builtin_amdgcn_readlane(mine[1], i), sizes = __builtin_amdgcn_readlane(mine[2], i);
    block -= __builtin_amdgcn_readlane(mine[3], i);
    return {(GLOBAL char*)((uint64_t)high << 32 | low), (int)(sizes & 0xFFFF) * 64, (int)(sizes >> 16) * 64, i};
}
// A matrix's tiles, of which a launch has workgroups for a multiple of eight: consecutive workgroups go round the XCDs, those that read the same rows to one XCD, whose L2 they share. Beyond the last: -1
__device__ __forceinline__ int tile_of(int block, int tiles) {
    const int tile = (block & 7) * ((tiles + 7) / 8) + (block >> 3);
    return block >> 3 < (tiles + 7) / 8 && tile < tiles ? tile : -1;
}
__device__ __forceinline__ void split(float v, f16& high, f16& low) { high = (f16)v; low = (f16)((v - (float)high) * LOW); }
__device__ __forceinline__ float whole(f16 high, f16 low) { return fmaf((float)low, UNLOW, (float)high); }

// The momentum, and the sum of the update's squares in 64 bits (no square of an fp32 number leaves their range). VECTORS: four elements at a time, where all buffers start on 16-byte boundaries. Memory bounds it (84 million
// elements: 172 us, 5.9 TB/s).
template <bool VECTORS> __device__ __forceinline__ double momentum(const Tensors& all, const Tensor& a, int part) {
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
__global__ __launch_bounds__(256) void momentum_kernel(Last launch) {
    __shared__ double sums[4];
    const Tensors& all = launch.tensors;
    const int block = blockIdx.x % PARTS, matrix = blockIdx.x / PARTS;
    const Tensor& a = all.t[matrix];
    const bool vectors = ((reinterpret_cast<uintptr_t>(a.g) | reinterpret_cast<uintptr_t>(a.m) | reinterpret_cast<uintptr_t>(a.next_m)) & 15) == 0 && (size_t)a.rows * a.cols % 4 == 0;
    double s = vectors ? momentum<true>(all, a, block) : momentum<false>(all, a, block);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)launch.entries.e[matrix].scratch)[block] = ((sums[0] + sums[1]) + sums[2]) + sums[3];
}

// X and its transpose, tiles of 64 x 64, zeros beyond the matrix; memory bounds it (84 million elements: 268 us, 5.0 TB/s)
__global__ __launch_bounds__(256) void normalise_kernel(Last launch) {
    __shared__ float tile[64][65];
    __shared__ double norms[4];
    int block = blockIdx.x;
    const Tensors& all = launch.tensors;
    const Matrix mat = matrix_of(launch.entries, block);
    const Tensor& a = all.t[mat.index];
    const bool tall = a.rows > a.cols;
    const int wide = tall ? mat.M : mat.N, high = tall ? mat.N : mat.M, across = wide / 64, r0 = block / across * 64, c0 = block % across * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float g[16], m[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int r = r0 + i * 4 + wave, c = c0 + lane;
        g[i] = m[i] = 0.0f;
        if (r < a.rows && c < a.cols) { g[i] = a.g[(size_t)r * a.cols + c]; m[i] = a.next_m[(size_t)r * a.cols + c]; }
    }
    double s = mat.sums()[threadIdx.x];
    static_assert(PARTS == 256, "");
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) norms[wave] = s;
    __syncthreads();
    const double inverse = (double)SCALE / (sqrt(((norms[0] + norms[1]) + norms[2]) + norms[3]) + (double)all.epsilon);
    GLOBAL f16* const rows = tall ? mat.t(0) : mat.x(); GLOBAL f16* const columns = tall ? mat.x() : mat.t(0);
    const size_t plane = mat.plane();
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int r = r0 + i * 4 + wave, c = c0 + lane;
        const float v = (float)((double)(all.nesterov ? fmaf(all.momentum, m[i], g[i]) : m[i]) * inverse);
        tile[i * 4 + wave][lane] = v;
        f16 h, l;
        split(v, h, l);
        rows[(size_t)r * wide + c] = h; rows[plane + (size_t)r * wide + c] = l;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) {
        f16 h, l;
        split(tile[lane][i * 4 + wave], h, l);
        columns[(size_t)(c0 + i * 4 + wave) * high + r0 + lane] = h; columns[plane + (size_t)(c0 + i * 4 + wave) * high + r0 + lane] = l;
    }
}

// C[i][j] = sum over k of P[i][k] Q[j][k], both with k side by side. GRAM: A = X X^T; SQUARE: b A + c A A (both symmetric: tiles on and below the diagonal, written twice); UPDATE: a X + (b A + c A A) X; LAST: the same,
// straight into the parameters.
enum Phase { GRAM, SQUARE, UPDATE, LAST };
template <int PHASE> constexpr bool SYMMETRIC = PHASE == GRAM || PHASE == SQUARE;
struct Product {
    const GLOBAL f16* P; const GLOBAL f16* Q; size_t p_plane, q_plane, square, plane;
    int depth, q_rows, ti, tj;
    int from, to, parts, job;     // the k of this workgroup; how many share the tile, and which of all jobs of the launch this is
};
template <int PHASE> struct ArgumentsOf { typedef Phases type; };
template <> struct ArgumentsOf<LAST> { typedef Last type; };
__device__ __forceinline__ const Tensors* tensors_of(const Phases&) { return nullptr; }
__device__ __forceinline__ const Tensors* tensors_of(const Last& launch) { return &launch.tensors; }
// which tile of `down` rows and `across` columns of tiles this is, and where its factors lie
template <int PHASE> __device__ __forceinline__ void place(const Matrix& a, int tile, int down, int across, int from, Product& p) {
    if (SYMMETRIC<PHASE>) {
        p.ti = (int)((sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f);
        while (p.ti * (p.ti + 1) / 2 > tile) p.ti--;
        while ((p.ti + 1) * (p.ti + 2) / 2 <= tile) p.ti++;
        p.tj = tile - p.ti * (p.ti + 1) / 2;
    } else {      // eight rows of tiles at a time, column by column
        const int band = tile / (8 * across), rows = min(8, down - band * 8), within = tile - band * 8 * across;
        p.tj = within / rows; p.ti = band * 8 + within - p.tj * rows;
    }
    p.square = a.square(); p.plane = a.plane();
    p.P = PHASE == GRAM ? a.x() : PHASE == SQUARE ? a.a() : a.b(); p.Q = PHASE == GRAM ? a.x() : PHASE == SQUARE ? a.a() : a.t(from);
    p.p_plane = PHASE == GRAM ? p.plane : p.square; p.q_plane = PHASE == SQUARE ? p.square : p.plane;
    p.q_rows = SYMMETRIC<PHASE> ? a.M : a.N;
}
template <int PHASE, int T> __device__ __forceinline__ bool product_of(const Entries& all, const Matrix& a, int block, Product& p) {
    const int down = (a.M + T - 1) / T, across = (a.N + T - 1) / T;
    p.depth = PHASE == GRAM ? a.N : a.M;
    p.parts = SYMMETRIC<PHASE> && T <= 128 ? (p.depth + all.length - 1) / all.length : 1;
    int tile = tile_of(block, (SYMMETRIC<PHASE> ? down * (down + 1) / 2 : down * across) * p.parts);
    if (tile < 0) return false;
    p.from = 0; p.to = p.depth; p.job = (int)blockIdx.x - block + tile;
    if (p.parts > 1) {
        const int part = tile % p.parts;
        tile /= p.parts;
        p.from = part * all.length; p.to = min(p.from + all.length, p.depth);
    }
    place<PHASE>(a, tile, down, across, all.from, p);
    return true;
}
// What becomes of a tile of 32 x 32. The sums come as the matrix instructions leave them, a column to a lane, and go through a square of LDS that belongs to the wavefront, so that memory sees eight elements of a row, or of a column, at a time
// (stores of single elements and of four, as they come: a launch over sixteen block matrices of 256 to 2,048 columns 46 us, so 38).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
constexpr int PITCH = 33;
typedef float Square[32 * PITCH];
struct Added { f16x8 high[2], low[2]; };      // of rows lane / 4 and lane / 4 + 16, columns lane % 4 * 8 and on: what the sums are added to
template <int PHASE> __device__ __forceinline__ void addends(const Matrix& a, const Product& p, int r0, int c0, Added& v) {
    if constexpr (PHASE != GRAM) {
        const int lane = threadIdx.x & 63;
        const GLOBAL f16* const from = PHASE == SQUARE ? a.a() : a.x();
        const size_t width = PHASE == SQUARE ? a.M : a.N, behind = PHASE == SQUARE ? p.square : p.plane;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const GLOBAL f16* const at = from + (size_t)(r0 + h * 16 + (lane >> 2)) * width + c0 + (lane & 3) * 8;
            v.high[h] = *(const GLOBAL f16x8*)at; v.low[h] = *(const GLOBAL f16x8*)(at + behind);
        }
    }
}
__device__ __forceinline__ void keep(const f32x16& sum, float* square) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < 16; e++) square[((e >> 2) * 8 + (lane >> 5) * 4 + (e & 3)) * PITCH + (lane & 31)] = sum[e];
}
// eight parameters from element `at` of a row on, of which `left` are there
__device__ __forceinline__ void step_parameters(const Tensors& all, const Tensor& t, size_t at, int left, const float (&v)[8]) {
    typedef float vector __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int half = 0; half < 2; half++, at += 4, left -= 4) {
        if (left >= 4) {
            const vector w = *reinterpret_cast<const vector*>(t.w + at);
            vector next;
#pragma unroll
            for (int e = 0; e < 4; e++) next[e] = fmaf(-t.factor, v[half * 4 + e] * UNSCALE, all.keep * w[e]);
            *reinterpret_cast<vector*>(t.next_w + at) = next;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) if (e < left) t.next_w[at + e] = fmaf(-t.factor, v[half * 4 + e] * UNSCALE, all.keep * t.w[at + e]);
        }
    }
}
template <int PHASE> __device__ __forceinline__ void finish(const Tensors* tensors, int from, const Matrix& a, const Product& p, int r0, int c0, float* square, const Added& added) {
    const int lane = threadIdx.x & 63, line = lane >> 2, chunk = (lane & 3) * 8;
    const bool tall = PHASE == LAST && tensors->t[a.index].rows > tensors->t[a.index].cols, turned = PHASE == UPDATE || (PHASE == LAST ? tall : p.ti != p.tj);
    GLOBAL f16* const out = PHASE == GRAM ? a.a() : PHASE == SQUARE ? a.b() : a.x();
    GLOBAL f16* const across = PHASE == UPDATE ? a.t(from ^ 1) : out;
    const size_t behind = PHASE == UPDATE ? p.plane : p.square, width = PHASE == UPDATE ? a.N : a.M;
    auto store = [&](GLOBAL f16* to, const float (&v)[8]) {
        f16x8 high, low;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            f16 h, l;
            split(v[e], h, l);
            high[e] = h; low[e] = l;
        }
        *(GLOBAL f16x8*)to = high; *(GLOBAL f16x8*)(to + behind) = low;
    };
    wave_sync();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = r0 + h * 16 + line, c = c0 + chunk;
        float* const own = square + (h * 16 + line) * PITCH + chunk;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = own[e] * UNSCALE;
            const float add = PHASE == GRAM ? 0.0f : whole(added.high[h][e], added.low[h][e]);
            if (PHASE == SQUARE) v[e] = fmaf(QC, v[e], QB * add);
            if (PHASE == UPDATE || PHASE == LAST) v[e] = fmaf(QA, add, v[e]);
            if (turned) own[e] = v[e];
        }
        if constexpr (PHASE == LAST) {
            const Tensor& t = tensors->t[a.index];
            if (!tall && r < t.rows) step_parameters(*tensors, t, (size_t)r * t.cols + c, t.cols - c, v);
        } else store(out + (size_t)r * width + c, v);
    }
    if (!turned) return;
    wave_sync();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int c = c0 + h * 16 + line, r = r0 + chunk;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = square[(chunk + e) * PITCH + h * 16 + line];
        if constexpr (PHASE == LAST) {
            const Tensor& t = tensors->t[a.index];
            if (c < t.rows) step_parameters(*tensors, t, (size_t)c * t.cols + r, t.cols - r, v);
        } else store(across + (size_t)c * a.M + r, v);
    }
}

// A tile whose k several workgroups share: each leaves its sums, and a launch behind adds them up, in the order of k. (The last workgroup of a tile to arrive did, which a ticket told it: the releases and acquires around the tickets write back and
// invalidate the XCDs' L2s, 25 us at 350 workgroups, where the launch costs 7.)
template <int W> __device__ __forceinline__ float* parts_of(const Entries& all, int job) { return all.parts + (size_t)job * (64 * W) * (64 * W) + threadIdx.x * 4; }      // tiles of 32 x 32 of the wavefronts, four sums of a lane at a time
template <int W> __device__ __forceinline__ void leave(const Entries& all, const Product& p, int i, const f32x16& v) {
    float* const to = parts_of<W>(all, p.job) + i * 4096;
#pragma unroll
    for (int e = 0; e < 4; e++) *reinterpret_cast<f32x4*>(to + e * 1024) = f32x4{v[e * 4], v[e * 4 + 1], v[e * 4 + 2], v[e * 4 + 3]};
}
template <int W> __device__ __forceinline__ f32x16 joined(const Entries& all, const Product& p, int i) {
    const float* from = parts_of<W>(all, p.job) + i * 4096;
    f32x16 total;
#pragma unroll
    for (int e = 0; e < 16; e++) total[e] = 0.0f;
    for (int part = 0; part < p.parts; part++, from += (64 * W) * (64 * W)) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(from + e * 1024);
#pragma unroll
            for (int n = 0; n < 4; n++) total[e * 4 + n] += v[n];
        }
    }
    return total;
}

// Tiles of 64 x 64, for few of them: a launch is bound by trips to memory then. What 128 k need is on its way ahead, what the sums are added to with it; four wavefronts have 32 x 32 of the tile each, factors come through LDS in stages of
// 64 k, and the three kinds of products have sums of their own, which are joined at the end: a chain of dependent matrix instructions is a third as long.
typedef f16 SmallStage[256 * 64];      // rows of P high, P low, Q high, Q low; chunks of eight changed about within a row
template <int PHASE> __device__ __forceinline__ f32x16 small_sums(SmallStage* lds, const Matrix& a, const Product& p, int r0, int c0, Added& added) {
    constexpr int BK = 64, LOADS = 8, DEPTH = 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = threadIdx.x >> 3, chunk = threadIdx.x & 7;
    const GLOBAL char* const p0 = (const GLOBAL char*)(p.P + (size_t)p.ti * 64 * p.depth); const GLOBAL char* const q0 = (const GLOBAL char*)(p.Q + (size_t)p.tj * 64 * p.depth);
    const unsigned own = (row * p.depth + chunk * 8) * (unsigned)sizeof(f16);
    f16x8 held[DEPTH][LOADS];
    auto ask = [&](int k, f16x8 (&to)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; i++)
            to[i] = *(const GLOBAL f16x8*)((i < 4 ? p0 + (i >> 1 & 1) * p.p_plane * sizeof(f16) : q0 + (i >> 1 & 1) * p.q_plane * sizeof(f16)) + ((size_t)(i & 1) * 32 * p.depth + k) * sizeof(f16) + own);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++) ask(min(p.from + d * BK, p.to - BK), held[d]);      // (the last stage again where there are no more: a branch around a load waits for it)
    addends<PHASE>(a, p, r0, c0, added);
    f32x16 sum[3];
#pragma unroll
    for (int i = 0; i < 3; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) sum[i][e] = 0.0f;
#pragma unroll 1
    for (int k0 = p.from; k0 < p.to; k0 += DEPTH * BK) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int k = k0 + d * BK;
            if (k >= p.to) break;
            f16* const to = lds[d & 1];
#pragma unroll
            for (int i = 0; i < LOADS; i++) *reinterpret_cast<f16x8*>(to + (i * 32 + row) * BK + (chunk ^ (row & 7)) * 8) = held[d][i];
            ask(min(k + DEPTH * BK, p.to - BK), held[d]);
            rlt_lds_barrier();
#pragma unroll
            for (int kk = 0; kk < BK / 16; kk++) {
                auto fragment = [&](int part, int half) {
                    const int r = part * 64 + half * 32 + (lane & 31);
                    return *reinterpret_cast<const f16x8*>(to + r * BK + ((kk * 2 + (lane >> 5)) ^ (r & 7)) * 8);
                };
                const f16x8 ph = fragment(0, wave >> 1), pl = fragment(1, wave >> 1), qh = fragment(2, wave & 1), ql = fragment(3, wave & 1);
                sum[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, sum[0], 0, 0, 0);
                sum[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, sum[1], 0, 0, 0);
                sum[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, sum[2], 0, 0, 0);
            }
        }
    }
    return sum[0] + (sum[1] + sum[2]) * UNLOW;
}
template <int PHASE> __global__ __launch_bounds__(256, SYMMETRIC<PHASE> ? 2 : 1) void product_small_kernel(typename ArgumentsOf<PHASE>::type launch) {
    __shared__ __attribute__((aligned(16))) SmallStage lds[2];
    int block = blockIdx.x;
    const Matrix a = matrix_of(launch.entries, block);
    Product p;
    if (!product_of<PHASE, 64>(launch.entries, a, block, p)) return;
    const int wave = threadIdx.x >> 6, r0 = p.ti * 64 + (wave >> 1) * 32, c0 = p.tj * 64 + (wave & 1) * 32;
    Added added;
    const f32x16 total = small_sums<PHASE>(lds, a, p, r0, c0, added);
    if (p.parts > 1) { leave<1>(launch.entries, p, 0, total); return; }
    float* const square = reinterpret_cast<Square*>(lds)[wave];
    rlt_lds_barrier();      // the stages are read
    keep(total, square);
    finish<PHASE>(tensors_of(launch), launch.entries.from, a, p, r0, c0, square, added);
}

// Tiles of 64 W x 64 W: four wavefronts share one, each has W x W tiles of 32 x 32, factors come through LDS in stages of 32 k. Half a stage ahead: while the products of one half run, the other half's factors come from LDS, the next stage's go there
// and the one after that is asked for, dealt out between the matrix instructions. 256 x 256: 1,100 to 1,126 TFLOP/s of 16-bit products at 4,096 x 20,480 x 4,096 (the clock is down to 1.6 GHz by then; a large library product: 1,080 to 1,135); the order brought 867 to 1,054 of
// it, before high parts were scaled for the low ones (1,138 without). 65 registers a lane wait in scratch memory for what comes behind the loop; none is read within it.
template <int W, int PHASE> __global__ __launch_bounds__(256, W < 3 ? 2 : 1) void product_kernel(typename ArgumentsOf<PHASE>::type launch) {
    constexpr int T = 64 * W, BK = 32, ROWS = 4 * T, LOADS = ROWS * 4 / 256, PRODUCTS = 3 * W * W, READS = 4 * W;      // rows of the tile in LDS: P high, P low, Q high, Q low
    extern __shared__ __attribute__((aligned(16))) f16 lds[];      // [2][ROWS][BK], chunks of eight changed about within a row so that the rows that are read together lie in different banks
    int block = blockIdx.x;
    const Matrix a = matrix_of(launch.entries, block);
    Product p;
    if (!product_of<PHASE, T>(launch.entries, a, block, p)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    const int row = threadIdx.x >> 2, chunk = threadIdx.x & 3;
    const unsigned own = (row * p.depth + chunk * 8) * (unsigned)sizeof(f16);
    f16x8 held[LOADS];
    auto ask = [&](int k) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int part = i / W, down = (part < 2 ? p.ti : p.tj) * T + i % W * 64, at_row = down < (part < 2 ? a.M : p.q_rows) ? down : 0;      // rows beyond the matrix: any that are there, nobody reads their sums
            const GLOBAL f16* const from = (part < 2 ? p.P + (part & 1) * p.p_plane : p.Q + (part & 1) * p.q_plane) + (size_t)at_row * p.depth + k;
            held[i] = *(const GLOBAL f16x8*)((const GLOBAL char*)from + own);
        }
    };
    f32x16 sum[W][W];
#pragma unroll
    for (int i = 0; i < W; i++)
#pragma unroll
        for (int j = 0; j < W; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum[i][j][e] = 0.0f;
    struct Fragments { f16x8 ph[W], pl[W], qh[W], ql[W]; };
    auto read = [&](const f16* from, int kk, Fragments& f) {
        auto fragment = [&](int part, int tile) {
            const int r = part * T + tile * 32 + (lane & 31);
            return *reinterpret_cast<const f16x8*>(from + r * BK + ((kk * 2 + (lane >> 5)) ^ (r >> 1 & 3)) * 8);
        };
#pragma unroll
        for (int i = 0; i < W; i++) {
            f.ph[i] = fragment(0, wi * W + i); f.pl[i] = fragment(1, wi * W + i);
            f.qh[i] = fragment(2, wj * W + i); f.ql[i] = fragment(3, wj * W + i);
        }
    };
    auto multiply = [&](const Fragments& f) {      // the high parts of products with low ones by 1 / LOW; sums that follow each other in the matrix pipeline are not the same
        f16x8 p[W], q[W];
#pragma unroll
        for (int term = 0; term < 3; term++) {
#pragma unroll
            for (int i = 0; i < W; i++) { p[i] = term == 0 ? f.pl[i] : term == 1 ? f.ph[i] * (f16)UNLOW : f.ph[i]; q[i] = term == 0 ? f.qh[i] * (f16)UNLOW : term == 1 ? f.ql[i] : f.qh[i]; }
#pragma unroll
            for (int i = 0; i < W; i++)
#pragma unroll
                for (int j = 0; j < W; j++) sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i], q[j], sum[i][j], 0, 0, 0);
        }
    };
    auto put = [&](f16* to) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int r = i * 64 + row;
            *reinterpret_cast<f16x8*>(to + r * BK + (chunk ^ (r >> 1 & 3)) * 8) = held[i];
        }
    };
    f16* here = lds; f16* there = lds + ROWS * BK;
    Fragments first, second;
    ask(p.from);
    put(here);
    ask(p.from + BK);
    rlt_lds_barrier();
    read(here, 0, first);
    const int stages = (p.to - p.from) / BK;      // two at the least
    for (int s = 0; s + 1 < stages; s++) {
        read(here, 1, second);
        multiply(first);
        put(there);
        ask(p.from + min(s + 2, stages - 1) * BK);
#pragma unroll
        for (int i = 0; i < READS; i++) { __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); }
        constexpr int LEFT = PRODUCTS > READS ? (PRODUCTS - READS) / LOADS : 0;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0); __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
            if (LEFT) __builtin_amdgcn_sched_group_barrier(0x8, LEFT, 0);
        }
        rlt_lds_barrier();
        read(there, 0, first);
        multiply(second);
#pragma unroll
        for (int i = 0; i < READS; i++) { __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); }
        f16* const t = here; here = there; there = t;
    }
    read(here, 1, second);
    multiply(first);
    multiply(second);
    if constexpr (W == 2 && SYMMETRIC<PHASE>) {
        if (p.parts > 1) {
#pragma unroll
            for (int i = 0; i < W * W; i++) leave<W>(launch.entries, p, i, sum[i / W][i % W]);
            return;
        }
    }
    // sums go through LDS, a row of tiles at a time: one copy of what is done with a tile, whose needs are no more than a tile's
    rlt_lds_barrier();
    Square* const squares = reinterpret_cast<Square*>(lds) + wave * W;
#pragma unroll
    for (int i = 0; i < W; i++) {
#pragma unroll
        for (int j = 0; j < W; j++) keep(sum[i][j], squares[j]);
#pragma unroll 1
        for (int j = 0; j < W; j++) {
            const int r0 = p.ti * T + (wi * W + i) * 32, c0 = p.tj * T + (wj * W + j) * 32;
            if (r0 >= a.M || c0 >= p.q_rows) continue;
            Added added;
            addends<PHASE>(a, p, r0, c0, added);
            finish<PHASE>(tensors_of(launch), launch.entries.from, a, p, r0, c0, squares[j], added);
        }
        wave_sync();
    }
}

// the sums of tiles that workgroups shared: a workgroup for every tile of 32 x 32 of each wavefront
template <int W, int PHASE> __global__ __launch_bounds__(256) void join_kernel(Phases launch) {
    __shared__ Square squares[4];
    int block = blockIdx.x / (W * W);
    const int i = blockIdx.x % (W * W), job = block, wave = threadIdx.x >> 6;
    const Matrix a = matrix_of(launch.entries, block);
    Product p;
    if (!product_of<PHASE, 64 * W>(launch.entries, a, block, p) || p.parts == 1 || p.from) return;      // (the job of a tile's first k stands for the tile)
    const int r0 = p.ti * 64 * W + ((wave >> 1) * W + i / W) * 32, c0 = p.tj * 64 * W + ((wave & 1) * W + i % W) * 32;
    if (r0 >= a.M || c0 >= p.q_rows) return;
    p.job += job - (int)blockIdx.x;
    Added added;
    addends<PHASE>(a, p, r0, c0, added);
    keep(joined<W>(launch.entries, p, i), squares[wave]);
    finish<PHASE>(tensors_of(launch), launch.entries.from, a, p, r0, c0, squares[wave], added);
}

// The whole step of matrices with a side of up to 64 and another of up to 256, a workgroup each: X, its transpose and A, or b A + c A A in A's place, stay in LDS, and a kind of products costs two barriers where it would be a launch (64 x 64: 20 us
// where the launches take 66; 64 x 256: 52 and 78). Where a larger matrix is in the call, the launches are there all the same and take the small ones along.
constexpr int LOCAL_COLUMNS = 4;      // in 64s
int local_bytes(int columns) { return (4 * 64 * columns * 64 + 2 * 64 * 64) * (int)sizeof(f16); }
__global__ __launch_bounds__(1024) void local_kernel(Last launch) {
    extern __shared__ __attribute__((aligned(16))) f16 lds[];
    __shared__ double norms[16];
    const Tensors& all = launch.tensors;
    const Tensor& a = all.t[blockIdx.x];
    const int N = launch.entries.e[blockIdx.x].N * 64, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f16* const x = lds; f16* const t = x + 128 * N; f16* const square = t + 128 * N;      // [64][N], [N][64] and [64][64], the low parts behind the high ones; chunks of eight changed about within a row
    auto at = [](int row, int k, int width) { return row * width + ((k >> 3) ^ (row >> 1 & 7)) * 8 + (k & 7); };
    const bool tall = a.rows > a.cols;
    const int across = tall ? 1 : N / 64, units = (tall ? N : 64) * across;      // 64 elements of a row, filled up
    constexpr int AHEAD = 4;
    float held[AHEAD];      // the first of a wavefront's updates; those behind them are worked out twice
    double s = 0.0;
    auto updates = [&](int u0, bool first) {
        float g[AHEAD], m[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int u = u0 + 16 * j, r = u / across, c = u % across * 64 + lane;
            const bool there = r < a.rows && c < a.cols;
            const size_t i = (size_t)r * a.cols + c;
            g[j] = there ? a.g[i] : 0.0f;
            m[j] = there ? (first ? a.m : a.next_m)[i] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int u = u0 + 16 * j, r = u / across, c = u % across * 64 + lane;
            const float next = first ? fmaf(all.momentum, m[j], g[j]) : m[j];
            if (first && r < a.rows && c < a.cols) a.next_m[(size_t)r * a.cols + c] = next;
            g[j] = all.nesterov ? fmaf(all.momentum, next, g[j]) : next;
            if (first) s = fma((double)g[j], (double)g[j], s);
        }
        if (!first || u0 == wave) {
#pragma unroll
            for (int j = 0; j < AHEAD; j++) held[j] = g[j];
        }
    };
    for (int u0 = wave; u0 < units; u0 += 16 * AHEAD) updates(u0, true);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) norms[wave] = s;
    __syncthreads();
    double sum_of_norms = 0.0;
#pragma unroll
    for (int w = 0; w < 16; w++) sum_of_norms += norms[w];
    const double inverse = (double)SCALE / (sqrt(sum_of_norms) + (double)all.epsilon);
    for (int u0 = wave; u0 < units; u0 += 16 * AHEAD) {
        if (u0 != wave) updates(u0, false);
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int u = u0 + 16 * j, pr = u / across, pc = u % across * 64 + lane, r = tall ? pc : pr, c = tall ? pr : pc;
            f16 h, l;
            split((float)((double)held[j] * inverse), h, l);
            x[at(r, c, N)] = h; x[64 * N + at(r, c, N)] = l;
            t[at(c, r, 64)] = h; t[64 * N + at(c, r, 64)] = l;
        }
    }
    __syncthreads();

    // sums over k of 16 rows of P and 16 of Q, in three kinds
    auto product = [&](const f16* P, int p_low, int p_row, const f16* Q, int q_low, int q_row, int depth) {
        f32x4 sum[3];
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[i][e] = 0.0f;
        const f16* const ps = P + (p_row + (lane & 15)) * depth; const f16* const qs = Q + (q_row + (lane & 15)) * depth;
#pragma unroll 2
        for (int k = 0; k < depth / 8; k += 4) {
            const int chunk = ((k + (lane >> 4)) ^ (lane >> 1 & 7)) * 8;
            const f16x8 ph = *reinterpret_cast<const f16x8*>(ps + chunk), pl = *reinterpret_cast<const f16x8*>(ps + p_low + chunk);
            const f16x8 qh = *reinterpret_cast<const f16x8*>(qs + chunk), ql = *reinterpret_cast<const f16x8*>(qs + q_low + chunk);
            sum[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, sum[0], 0, 0, 0);
            sum[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, sum[1], 0, 0, 0);
            sum[2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, sum[2], 0, 0, 0);
        }
        return sum[0] + (sum[1] + sum[2]) * UNLOW;
    };
    // A lane has a column and, four by four, rows of it: column c of the sums as row c of what is written, which for A and b A + c A A is the same (sums are alike on both sides of the diagonal, bit by bit).
    typedef f16 f16x4 __attribute__((ext_vector_type(4)));
    auto get = [&](const f16* from, int low, int r, int c, float (&v)[4]) {
        const f16x4 h = *reinterpret_cast<const f16x4*>(from + at(c, r, 64)), l = *reinterpret_cast<const f16x4*>(from + low + at(c, r, 64));
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = whole(h[e], l[e]);
    };
    auto put = [&](f16* to, int low, int r, int c, const float (&v)[4], f16x4& high, f16x4& rest) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f16 h, l;
            split(v[e], h, l);
            high[e] = h; rest[e] = l;
        }
        *reinterpret_cast<f16x4*>(to + at(c, r, 64)) = high; *reinterpret_cast<f16x4*>(to + low + at(c, r, 64)) = rest;
    };
    const int r0 = (wave >> 2) * 16, c0 = (wave & 3) * 16, r = r0 + (lane >> 4) * 4, c = c0 + (lane & 15);
    for (int k = 0; k < launch.iterations; k++) {
        f16x4 high, rest;
        f32x4 total = product(x, 64 * N, r0, x, 64 * N, c0, N);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = total[e] * UNSCALE;
        put(square, 4096, r, c, v, high, rest);
        __syncthreads();
        total = product(square, 4096, r0, square, 4096, c0, 64);
        get(square, 4096, r, c, v);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = fmaf(QC, total[e] * UNSCALE, QB * v[e]);
        __syncthreads();
        put(square, 4096, r, c, v, high, rest);
        __syncthreads();
        // a wavefront has a tile of 16 x 16 in each 64 columns
        float next[LOCAL_COLUMNS][4];
#pragma unroll
        for (int i = 0; i < LOCAL_COLUMNS; i++)
            if (i * 64 < N) {
                total = product(square, 4096, r0, t, 64 * N, i * 64 + c0, 64);
                get(t, 64 * N, r, i * 64 + c, next[i]);
#pragma unroll
                for (int e = 0; e < 4; e++) next[i][e] = fmaf(QA, next[i][e], total[e] * UNSCALE);
            }
        __syncthreads();
        if (k + 1 < launch.iterations) {
#pragma unroll
            for (int i = 0; i < LOCAL_COLUMNS; i++)
                if (i * 64 < N) {
                    put(t, 64 * N, r, i * 64 + c, next[i], high, rest);
#pragma unroll
                    for (int e = 0; e < 4; e++) { x[at(r + e, i * 64 + c, N)] = high[e]; x[64 * N + at(r + e, i * 64 + c, N)] = rest[e]; }
                }
            __syncthreads();
            continue;
        }
#pragma unroll
        for (int i = 0; i < LOCAL_COLUMNS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = tall ? i * 64 + c : r + e, column = tall ? r + e : i * 64 + c;
                if (i * 64 < N && row < a.rows && column < a.cols) {
                    const size_t j = (size_t)row * a.cols + column;
                    a.next_w[j] = fmaf(-a.factor, next[i][e] * UNSCALE, all.keep * a.w[j]);
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
constexpr size_t SHARED_BYTES = (size_t)JOBS / 2 * 128 * 128 * sizeof(float);      // of jobs that share tiles: half of JOBS of 128 x 128, or JOBS of 64 x 64
int filled(int n) { return (n + 63) / 64 * 64; }
size_t bytes_of(const rlt_muon_tensor& t) {
    const size_t M = filled(t.rows < t.cols ? t.rows : t.cols), N = filled(t.rows < t.cols ? t.cols : t.rows);
    return PARTS * sizeof(double) + (6 * M * N + 4 * M * M) * sizeof(f16);
}
template <int W, int PHASE> size_t tiles_of(const Entry& m) {
    const size_t down = (m.M + W - 1) / W, across = (m.N + W - 1) / W;
    return SYMMETRIC<PHASE> ? down * (down + 1) / 2 : down * across;
}
template <int W, int PHASE> size_t tiles_of(const Entries& all) {
    size_t n = 0;
    for (int i = 0; i < all.n; i++) n += tiles_of<W, PHASE>(all.e[i]);
    return n;
}
int depth_of(const Entry& m, int phase) { return 64 * (phase == GRAM ? m.N : m.M); }
// Jobs of a launch whose tiles are shared out in lengths of `length` k. Lengths are 512 at the least, where a launch more is worth it, and leave no more than JOBS jobs (GRAM of 88 tiles of 128 x 128, up to 2,048 k: 49 us as they are, 35 shared)
template <int W, int PHASE> size_t jobs_of(const Entries& all, int length) {
    size_t n = 0;
    for (int i = 0; i < all.n; i++) n += (tiles_of<W, PHASE>(all.e[i]) * ((depth_of(all.e[i], PHASE) + length - 1) / length) + 7) / 8 * 8;
    return n;
}
int deepest_of(const Entries& all, int phase) {
    int deepest = 0;
    for (int i = 0; i < all.n; i++) deepest = std::max(deepest, depth_of(all.e[i], phase));
    return deepest;
}
constexpr int WHOLE = 1 << 30;
template <int W, int PHASE> int length_of(const Entries& all) {
    if (W > 2 || !SYMMETRIC<PHASE>) return WHOLE;
    const int deepest = deepest_of(all, PHASE);
    for (int length = 512; length < deepest; length *= 2)
        if (jobs_of<W, PHASE>(all, length) <= (W == 1 ? JOBS : JOBS / 2)) return length;
    return WHOLE;
}
// Microseconds that a launch takes, round by round of 256 tiles: for 512 k of a tile with few others, with one on every compute unit, and for its sums' way out. Against all four sizes measured, from one matrix of 256 x 256 to two of 4,096 columns, the size
// that costs least is the fastest one or within 4 us of it (profiles/muon_tiles.txt).
template <int W, int PHASE> double cost_of(const Entries& all) {
    constexpr double few[5] = {0, 5.5, 12, 15, 26}, full[5] = {0, 6.5, 14, 27, 46}, out[5] = {0, 3, 6, 18, 23};
    const int length = length_of<W, PHASE>(all);
    double cost = length == WHOLE ? 0.0 : 6.0;
    size_t jobs = 0, in_round = 0;
    int deepest = 0;
    auto round = [&] { cost += deepest / 512.0 * (few[W] + (full[W] - few[W]) * in_round / 256.0) + out[W]; in_round = 0; deepest = 0; };
    for (int i = 0; i < all.n; i++) {
        const int depth = depth_of(all.e[i], PHASE);
        for (jobs = tiles_of<W, PHASE>(all.e[i]) * ((depth + length - 1) / length); jobs; ) {
            const size_t taken = std::min(jobs, 256 - in_round);
            jobs -= taken; in_round += taken; deepest = std::max(deepest, std::min(depth, length));
            if (in_round == 256) round();
        }
    }
    if (in_round) round();
    return cost;
}
template <int W, int PHASE> int launch_width(rlt_rocm_device* device, typename ArgumentsOf<PHASE>::type all) {
    size_t blocks = 0;
    Entries& entries = all.entries;
    entries.length = length_of<W, PHASE>(entries);
    for (int i = 0; i < entries.n; i++) {
        const size_t parts = SYMMETRIC<PHASE> ? (depth_of(entries.e[i], PHASE) + entries.length - 1) / entries.length : 1;
        entries.e[i].first = (int)blocks;
        blocks += (tiles_of<W, PHASE>(entries.e[i]) * parts + 7) / 8 * 8;
    }
    if constexpr (W == 1) hipLaunchKernelGGL((product_small_kernel<PHASE>), dim3((unsigned)blocks), dim3(256), 0, device->stream, all);
    else {
        const auto kernel = product_kernel<W, PHASE>;
        const int bytes = 2 * 4 * 64 * W * 32 * (int)sizeof(f16);
        RLT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), bytes, device->stream, all);
    }
    if constexpr (W <= 2 && SYMMETRIC<PHASE>) {
        if (entries.length != WHOLE) {
            const int rc = rlt_launch_status(device);
            if (rc) return rc;
            hipLaunchKernelGGL((join_kernel<W, PHASE>), dim3((unsigned)blocks * W * W), dim3(256), 0, device->stream, all);
        }
    }
    return rlt_launch_status(device);
}
template <int PHASE> int launch(rlt_rocm_device* device, const typename ArgumentsOf<PHASE>::type& all) {
    const Entries& e = all.entries;
    const double cost[4] = {cost_of<1, PHASE>(e), cost_of<2, PHASE>(e), cost_of<3, PHASE>(e), cost_of<4, PHASE>(e)};
    const int best = (int)(std::min_element(cost, cost + 4) - cost);
    return best == 0 ? launch_width<1, PHASE>(device, all) : best == 1 ? launch_width<2, PHASE>(device, all) : best == 2 ? launch_width<3, PHASE>(device, all) : launch_width<4, PHASE>(device, all);
}
int run(rlt_rocm_device* device, Last& all, int iterations, bool local) {
    size_t tiles = 0;
    Entries& e = all.entries;
    all.iterations = iterations;
    if (local) {
        int columns = 1;
        for (int i = 0; i < e.n; i++) columns = std::max(columns, (int)e.e[i].N);
        RLT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(local_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, local_bytes(LOCAL_COLUMNS)));
        hipLaunchKernelGGL(local_kernel, dim3(e.n), dim3(1024), local_bytes(columns), device->stream, all);
        return rlt_launch_status(device);
    }
    hipLaunchKernelGGL(momentum_kernel, dim3(e.n * PARTS), dim3(256), 0, device->stream, all);
    int rc = rlt_launch_status(device);
    if (rc) return rc;
    for (int i = 0; i < e.n; i++) { e.e[i].first = (int)tiles; tiles += (size_t)e.e[i].M * e.e[i].N; }
    hipLaunchKernelGGL(normalise_kernel, dim3((unsigned)tiles), dim3(256), 0, device->stream, all);
    if ((rc = rlt_launch_status(device))) return rc;
    e.from = 0;
    for (int k = 0; k < iterations; k++, e.from ^= 1) {
        const Phases phases = {e};
        if ((rc = launch<GRAM>(device, phases)) || (rc = launch<SQUARE>(device, phases))) return rc;
        if ((rc = k + 1 < iterations ? launch<UPDATE>(device, phases) : launch<LAST>(device, all))) return rc;
    }
    return 0;
}

}  // namespace

extern "C" {

size_t rlt_rocm_muon_workspace_bytes(const rlt_muon_tensor* tensors, int n) {
    if (!described(tensors, n) || !supported(tensors, n)) return 0;
    size_t bytes = 0;
    for (int i = 0; i < n; i++) bytes += bytes_of(tensors[i]);
    return bytes + SHARED_BYTES;
}

int rlt_rocm_muon_step(rlt_rocm_device* device, const rlt_muon_tensor* tensors, int n, const rlt_muon_parameters* parameters, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(tensors, n) && parameters && parameters->iterations > 0 && parameters->iterations <= MAX_ITERATIONS && parameters->epsilon >= 0.0f);
    for (int i = 0; i < n; i++) {
        const rlt_muon_tensor& t = tensors[i];
        RLT_REQUIRE(t.parameters && t.gradient && t.momentum && t.next_parameters && t.next_momentum && t.next_momentum != t.gradient && t.next_parameters != t.gradient && t.next_parameters != t.next_momentum &&
                    t.next_parameters != t.momentum && t.next_momentum != t.parameters);
        for (int j = 0; j < n; j++) {      // a matrix twice, or one that another reads
            const rlt_muon_tensor& o = tensors[j];
            RLT_REQUIRE(j == i || (t.next_parameters != o.next_parameters && t.next_momentum != o.next_momentum && t.next_parameters != o.parameters && t.next_parameters != o.gradient && t.next_parameters != o.momentum &&
                                   t.next_parameters != o.next_momentum && t.next_momentum != o.parameters && t.next_momentum != o.gradient && t.next_momentum != o.momentum));
        }
    }
    if (!supported(tensors, n)) return RLT_E_UNSUPPORTED;
    RLT_REQUIRE(workspace && workspace_bytes >= rlt_rocm_muon_workspace_bytes(tensors, n) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
    char* at = (char*)workspace;
    // the longest products of a launch first: behind each matrix the largest of those that are no larger, in the caller's order where they are alike
    auto before = [&](int i, int j) {
        const int64_t a = (int64_t)tensors[i].rows * tensors[i].cols, b = (int64_t)tensors[j].rows * tensors[j].cols;
        return a != b ? a > b : i < j;
    };
    auto behind = [&](int last) {
        int next = -1;
        for (int i = 0; i < n; i++) if ((last < 0 || before(last, i)) && (next < 0 || before(i, next))) next = i;
        return next;
    };
    Last all{};
    all.entries.parts = (float*)at;
    at += SHARED_BYTES;
    all.tensors.momentum = parameters->momentum; all.tensors.epsilon = parameters->epsilon; all.tensors.keep = 1.0f - parameters->alpha * parameters->weight_decay; all.tensors.nesterov = parameters->nesterov;
    bool local = true;
    for (int i = 0; i < n; i++) local = local && std::min(tensors[i].rows, tensors[i].cols) <= 64 && std::max(tensors[i].rows, tensors[i].cols) <= 64 * LOCAL_COLUMNS;
    int last = -1;
    for (int i = 0; i < n; i++) {
        last = behind(last);
        const rlt_muon_tensor& t = tensors[last];
        const int low = t.rows < t.cols ? t.rows : t.cols, high = t.rows < t.cols ? t.cols : t.rows;
        all.entries.e[all.entries.n] = {at, (uint16_t)(filled(low) / 64), (uint16_t)(filled(high) / 64), 0};
        all.tensors.t[all.entries.n++] = {t.parameters, t.gradient, t.momentum, t.next_parameters, t.next_momentum, t.rows, t.cols, parameters->alpha * sqrtf(t.rows > t.cols ? (float)t.rows / t.cols : 1.0f)};
        at += bytes_of(t);
        if (all.entries.n == GROUP || i == n - 1) {
            const int rc = run(device, all, parameters->iterations, local);
            if (rc) return rc;
            all.entries.n = 0;
        }
    }
    return 0;
}

}  // extern "C"
