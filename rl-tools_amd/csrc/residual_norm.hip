// The norm after a block, its gate and residual scale, and the norm before the next block: one pass over the rows forward, one backward.
#include "typed.h"
#include <type_traits>

namespace {

constexpr int MAX_DIM = 8192, HELD_DIM = 4096, MAX_ROWS = 1 << 30;      // a row's index and a step over the grid's rows fit 32 bits
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

// THREADS share a row: a part of a wavefront, a wavefront, several or all of a workgroup of WIDTH threads.
template <int THREADS> constexpr int FORWARD_WIDTH = THREADS <= 64 ? 256 : THREADS;
template <int THREADS> constexpr int BACKWARD_WIDTH = THREADS < 256 ? 256 : THREADS;      // half the column sums to join that workgroups of 128 have, at as many wavefronts (4,001 x 1,000 fp32: 36 us, 40 with 128)

// a thread's place in its row, and its row's in the workgroup (the same for all of a wavefront where a row has one or more: addresses of rows stay scalar)
template <int THREADS> __device__ __forceinline__ int thread_of() { return (int)(threadIdx.x % THREADS); }
template <int THREADS, int WIDTH> __device__ __forceinline__ int row_of() {
    return WIDTH == THREADS ? 0 : THREADS >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : (int)(threadIdx.x / THREADS);
}

// Sums over the threads that share a row, every one of which receives them. Consecutive calls take turns with two halves of `lds`: a wavefront that writes one has passed the barrier
// behind which everybody had read it.
template <int THREADS, int WIDTH, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* lds, int& turn) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        asm volatile("" : "+v"(v[i]));      // no contraction into the first exchange: both sides of an exchange round alike (rlt_wave_sum)
#pragma unroll
        for (int off = (THREADS < 64 ? THREADS : 64) / 2; off > 0; off >>= 1) v[i] += __shfl_xor(v[i], off, 64);
    }
    if constexpr (THREADS > 64) {
        constexpr int WAVES = THREADS / 64;
        float* half = lds + turn * (WIDTH / 64) * 4;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) half[(threadIdx.x >> 6) * 4 + i] = v[i];
        }
        if (WIDTH > THREADS) half += row_of<THREADS, WIDTH>() * WAVES * 4;
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

// Thread t of a row's THREADS has vectors t, t + THREADS, ... of V elements (16 bytes), K of them. WHOLE: rows start on 16-byte boundaries and hold whole vectors. Otherwise the same loads and stores start at any element, which the
// memory instructions allow; a row's last vector is loaded where it ends with the row, and its elements move down when they are needed, so that no load waits for a branch. (8,192 rows of 1,001 bfloat16 values: 22 to 27 us
// forward, 43 to 45 us backward; 52 and 71 with an element to a load.)
template <typename T, int V, bool WHOLE> struct Row { typedef T Vector __attribute__((ext_vector_type(V))); };
template <typename T, int V> struct Row<T, V, false> { typedef T Vector __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T, int V, int K> struct Raw { typedef T Vector __attribute__((ext_vector_type(V))); Vector v[K]; };
template <int V, int K, int THREADS, bool WHOLE, typename T> __device__ __forceinline__ void load_raw(const T* src, int dim, Raw<T, V, K>& to) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + thread_of<THREADS>()) * V;
        to.v[k] = typename Raw<T, V, K>::Vector{};
        if constexpr (WHOLE) {
            if (c < dim) to.v[k] = *reinterpret_cast<const typename Row<T, V, WHOLE>::Vector*>(src + c);
        } else if (dim >= V) {
            if (c < dim) to.v[k] = *reinterpret_cast<const typename Row<T, V, WHOLE>::Vector*>(src + (c + V <= dim ? c : dim - V));
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) to.v[k][i] = c + i < dim ? src[c + i] : (T)0.0f;
        }
    }
}
template <int V, int K, int THREADS, bool WHOLE, typename T> __device__ __forceinline__ void unpack(const Raw<T, V, K>& from, int dim, float (&v)[V * K]) {
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int i = 0; i < V; i++) v[k * V + i] = (float)from.v[k][i];
        const int c = (k * THREADS + thread_of<THREADS>()) * V, beyond = c + V - dim;
        if (!WHOLE && beyond > 0 && c < dim && dim >= V) {
#pragma unroll
            for (int n = 1; n < V; n *= 2) {
#pragma unroll
                for (int i = 0; i < V; i++) v[k * V + i] = beyond & n ? (i + n < V ? v[k * V + (i + n) % V] : 0.0f) : v[k * V + i];
            }
        }
    }
}
template <int V, int K, int THREADS, bool WHOLE, typename T> __device__ __forceinline__ void load_row(const T* src, int dim, float (&v)[V * K]) {
    if constexpr (WHOLE && sizeof(T) == sizeof(float)) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * THREADS + thread_of<THREADS>()) * V;
            if (c < dim) rlt_load<V>(src + c, v + k * V);
            else {
#pragma unroll
                for (int i = 0; i < V; i++) v[k * V + i] = 0.0f;
            }
        }
    } else {
        Raw<T, V, K> raw;
        load_raw<V, K, THREADS, WHOLE>(src, dim, raw);
        unpack<V, K, THREADS, WHOLE>(raw, dim, v);
    }
}
// rounds to nearest, ties to even
template <int V, int K, int THREADS, bool WHOLE, typename T> __device__ __forceinline__ void store_row(T* dst, int dim, const float (&v)[V * K]) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + thread_of<THREADS>()) * V;
        if (WHOLE ? c < dim : c + V <= dim) {
            typename Raw<T, V, K>::Vector x;
#pragma unroll
            for (int i = 0; i < V; i++) x[i] = (T)v[k * V + i];
            *reinterpret_cast<typename Row<T, V, WHOLE>::Vector*>(dst + c) = x;
        } else if (!WHOLE && c < dim) {
#pragma unroll
            for (int i = 0; i < V - 1; i++) if (c + i < dim) dst[c + i] = (T)v[k * V + i];
        }
    }
}
// parameters of this thread's columns, zero beyond dim; `otherwise` where there are none
template <int V, int K, int THREADS, bool WHOLE> __device__ __forceinline__ void load_parameters(const float* src, float otherwise, int dim, float (&v)[V * K]) {
#pragma unroll
    for (int i = 0; i < V * K; i++) v[i] = otherwise;
    if (!src) return;
    int t = thread_of<THREADS>();
    asm volatile("" : "+v"(t));      // addresses are formed here, not ahead of a loop over rows, whose registers they would take
#pragma unroll
    for (int n = 0; n < V * K; n += 4) {
        const int c = (n / V * THREADS + t) * V + n % V, beyond = c + 4 - dim;
        rlt_f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (WHOLE || dim >= 4) {
            if (c < dim) x = *reinterpret_cast<const Row<float, 4, false>::Vector*>(src + (WHOLE || beyond <= 0 ? c : dim - 4));
            if (!WHOLE && beyond > 0) {
                if (beyond & 1) x = rlt_f32x4{x[1], x[2], x[3], 0.0f};
                if (beyond & 2) x = rlt_f32x4{x[2], x[3], 0.0f, 0.0f};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) if (c + i < dim) x[i] = src[c + i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) v[n + i] = x[i];
    }
}
// subtracts a row's mean; columns beyond dim stay zero
template <int V, int K, int THREADS, bool WHOLE> __device__ __forceinline__ void subtract(float (&v)[V * K], float mean, int dim) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + thread_of<THREADS>()) * V;
        if (c < dim) {
#pragma unroll
            for (int i = 0; i < V; i++) if (WHOLE || c + i < dim) v[k * V + i] -= mean;
        }
    }
}
template <int V, int K, int THREADS, bool WHOLE> __device__ __forceinline__ void zero_beyond(float (&v)[V * K], int dim) {
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int c = (k * THREADS + thread_of<THREADS>()) * V;
        if (WHOLE ? c >= dim : c + V > dim) {
#pragma unroll
            for (int i = 0; i < V; i++) if (WHOLE || c + i >= dim) v[k * V + i] = 0.0f;
        }
    }
}

// a row's values less their mean (RLT_NORM_LAYER), and 1 / deviation
template <int V, int K, int THREADS, bool WHOLE> __device__ __forceinline__ float normalise(float (&v)[V * K], int kind, float epsilon, int dim, float* lds, int& turn) {
    constexpr int N = V * K;
    if (kind == RLT_NORM_NONE) return 1.0f;
    const float inverse_dim = 1.0f / dim;
    float s[1];
    if (kind == RLT_NORM_LAYER) {
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += v[i];
        row_sums<THREADS, FORWARD_WIDTH<THREADS>>(s, lds, turn);
        subtract<V, K, THREADS, WHOLE>(v, s[0] * inverse_dim, dim);
    }
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) s[0] = fmaf(v[i], v[i], s[0]);
    row_sums<THREADS, FORWARD_WIDTH<THREADS>>(s, lds, turn);
    return 1.0f / sqrtf(s[0] * inverse_dim + epsilon);
}

// The gates' activations, in place, and their derivatives. One loop over a thread's gates for each function, not a choice for each gate. Functions as rlt_act has them; sigmoid and GELU, as x / (1 + e^(-2 z)),
// keep their relative accuracy where 1 + tanh(z) cancels.
template <typename T, int N, bool SLOPES> __device__ __forceinline__ void gates_of(float (&g)[N], float (&slope)[N], int kind) {
    if (kind == RLT_ACT_SIGMOID) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            // e^-|g| as a power of two, whose rounded exponent alone leaves it off by about |g| units of 2^-24. fp32 tensors take what is left of the exponent along; bfloat16 ones do without: at a gate of -64 it is a 2^10th of the
            // output's own rounding, and costs 3 % (16,384 x 4,096 backward: 237 us, 247 with it).
            const float t = -fabsf(g[i]), at = t * 1.44269504088896341f, p = __builtin_amdgcn_exp2f(at);
            float e = p;
            if (sizeof(T) == sizeof(float)) {
                const float rest = fmaf(t, 1.44269504088896341f, -at) + t * 1.925963033500721e-8f;
                e = at > -126.0f ? fmaf(p, rest * 0.6931471805599453f, p) : p;
            }
            const float large = __fdividef(1.0f, 1.0f + e), small = e * large;      // e in [0, 1]
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
            const float x = g[i] > 30.0f ? 30.0f : g[i] < -30.0f ? -30.0f : g[i];      // beyond, p and q are 0 and 1, and powers of x need not fit fp32
            const float z = 2.0f * a * fmaf(b * x * x, x, x), e = expf(-fabsf(z)), large = 1.0f / (1.0f + e), small = e * large, p = z >= 0.0f ? large : small, q = z >= 0.0f ? small : large;
            if (SLOPES) slope[i] = p * fmaf(2.0f * x * q, a * fmaf(3.0f * b * x, x, 1.0f), 1.0f);
            g[i] *= p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) { if (SLOPES) slope[i] = rlt_dact(g[i], kind); g[i] = rlt_act(g[i], kind); }
    }
}

// Memory bounds this pass: three rows in, two out, all of a row's elements in registers from its loads to its stores (16,384 x 4,096 bfloat16: 152 us, 4.4 TB/s; 65,536 x 256 fp32: 66 us, 5.0 TB/s; a launch at 256 x 256: 4.3 us).
// bfloat16 rows are converted behind the last load: a conversion in a load's branch waits for it (163 us); fp32 rows need none and are faster without the copy (66 us, 74 with it).
template <typename T, int V, int K, int THREADS, bool WHOLE> __global__ __launch_bounds__(FORWARD_WIDTH<THREADS>) void norm_forward_kernel(NormForward a) {
    constexpr int N = V * K, ROWS = FORWARD_WIDTH<THREADS> / THREADS;
    __shared__ float lds[THREADS > 64 ? 2 * (THREADS / 64) * 4 : 1];
    int turn = 0;
    const int dim = a.p.dim;
    float bw[N], bb[N], ow[N], ob[N], scale[N];
    load_parameters<V, K, THREADS, WHOLE>(a.p.branch_weights, 1.0f, dim, bw); load_parameters<V, K, THREADS, WHOLE>(a.p.branch_biases, 0.0f, dim, bb);
    load_parameters<V, K, THREADS, WHOLE>(a.p.output_weights, 1.0f, dim, ow); load_parameters<V, K, THREADS, WHOLE>(a.p.output_biases, 0.0f, dim, ob);
    load_parameters<V, K, THREADS, WHOLE>(a.p.residual_scale, 1.0f, dim, scale);
    for (int row = blockIdx.x * ROWS + row_of<THREADS, FORWARD_WIDTH<THREADS>>(); row < a.rows; row += gridDim.x * ROWS) {
        float y[N], u[N], g[N];
        if (a.branch) load_row<V, K, THREADS, WHOLE>((const T*)a.branch + (size_t)row * a.ldb, dim, u);
        load_row<V, K, THREADS, WHOLE>((const T*)a.x + (size_t)row * a.ldx, dim, y);
        if (a.branch && a.gate) load_row<V, K, THREADS, WHOLE>((const T*)a.gate + (size_t)row * a.ldg, dim, g);
        if (a.branch) {
            const float inverse = normalise<V, K, THREADS, WHOLE>(u, a.p.branch_norm, a.p.epsilon, dim, lds, turn);
            float slope[N];
            if (a.gate) gates_of<T, N, false>(g, slope, a.p.gate_activation);
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = fmaf(a.gate ? scale[i] * g[i] : scale[i], fmaf(u[i] * inverse, bw[i], bb[i]), y[i]);
            // columns beyond dim: u, g and y are zero, a bias is too
        }
        if (a.y) store_row<V, K, THREADS, WHOLE>((T*)a.y + (size_t)row * a.ldy, dim, y);
        if (a.h) {
            const float inverse = normalise<V, K, THREADS, WHOLE>(y, a.p.output_norm, a.p.epsilon, dim, lds, turn);
#pragma unroll
            for (int i = 0; i < N; i++) y[i] = fmaf(y[i] * inverse, ow[i], ob[i]);
            store_row<V, K, THREADS, WHOLE>((T*)a.h + (size_t)row * a.ldh, dim, y);
        }
    }
}

// Memory bounds this pass: five rows in, three out, 4.6 TB/s at 16,384 rows of 4,096 bfloat16 values (236 to 268 us), 4.8 at 16,384 of 2,048 fp32 values; few rows are bound by the trips to memory of the two or three that a workgroup
// has (4,001 x 1,000 fp32: 36 us). The next row's values are asked for before this row's sums, of which a row has two rounds (three with means): what the statistics and the output norm's gradient need
// is added up together.
template <typename T, int V, int K, int THREADS, bool BIASES, bool WHOLE> __global__ __launch_bounds__(BACKWARD_WIDTH<THREADS>) void norm_backward_kernel(NormBackward a) {
    constexpr int N = V * K, WIDTH = BACKWARD_WIDTH<THREADS>, ROWS = WIDTH / THREADS;
    // Parameters and column sums stay in registers from row to row. Rows wider than 4,096 leave none for them: parameters are read again, from L2, and the sums are kept in LDS, each by its own thread (4,096 rows of 8,192 bfloat16
    // values: 183 us; 536 with 1,024 threads of eight columns, whose registers spill. 16,384 rows of 4,096: 266 us with registers, 332 so). fp32 rows this wide spill all the same with biases, or where no vectors divide them (56 to 116 bytes of
    // scratch memory a lane): 4,096 rows of 8,192 fp32 values 242 us, 334 with biases, of 8,191 with biases 536; bfloat16 184, 215 and 317.
    constexpr bool HELD = N * THREADS <= HELD_DIM, AHEAD = HELD || (WHOLE && V == 8);
    __shared__ float lds[ROWS == 1 ? 2 * (THREADS / 64) * 4 : WIDTH * N];
    extern __shared__ __attribute__((aligned(16))) float column_sums[];
    int turn = 0;
    const int dim = a.p.dim, stride = gridDim.x * ROWS;
    const float inverse_dim = 1.0f / dim;
    const bool output_layer = a.d_h && a.p.output_norm == RLT_NORM_LAYER, branch_layer = a.branch && a.p.branch_norm == RLT_NORM_LAYER;
    float bw[N], bb[N], ow[N], scale[N];
    auto output_parameters = [&] { load_parameters<V, K, THREADS, WHOLE>(a.p.output_weights, 1.0f, dim, ow); };
    auto branch_parameters = [&] {
        load_parameters<V, K, THREADS, WHOLE>(a.p.branch_weights, 1.0f, dim, bw); load_parameters<V, K, THREADS, WHOLE>(BIASES ? a.p.branch_biases : nullptr, 0.0f, dim, bb);
        load_parameters<V, K, THREADS, WHOLE>(a.p.residual_scale, 1.0f, dim, scale);
    };
    if (HELD) { output_parameters(); branch_parameters(); }
    // Sum j of this thread's columns: in a register, or in LDS, 16 bytes of every thread side by side. 160 KB hold four sums of the widest rows and not the fifth.
    constexpr int SLOT[SUMS] = {0, 3, 1, 4, 2}, SLOTS = BIASES ? 4 : 3;
    float sums[HELD ? SUMS : 1][N];
    auto add = [&](auto which, const float (&v)[N]) {
        constexpr int j = decltype(which)::value;
        if constexpr (HELD || SLOT[j] >= SLOTS) {
#pragma unroll
            for (int i = 0; i < N; i++) sums[HELD ? j : 0][i] += v[i];
        } else {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                __builtin_amdgcn_sched_barrier(0);
                rlt_f32x4* const at = reinterpret_cast<rlt_f32x4*>(column_sums) + (SLOT[j] * (N / 4) + k / 4) * THREADS + threadIdx.x;
                rlt_f32x4 x = *at;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] += v[k + i];
                *at = x;
            }
        }
    };
#pragma unroll
    for (int j = 0; j < (HELD ? SUMS : 1); j++)
#pragma unroll
        for (int i = 0; i < N; i++) sums[j][i] = 0.0f;
    if constexpr (!HELD) {
#pragma unroll
        for (int j = 0; j < SLOTS * (N / 4); j++) reinterpret_cast<rlt_f32x4*>(column_sums)[j * THREADS + threadIdx.x] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#define NORM_SUM(j) std::integral_constant<int, j>{}
    Raw<T, V, K> next_e{}, next_y{}, next_d{}, next_u{}, next_g{};
    auto ask = [&](int row) {
        const int dim = ROWS == 1 || row < a.rows ? a.p.dim : 0;      // rows that a workgroup has no more: zeros, which add nothing
        if (a.d_h) {
            load_raw<V, K, THREADS, WHOLE>((const T*)a.d_h + (size_t)row * a.lddh, dim, next_e);
            load_raw<V, K, THREADS, WHOLE>((const T*)a.y + (size_t)row * a.ldy, dim, next_y);
        }
        if (a.d_y) load_raw<V, K, THREADS, WHOLE>((const T*)a.d_y + (size_t)row * a.lddy, dim, next_d);
        if (a.branch) {
            load_raw<V, K, THREADS, WHOLE>((const T*)a.branch + (size_t)row * a.ldb, dim, next_u);
            if (a.gate) load_raw<V, K, THREADS, WHOLE>((const T*)a.gate + (size_t)row * a.ldg, dim, next_g);
        }
    };
    if (AHEAD) ask(blockIdx.x * ROWS + row_of<THREADS, WIDTH>());
    for (int first = blockIdx.x * ROWS; first < a.rows; first += stride) {      // all rows of a workgroup at once: they share its barriers
        const int row = first + row_of<THREADS, WIDTH>();
        const bool here = ROWS == 1 || row < a.rows;
        float d[N], e[N], y[N], u[N], g[N];      // d: the gradient that reaches the residual stream
        if (!AHEAD) ask(row);
        unpack<V, K, THREADS, WHOLE>(next_e, dim, e); unpack<V, K, THREADS, WHOLE>(next_y, dim, y); unpack<V, K, THREADS, WHOLE>(next_d, dim, d); unpack<V, K, THREADS, WHOLE>(next_u, dim, u); unpack<V, K, THREADS, WHOLE>(next_g, dim, g);
        if (AHEAD && first + stride < a.rows) ask(row + stride);
        if (output_layer || branch_layer) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < N; i++) { s[0] += y[i]; s[1] += u[i]; }
            row_sums<THREADS, WIDTH>(s, lds, turn);
            if (output_layer) subtract<V, K, THREADS, WHOLE>(y, s[0] * inverse_dim, dim);
            if (branch_layer) subtract<V, K, THREADS, WHOLE>(u, s[1] * inverse_dim, dim);
        }
        if (!HELD) { output_parameters(); __builtin_amdgcn_sched_barrier(0); }
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // of y^2, of the output norm's gradient times y, of that gradient, of branch^2
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float w = e[i] * ow[i];
            s[0] = fmaf(y[i], y[i], s[0]); s[1] = fmaf(w, y[i], s[1]); s[2] += w; s[3] = fmaf(u[i], u[i], s[3]);
        }
        row_sums<THREADS, WIDTH>(s, lds, turn);
        if (a.d_h) {
            const bool none = a.p.output_norm == RLT_NORM_NONE;
            const float inverse = none ? 1.0f : 1.0f / sqrtf(s[0] * inverse_dim + a.p.epsilon), along = none ? 0.0f : inverse * s[1] * inverse_dim, mean = output_layer ? s[2] * inverse_dim : 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float n = y[i] * inverse;
                y[i] = e[i] * n;
                d[i] = fmaf(inverse, fmaf(e[i], ow[i], -n * along) - mean, d[i]);
            }
            if (!HELD) __builtin_amdgcn_sched_barrier(0);
            add(NORM_SUM(OUTPUT_W), y);
            if constexpr (BIASES) add(NORM_SUM(OUTPUT_B), e);
            if (mean != 0.0f) zero_beyond<V, K, THREADS, WHOLE>(d, dim);      // the sums that follow take no column beyond dim
        }
        if (a.d_x && here) store_row<V, K, THREADS, WHOLE>((T*)a.d_x + (size_t)row * a.lddx, dim, d);
        if (a.branch) {
            const bool none = a.p.branch_norm == RLT_NORM_NONE;
            const float inverse = none ? 1.0f : 1.0f / sqrtf(s[3] * inverse_dim + a.p.epsilon);
            if (!HELD) { __builtin_amdgcn_sched_barrier(0); branch_parameters(); }
            float slope[N], t[2] = {0.0f, 0.0f};
            if (a.gate) gates_of<T, N, true>(g, slope, a.p.gate_activation);
#pragma unroll
            for (int i = 0; i < N; i++) {
                u[i] *= inverse;
                const float n = BIASES ? fmaf(u[i], bw[i], bb[i]) : u[i] * bw[i], m = a.gate ? g[i] : 1.0f, ds = d[i] * scale[i], dn = ds * m;
                if (a.gate) slope[i] *= ds * n;
                y[i] = d[i] * m * n; d[i] = dn * u[i]; g[i] = dn;      // summands of the columns
                e[i] = dn * bw[i];
                t[0] = fmaf(e[i], u[i], t[0]); t[1] += e[i];
            }
            add(NORM_SUM(SCALE), y); add(NORM_SUM(BRANCH_W), d);
            if constexpr (BIASES) add(NORM_SUM(BRANCH_B), g);
            if (a.d_gate && here) store_row<V, K, THREADS, WHOLE>((T*)a.d_gate + (size_t)row * a.lddg, dim, slope);
            if (a.d_branch) {
                if (!none) {
                    row_sums<THREADS, WIDTH>(t, lds, turn);
                    const float along = t[0] * inverse_dim, mean = branch_layer ? t[1] * inverse_dim : 0.0f;
#pragma unroll
                    for (int i = 0; i < N; i++) e[i] = inverse * (e[i] - u[i] * along - mean);
                }
                if (here) store_row<V, K, THREADS, WHOLE>((T*)a.d_branch + (size_t)row * a.lddb, dim, e);
            }
        }
    }
    float* const wanted[SUMS] = {a.p.d_branch_weights, a.p.d_branch_biases, a.p.d_output_weights, a.p.d_output_biases, a.p.d_residual_scale};
    float* out = a.partial + (size_t)blockIdx.x * SUMS * dim;
#pragma unroll
    for (int j = 0; j < SUMS; j++) {
        if (!wanted[j] || (!BIASES && (j == BRANCH_B || j == OUTPUT_B))) continue;
        if constexpr (ROWS > 1) {      // the rows' threads side by side, then column by column in their order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) lds[(threadIdx.x / THREADS) * THREADS * N + (k * THREADS + threadIdx.x % THREADS) * V + i] = sums[HELD ? j : 0][k * V + i];
            __syncthreads();
            for (int c = threadIdx.x; c < dim; c += WIDTH) {
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
                    const int c = (k * THREADS + (int)threadIdx.x) * V + i, n = k * V + i;
                    if (c < dim) out[(size_t)j * dim + c] = HELD || SLOT[j] >= SLOTS ? sums[HELD ? j : 0][n] : column_sums[((SLOT[j] * (N / 4) + n / 4) * THREADS + threadIdx.x) * 4 + n % 4];
                }
        }
    }
}
#undef NORM_SUM

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

// threads that share a row in the backward pass, eight columns each, or sixteen
int backward_threads(int dim) { return dim <= 128 ? 16 : dim <= 512 ? 64 : dim <= 1024 ? 128 : dim <= 2048 ? 256 : 512; }
int backward_blocks(const rlt_residual_norm* p, int rows) {
    const int threads = backward_threads(p->dim), at_once = threads < 256 ? 256 / threads : 1, blocks = (rows + at_once - 1) / at_once;
    return blocks < 512 ? blocks : 512;
}

template <typename T, int V, bool WHOLE> void launch_forward(rlt_rocm_device* device, const NormForward& a) {
    const int dim = a.p.dim;
    auto go = [&](auto kernel, int threads) {
        const int workgroup = threads <= 64 ? 256 : threads, at_once = workgroup / threads, blocks = (a.rows + at_once - 1) / at_once;
        hipLaunchKernelGGL(kernel, dim3(blocks < 2048 ? blocks : 2048), dim3(workgroup), 0, device->stream, a);
    };
    if (dim <= 128) go(norm_forward_kernel<T, V, 8 / V, 16, WHOLE>, 16);
    else if (dim <= 512) go(norm_forward_kernel<T, V, 8 / V, 64, WHOLE>, 64);
    else if (dim <= 1024) go(norm_forward_kernel<T, V, 8 / V, 128, WHOLE>, 128);
    else if (dim <= 2048) go(norm_forward_kernel<T, V, 8 / V, 256, WHOLE>, 256);
    else if (dim <= 4096) go(norm_forward_kernel<T, V, 8 / V, 512, WHOLE>, 512);
    else go(norm_forward_kernel<T, V, 8 / V, 1024, WHOLE>, 1024);
}
template <typename T, int V, bool BIASES, bool WHOLE> int launch_backward(rlt_rocm_device* device, const NormBackward& a) {
    const int threads = backward_threads(a.p.dim);
    const size_t bytes = a.p.dim > HELD_DIM ? (size_t)(BIASES ? 4 : 3) * MAX_DIM * sizeof(float) : 0;
    hipError_t e = hipSuccess;
    auto go = [&](auto kernel) {
        if (bytes) e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == hipSuccess) hipLaunchKernelGGL(kernel, dim3(backward_blocks(&a.p, a.rows)), dim3(threads < 256 ? 256 : threads), bytes, device->stream, a);
    };
    if (threads == 16) go(norm_backward_kernel<T, V, 8 / V, 16, BIASES, WHOLE>);
    else if (threads == 64) go(norm_backward_kernel<T, V, 8 / V, 64, BIASES, WHOLE>);
    else if (threads == 128) go(norm_backward_kernel<T, V, 8 / V, 128, BIASES, WHOLE>);
    else if (threads == 256) go(norm_backward_kernel<T, V, 8 / V, 256, BIASES, WHOLE>);
    else if (a.p.dim <= HELD_DIM) go(norm_backward_kernel<T, V, 8 / V, 512, BIASES, WHOLE>);
    else go(norm_backward_kernel<T, V, 16 / V, 512, BIASES, WHOLE>);
    RLT_HIP(e);
    return rlt_launch_status(device);
}
// whole vectors where every tensor's rows start on 16-byte boundaries and hold such
template <typename T> void forward(rlt_rocm_device* device, const NormForward& a) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = a.p.dim % V == 0 && rlt_vectors<T>(a.x, a.ldx) && rlt_vectors<T>(a.branch, a.branch ? a.ldb : 0) && rlt_vectors<T>(a.gate, a.gate ? a.ldg : 0) &&
                         rlt_vectors<T>(a.y, a.y ? a.ldy : 0) && rlt_vectors<T>(a.h, a.h ? a.ldh : 0);
    if (vectors) launch_forward<T, V, true>(device, a); else launch_forward<T, V, false>(device, a);
}
template <typename T> int backward(rlt_rocm_device* device, const NormBackward& a) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = a.p.dim % V == 0 && rlt_vectors<T>(a.branch, a.branch ? a.ldb : 0) && rlt_vectors<T>(a.gate, a.gate ? a.ldg : 0) && rlt_vectors<T>(a.y, a.d_h ? a.ldy : 0) &&
                         rlt_vectors<T>(a.d_y, a.d_y ? a.lddy : 0) && rlt_vectors<T>(a.d_h, a.d_h ? a.lddh : 0) && rlt_vectors<T>(a.d_x, a.d_x ? a.lddx : 0) &&
                         rlt_vectors<T>(a.d_branch, a.d_branch ? a.lddb : 0) && rlt_vectors<T>(a.d_gate, a.d_gate ? a.lddg : 0);
    const bool biases = a.p.branch_biases || a.p.d_branch_biases || a.p.d_output_biases;
    if (vectors) return biases ? launch_backward<T, V, true, true>(device, a) : launch_backward<T, V, false, true>(device, a);
    return biases ? launch_backward<T, V, true, false>(device, a) : launch_backward<T, V, false, false>(device, a);
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
    if (dim > MAX_DIM || rows > MAX_ROWS) return RLT_E_UNSUPPORTED;
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
    if (dim > MAX_DIM || rows > MAX_ROWS) return RLT_E_UNSUPPORTED;
    const bool sums = layer->d_branch_weights || layer->d_branch_biases || layer->d_output_weights || layer->d_output_biases || layer->d_residual_scale;
    RLT_REQUIRE(!sums || (workspace && workspace_bytes >= rlt_rocm_residual_norm_workspace_bytes(layer, rows)));
    const NormBackward a = {*layer, branch, gate, y, d_y, d_h, d_x, d_branch, d_gate, ldb, ldg, ldy, lddy, lddh, lddx, lddb, lddg, rows, (float*)workspace};
    const int rc = layer->type == RLT_TYPE_F32 ? backward<float>(device, a) : backward<rlt_bf16>(device, a);
    if (rc || !sums) return rc;
    hipLaunchKernelGGL(norm_sum_kernel, dim3((dim + 63) / 64, SUMS), dim3(1024), 0, device->stream, (const float*)workspace, backward_blocks(layer, rows), dim, *layer, accumulate);
    return rlt_launch_status(device);
}

}  // extern "C"
