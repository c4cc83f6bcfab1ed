// Linear attention with a decay for each head: sequences forward and backward, and single steps on a kept state.
#include "typed.h"
#include <type_traits>

namespace {

constexpr int MAX_WIDTH = 128, CHUNK = 64, STEP_NARROW = 1024, MAX_STEPS = 1 << 30;

// a tensor as the kernels see it: heads / group of it; channels side by side are read and written as vectors where `vectors` is set
struct Part { void* data; int64_t step, row, head; int group, vectors; };      // vectors: of 16 bytes (inputs), of four channels (outputs)
// One direction of the layer over segments of the steps. "key" and "value" are the two factors of what is added to the state [key x value], "query" what reads it.
struct Walk {
    Part q, k, v, out;
    Part with;                    // SLOPE: what the output's derivative by the decay's logarithm is multiplied with
    const float* log_decay;
    const float* entry;           // state that a walk starts from (NULL: zeros): of row and head, or of row, head and segment where there are several
    float* exit;                  // state that it ends with (NULL: not wanted), the same
    const float* entry_slope; float* exit_slope;
    const float* d_final;         // SLOPE: gradient with respect to the final state (NULL: zeros)
    double* partial;              // SLOPE: [rows x heads x segments]
    float2* factors;              // STATE: what a segment multiplies the state by (0: it forgets), and its steps
    const uint8_t* reset; const int32_t* lengths;
    float score_scale, read_scale, added_scale;
    int batch, heads, steps, key, value, segments, segment_steps;
    int state_key, state_value;   // strides of the state in memory
    int last_wanted;              // STATE: the last segment's state too
};

template <typename T> __device__ __forceinline__ T* at(const Part& p, int t, int b, int h) {
    return (T*)p.data + ((int64_t)t * p.step + (int64_t)b * p.row + (int64_t)(h / p.group) * p.head);
}

// Operands of the matrix instructions: eight values a lane, lane l having row (column) l % 16 and, of 32 summands, those that its quarter l / 16 selects. bfloat16: one 16x16x32 instruction; fp32: eight
// 16x16x4 instructions, the e-th of which takes value e of every lane. Which summands a quarter has is free as long as both operands agree.
typedef float rlt_f32x8 __attribute__((ext_vector_type(8)));
template <typename T> struct Operand;
template <> struct Operand<float> { typedef rlt_f32x8 Vector; typedef rlt_f32x4 Quad, Bytes16; };
template <> struct Operand<rlt_bf16> { typedef rlt_bf16x8 Vector, Bytes16; typedef rlt_bf16x4 Quad; };
__device__ __forceinline__ rlt_f32x4 multiply(rlt_f32x8 a, rlt_f32x8 b, rlt_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ rlt_f32x4 multiply(rlt_bf16x8 a, rlt_bf16x8 b, rlt_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// fp32 values (scores, states, weighted values) as operands. For bfloat16 kernels they are cut into three parts, whose sum they are exactly to fp32. (Two
// leave 2^-18 of a value out, for which ten times as many outputs as with three are the second-nearest bfloat16 number.)
template <typename T> constexpr int PARTS = sizeof(T) == 4 ? 1 : 3;
template <typename T> struct Cut {
    rlt_bf16x8 part[PARTS<T>];
    __device__ __forceinline__ explicit Cut(rlt_f32x8 x) {
#pragma unroll
        for (int p = 0; p < PARTS<T>; p++) {
            part[p] = __builtin_convertvector(x, rlt_bf16x8);
            if (p + 1 < PARTS<T>) x -= __builtin_convertvector(part[p], rlt_f32x8);
        }
    }
};
template <> struct Cut<float> {
    rlt_f32x8 part[1];
    __device__ __forceinline__ explicit Cut(rlt_f32x8 x) { part[0] = x; }
};

// whether some of 16-byte vectors' values are not finite (exponents of ones)
template <int N> __device__ __forceinline__ bool not_finite(const rlt_f32x4 (&x)[N]) {
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) zero = fmaf(x[i][e], 0.0f, zero);
    return zero != 0.0f;
}
template <int N> __device__ __forceinline__ bool not_finite(const rlt_bf16x8 (&x)[N]) {
    typedef unsigned Words __attribute__((ext_vector_type(4)));
    unsigned carried = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const Words w = __builtin_bit_cast(Words, x[i]);
#pragma unroll
        for (int e = 0; e < 4; e++) carried |= (w[e] & 0x7f807f80u) + 0x00800080u;      // two to a word
    }
    return (carried & 0x80008000u) != 0;
}

// decay^n; n = 0 gives 1 also for a decay of zero. The logarithm to the base of 2 is a sum of two numbers: one alone is off by 2^-24 of itself, its n-fold by that of n times as much, and every row and step would meet the same error.
struct Log2 {
    float high, low;
    __device__ __forceinline__ explicit Log2(float log_decay) : high(log_decay * 1.44269504088896341f), low(fmaf(log_decay, 1.44269504088896341f, -high) + log_decay * 1.925963033500721e-8f) {}
};
__device__ __forceinline__ float power(const Log2& decay, int n) {
    const float at = decay.high * (float)n, p = __builtin_amdgcn_exp2f(at), rest = fmaf(decay.high, (float)n, -at) + decay.low * (float)n;
    return n == 0 ? 1.0f : fabsf(at) < 126.0f ? fmaf(p, rest * 0.6931471805599453f, p) : p;      // powers beyond fp32 are 0 or infinity as they are
}

// Shape of a workgroup for heads of up to D channels: a wavefront owns TILES x 16 of the value columns. SPLIT workgroups share a head's columns where two states would not fit the registers of one: the scores are then
// formed in each of them (bfloat16). fp32 takes one of eight wavefronts, which LDS has room for as it has for one of four (d_q of 2,846 heads of 64 x 127, 35 steps: 291 us, 524 with two workgroups a head).
template <typename T, int D, bool SLOPE, bool STATE> struct Layout {
    static constexpr int SPLIT = SLOPE && D == 128 && sizeof(T) == 2 ? 2 : 1, COLUMNS = D / SPLIT;
    static constexpr int TILES = D == 128 && sizeof(T) == 2 && !SLOPE ? 2 : 1, WAVES = COLUMNS / (16 * TILES), THREADS = 64 * WAVES;
    static constexpr int PAD = 16 / sizeof(T), ROW = D + PAD, COLUMN_ROW = COLUMNS + PAD, SCORES = CHUNK + PAD;      // rows start 4 (of 64) banks after each other: sixteen of them side by side in 16 bytes each meet no bank twice
    static constexpr int PLANES = PARTS<T>;
    // keys, values, what the slope is multiplied with, the queries, the scores: in the queries' place (for a barrier more) where that leaves room for another workgroup, which 128 channels of two bytes have no registers for
    static constexpr bool OVER = !(D == 128 && sizeof(T) == 2 && !SLOPE);
    static constexpr int K = 0, V = K + CHUNK * ROW, W = V + CHUNK * COLUMN_ROW, Q = W + (SLOPE && !STATE ? CHUNK * COLUMN_ROW : 0), P = OVER ? Q : Q + CHUNK * ROW;
    static constexpr int FLAGS = STATE ? Q : OVER && ROW > PLANES * SCORES ? Q + CHUNK * ROW : P + CHUNK * PLANES * SCORES;
    static constexpr int SCORE_TILES = (10 + WAVES - 1) / WAVES;      // of a wavefront
    static constexpr size_t BYTES = FLAGS * sizeof(T) + (4 * CHUNK + 16 + 2 * WAVES) * sizeof(float);
    // wavefronts that the registers of a SIMD are shared by: as many as LDS has room for workgroups
    static constexpr int FIT = (int)(163840 / BYTES) * WAVES / 4, MOST = D == 128 || (SLOPE && !STATE) ? 2 : 3, RESIDENT = FIT < 1 ? 1 : FIT > MOST ? MOST : FIT;
};

// Chunks of up to 64 steps. With i, s the steps of a chunk (n of them within the row's length), S the state before it and a the decay:
//     out_i = sum over s <= i of a^(i-s) (q_i k_s) v_s + a^(i+1) q_i S,     S <- a^n S + sum over s of a^(n-1-s) k_s^T v_s
// where a reset between the two steps of a power makes it zero. REVERSE is the transposed recurrence of the gradients, from the last step to the first:
//     out_i = sum over s >= i of a^(s-i) (q_i k_s) v_s + a^(n-1-i) q_i R,   R <- a (a^(n-1) R + sum over s of a^s k_s^T v_s).
// A wavefront owns some of the value columns: their state stays in its accumulators from chunk to chunk, laid out as the matrix instruction leaves them, which is (with the summands in an order of their own) how the
// product with the queries takes them. Scores of a chunk are shared out in tiles of 16 x 16, weighted, and exchanged through LDS. SLOPE carries the state's derivative by the decay's logarithm along.
// STATE: only the state, of a segment that starts from nothing. A launch may hold two walks over the same rows (gradients of keys and of values), whose workgroups take turns on an XCD and so find each other's inputs in its L2.
// What bounds it: whole heads of 128 bfloat16 channels, the vector and matrix instructions of two wavefronts a SIMD (81 to 83 % busy) beside 1.3 to 1.8 TB/s: 4 rows x 16 heads, 8,192 steps, a walk forward 206 us, d_q with the slope 439, d_k and d_v 382;
// 16,384 steps of 16 heads forward 140 to 150 us in all. Short sequences in fp32, the parts of one chunk one after the other in eight wavefronts a compute unit, as many as LDS has room for (36 KB a workgroup of 32 channels): 64 steps,
// 1,024 rows, 2 heads of 32: 34, 55 and 56 us, of which the matrix instructions take 8, 14 and 15. Fewer rows and heads than compute units leave a chunk's latency alone: 333 steps, 37 rows, 6 heads of 24 x 41: 47, 73 and 67 us.
// Few steps on many rows: reading and writing the states, two wavefronts a SIMD: 20 steps, 2,240 rows, 8 heads of 64, bfloat16: 217, 382 and 386 us.
// Steps that go back in memory take the kernel for any width: 1,024 steps, 64 rows, 8 heads of 64, fp32: 207 us, 190 with steps that go forward.
struct Walks { Walk first, second; int items, two; };
template <typename T, typename O, int D, bool REVERSE, bool SLOPE, bool STATE, bool FULL> __global__ __launch_bounds__((Layout<T, D, SLOPE, STATE>::THREADS), (Layout<T, D, SLOPE, STATE>::RESIDENT)) void walk_kernel(Walks walks) {
    typedef typename Operand<T>::Vector Vector;
    typedef typename Operand<T>::Quad Quad;
    typedef Layout<T, D, SLOPE, STATE> L;
    constexpr int KEY_TILES = D / 16, KEY_BLOCKS = D / 32, TILES = L::TILES;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_bytes[];
    T* const lds = (T*)lds_bytes;
    // weights of a chunk's steps: in the state after it, and of the state before it in their outputs
    float* const added_weights = (float*)(lds_bytes + L::FLAGS * sizeof(T)); float* const read_weights = added_weights + CHUNK; float* const lagged_weights = read_weights + CHUNK;
    float* const score_weights = lagged_weights + CHUNK + 16; float* const flags = score_weights + CHUNK;      // of scores by their lag, -16 ... 63 (zero below 0)
    const bool other = walks.two && (blockIdx.x / 8) % 2;
    const int item = (walks.two ? blockIdx.x / 16 * 8 + blockIdx.x % 8 : blockIdx.x) / L::SPLIT, half = L::SPLIT > 1 ? blockIdx.x % L::SPLIT : 0;
    if (item >= walks.items) return;
    const Walk& a = other ? walks.second : walks.first;
    const int pair = item / a.segments, segment = item % a.segments, b = pair / a.heads, h = pair % a.heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int l = lane & 15, quarter = lane >> 4;
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.steps) : a.steps;
    const Log2 log2_decay(a.log_decay[h]);
    const bool grows = log2_decay.high >= 2.0f;      // weights of a chunk may be infinite: scores of zero (of steps beyond the chunk's n) are kept from them
    const bool last = segment == (REVERSE ? 0 : a.segments - 1);      // of the walk
    if (STATE && last && !a.last_wanted) return;                      // no segment starts from the state after it
    const int begin = segment * a.segment_steps, end = min(begin + a.segment_steps, a.steps);

    // state: tile k, element r of this lane is row 16 k + 4 quarter + r, column 16 (TILES wave + tile) + l
    rlt_f32x4 state[TILES][KEY_TILES], slope[SLOPE ? TILES : 1][SLOPE ? KEY_TILES : 1];
    const int part0 = half * L::COLUMNS, inner0 = 16 * TILES * wave, column0 = part0 + inner0;      // first column of the workgroup, of the wavefront within it, of the wavefront
    const bool idle = !FULL && column0 >= a.value;      // a wavefront without columns, which takes part in loads and scores
    if (L::SPLIT > 1 && !FULL && part0 >= a.value) {    // a workgroup without any
        if (SLOPE && !STATE && threadIdx.x == 0) a.partial[item * L::SPLIT + half] = 0.0;
        return;
    }
    const size_t state_base = (size_t)item * a.key * a.value;
    const int state_key = a.state_key, state_value = a.state_value;
    auto over_state = [&](auto f) {
#pragma unroll
        for (int tile = 0; tile < TILES; tile++)
#pragma unroll
            for (int k = 0; k < KEY_TILES; k++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = 16 * k + 4 * quarter + r, column = column0 + 16 * tile + l;
                    f(tile, k, r, FULL || (row < a.key && column < a.value), row * state_key + column * state_value);
                }
    };
    over_state([&](int tile, int k, int r, bool there, int i) {
        state[tile][k][r] = 0.0f;
        if constexpr (SLOPE) slope[tile][k][r] = 0.0f;
    });
    // f(tile, k, the four elements r = 0 ... 3 of a state in memory). Those of a state that is read across lie side by side: one load of 16 bytes. Elements outside are read as the first one and dropped when all have
    // been asked for: a branch or a choice behind each would wait for each.
    typedef float Four __attribute__((ext_vector_type(4), aligned(4)));
    auto read_state = [&](const float* from, auto f) {
        const bool across = state_key == 1 && (FULL || a.key % 4 == 0);
#pragma unroll
        for (int tile = 0; tile < TILES; tile++)
#pragma unroll
            for (int k = 0; k < KEY_TILES; k++) {
                const int row = 16 * k + 4 * quarter, column = column0 + 16 * tile + l;
                rlt_f32x4 x;
                if (across) x = *reinterpret_cast<const Four*>(from + (FULL || (row < a.key && column < a.value) ? row + column * state_value : 0));
                else {
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = from[FULL || (row + r < a.key && column < a.value) ? (row + r) * state_key + column * state_value : 0];
                }
                f(tile, k, x);
            }
    };
    if (const float* from = STATE ? nullptr : a.entry) {
        read_state(from + state_base, [&](int tile, int k, rlt_f32x4 x) { state[tile][k] = x; });
        if (!FULL) over_state([&](int tile, int k, int r, bool there, int i) { if (!there) state[tile][k][r] = 0.0f; });
    }
    if constexpr (SLOPE && !STATE)
        if (const float* from = a.entry_slope) {
            read_state(from + state_base, [&](int tile, int k, rlt_f32x4 x) { slope[tile][k] = x; });
            if (!FULL) over_state([&](int tile, int k, int r, bool there, int i) { if (!there) slope[tile][k][r] = 0.0f; });
        }

    // what a thread carries from memory to LDS, in rounds: 16 bytes of a step of each tensor, of all D channels or of the workgroup's columns
    typedef typename Operand<T>::Bytes16 Bytes16;
    constexpr int V = 16 / sizeof(T), ROUNDS = CHUNK * D / (V * L::THREADS), COLUMN_ROUNDS = CHUNK * L::COLUMNS / (V * L::THREADS);
    Bytes16 next_q[STATE ? 1 : ROUNDS], next_k[ROUNDS], next_v[COLUMN_ROUNDS], next_with[SLOPE && !STATE ? COLUMN_ROUNDS : 1];
    uint8_t next_reset = 0;
    constexpr std::integral_constant<int, D> whole{};
    constexpr std::integral_constant<int, L::COLUMNS> columns{};
    // Whole chunks of whole heads: a uniform address and a thread's offset in bytes, which is added without a sign (32 bits: the steps of FULL tensors go forward in memory and leave room).
    auto offset_of = [&](const Part& p, int from, auto across) {
        constexpr int ACROSS = decltype(across)::value;
        unsigned thread = threadIdx.x;
        if constexpr (SLOPE && !STATE) asm volatile("" : "+v"(thread));      // formed anew for each chunk
        return (thread / (ACROSS / V) * (unsigned)p.step + from + thread % (ACROSS / V) * V) * (unsigned)sizeof(T);
    };
    auto fetch = [&](const Part& p, int from, int width, int t0, int stop, auto& to, auto across) {
        constexpr int ACROSS = decltype(across)::value, N = CHUNK * ACROSS / (V * L::THREADS), STEPS = L::THREADS * V / ACROSS;
        const T* const row0 = at<T>(p, t0, b, h);
        if (FULL && stop - t0 == CHUNK) {
            const unsigned offset = offset_of(p, from, across);
#pragma unroll
            for (int round = 0; round < N; round++) to[round] = *reinterpret_cast<const Bytes16*>(reinterpret_cast<const char*>(row0 + (round * STEPS) * p.step) + offset);
        } else if (stop <= t0) {
#pragma unroll
            for (int round = 0; round < N; round++) to[round] = Bytes16{};
        } else {      // what lies outside is read from inside and dropped: no branch between the loads
            int thread = threadIdx.x;
            asm volatile("" : "+v"(thread));
            const int channel = from + (thread % (ACROSS / V)) * V, first = thread / (ACROSS / V), most = stop - t0 - 1;
            if (FULL) {
#pragma unroll
                for (int round = 0; round < N; round++) {
                    const int step = first + round * STEPS;
                    to[round] = *reinterpret_cast<const Bytes16*>(row0 + min(step, most) * p.step + channel);
                    if (step > most) to[round] = Bytes16{};
                }
            } else if (width >= V) {      // dropped by settle, when it is needed: no load is waited for here. Vectors start at any element, which the memory instructions allow.
                typedef T Anywhere __attribute__((ext_vector_type(V), aligned(sizeof(T))));
#pragma unroll
                for (int round = 0; round < N; round++) to[round] = *reinterpret_cast<const Anywhere*>(row0 + min(first + round * STEPS, most) * p.step + min(channel, width - V));
            } else {
#pragma unroll
                for (int round = 0; round < N; round++) {
                    const T* const row = row0 + min(first + round * STEPS, most) * p.step;
#pragma unroll
                    for (int c = 0; c < V; c++) to[round][c] = channel + c < width ? row[channel + c] : (T)0.0f;
                }
            }
        }
    };
    // !FULL: what fetch has read from elsewhere, steps beyond the chunk's n and channels beyond the width
    auto settle = [&](int from, int width, int n, auto& to, auto across) {
        constexpr int ACROSS = decltype(across)::value, N = CHUNK * ACROSS / (V * L::THREADS), STEPS = L::THREADS * V / ACROSS;
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        const int channel = from + (thread % (ACROSS / V)) * V, first = thread / (ACROSS / V), beyond = width >= V ? channel + V - width : 0;
        if (beyond > 0 && beyond < V) {
#pragma unroll
            for (int round = 0; round < N; round++) to[round] = __builtin_bit_cast(Bytes16, __builtin_bit_cast(unsigned __int128, to[round]) >> (beyond * 8 * (int)sizeof(T)));      // elements move down to their channels, zeros behind them
        }
#pragma unroll
        for (int round = 0; round < N; round++) if (first + round * STEPS >= n || beyond >= V) to[round] = Bytes16{};
    };
    auto settle_chunk = [&](int n) {
        if constexpr (!FULL) {
            if constexpr (!STATE) settle(0, a.key, n, next_q, whole);
            settle(0, a.key, n, next_k, whole);
            settle(part0, a.value, n, next_v, columns);
            if constexpr (SLOPE && !STATE) settle(part0, a.value, n, next_with, columns);
        }
    };
    // products over a chunk's steps, sixteen to a tile: one, two or all four tiles
    auto by_steps = [&](int n, auto f) {
        if (n > 32) f(std::integral_constant<int, 4>{}); else if (n > 16) f(std::integral_constant<int, 2>{}); else if (n > 0) f(std::integral_constant<int, 1>{});
    };
    auto steps_of = [&](int t0, int stop) { return min(max(min(length, stop) - t0, 0), CHUNK); };
    auto fetch_chunk = [&](int t0, int stop) {
        stop = min(stop, length);
        if constexpr (!STATE) fetch(a.q, 0, a.key, t0, stop, next_q, whole);
        fetch(a.k, 0, a.key, t0, stop, next_k, whole);
        fetch(a.v, part0, a.value, t0, stop, next_v, columns);
        if constexpr (SLOPE && !STATE) fetch(a.with, part0, a.value, t0, stop, next_with, columns);
        next_reset = a.reset && t0 + lane < stop ? a.reset[(size_t)(t0 + lane) * a.batch + b] : (uint8_t)0;
    };
    auto put = [&](int base, const auto& from, auto across) {
        constexpr int ACROSS = decltype(across)::value, N = CHUNK * ACROSS / (V * L::THREADS), STEPS = L::THREADS * V / ACROSS;
        const int channel = (threadIdx.x % (ACROSS / V)) * V, first = threadIdx.x / (ACROSS / V);
#pragma unroll
        for (int round = 0; round < N; round++) *reinterpret_cast<Bytes16*>(lds + base + (first + round * STEPS) * (ACROSS + L::PAD) + channel) = from[round];
    };
    // operands: eight summands 32 block + 8 quarter ... of a row; of a row in the order of the accumulators; of column 16 tile + l over the steps
    auto row_operand = [&](int base, int stride, int row, int block) { return *reinterpret_cast<const Vector*>(lds + base + row * stride + 32 * block + 8 * quarter); };
    auto tiled_operand = [&](int base, int row, int block) {
        const Quad x = *reinterpret_cast<const Quad*>(lds + base + row * L::ROW + 32 * block + 4 * quarter), y = *reinterpret_cast<const Quad*>(lds + base + row * L::ROW + 32 * block + 16 + 4 * quarter);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto column_operand = [&](int base, int stride, int tile, int block) {
        if constexpr (sizeof(T) == 2) {      // the transposing load: of sixteen lanes, lane p names four channels 4 (p % 4) ... of step p / 4, and lane l receives channel l of the four steps
            typedef short Raw __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) Raw* Address;
            T* const from = lds + base + (32 * block + 8 * quarter + l / 4) * stride + 16 * tile + 4 * (l % 4);
            const Raw x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Address)from), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Address)(from + 4 * stride));
            return __builtin_bit_cast(Vector, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            Vector x;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = lds[base + (32 * block + 8 * quarter + e) * stride + 16 * tile + l];
            return x;
        }
    };

    if (!STATE && wave == 0) {
        if (lane < 16) score_weights[lane - 16] = 0.0f;
        score_weights[lane] = power(log2_decay, lane) * a.score_scale;
    }
    O* const lane_out = STATE ? nullptr : at<O>(a.out, 0, b, h) + l * a.out.step + column0 + 4 * quarter;
    double total = 0.0;                                 // SLOPE: of terms of either sign, which leave little of each other
    int weights_n = -1; uint64_t weights_resets = 0;    // the steps and the resets that the weights in LDS are for
    int counted = 0; bool forgotten = false;            // STATE
    // no state before the first steps, none asked for after the last: the products are left out
    bool nothing = !STATE && !a.entry;
    const bool last_unread = !STATE && !a.exit && !(SLOPE && a.d_final && last);
    int t0 = REVERSE ? max(begin, end - CHUNK) : begin, stop = REVERSE ? end : min(begin + CHUNK, end);
    fetch_chunk(t0, stop);
    while (true) {
        if constexpr (SLOPE && !STATE) {      // two states leave no registers for addresses that hold from chunk to chunk: they are formed anew
            asm volatile("" : "+v"(l));
            asm volatile("" : "+v"(quarter));
        }
        uint64_t resets = __ballot(next_reset != 0);
        int n = steps_of(t0, stop);
        settle_chunk(n);
        if (resets & ~1ull) {
            // A step's weight of zero keeps other episodes out of sums of products as long as their values are finite. Where some are not, the chunk ends at its first reset (REVERSE: begins at its last).
            const bool some = __any(not_finite(next_k) || not_finite(next_v));
            if (lane == 0) flags[wave] = some ? 1.0f : 0.0f;
        }
        rlt_lds_barrier();
        if (resets & ~1ull) {
            float any = 0.0f;
            for (int w = 0; w < L::WAVES; w++) any += flags[w];
            if (any != 0.0f) {
                if (REVERSE) t0 += 63 - __builtin_clzll(resets); else stop = t0 + __builtin_ctzll(resets & ~1ull);
                fetch_chunk(t0, stop);
                resets = __ballot(next_reset != 0);
                n = steps_of(t0, stop);
                settle_chunk(n);
            }
        }
        const int last_reset = resets ? 63 - __builtin_clzll(resets) : -1, first_reset = resets ? __builtin_ctzll(resets) : CHUNK;
        if (n != weights_n || resets != weights_resets) {
            weights_n = n; weights_resets = resets;
            if (wave == 0) {
                const bool in = lane < n && (REVERSE ? lane < first_reset : lane >= last_reset), sees = lane < n && (REVERSE ? last_reset <= lane : first_reset > lane);
                added_weights[lane] = in ? power(log2_decay, REVERSE ? lane : n - 1 - lane) * a.added_scale : 0.0f;
                if constexpr (SLOPE) lagged_weights[lane] = added_weights[lane] * (float)(n - 1 - lane);
                read_weights[lane] = sees ? power(log2_decay, REVERSE ? n - 1 - lane : lane + 1) * a.read_scale : 0.0f;
            }
        }
        put(L::K, next_k, whole);
        put(L::V, next_v, columns);
        if constexpr (!STATE) {
            const bool some = __any(not_finite(next_v));
            if (lane == 0) flags[L::WAVES + wave] = some ? 1.0f : 0.0f;
        }
        if constexpr (!STATE) put(L::Q, next_q, whole);
        if constexpr (SLOPE && !STATE) put(L::W, next_with, columns);
        rlt_lds_barrier();
        const bool done = REVERSE ? t0 <= begin : stop >= end;
        const int next_t0 = REVERSE ? max(begin, t0 - CHUNK) : stop, next_stop = REVERSE ? t0 : min(stop + CHUNK, end);
        if constexpr (!SLOPE || STATE) { if (!done) fetch_chunk(next_t0, next_stop); }

        if constexpr (!STATE) {
            // scores, by tiles on and below (REVERSE: above) the diagonal: rows are the steps that are added, columns those that read
            rlt_f32x4 score[L::SCORE_TILES];
            int first_tile = wave;
            asm volatile("" : "+s"(first_tile));      // the tiles' addresses are formed here, not kept in registers from chunk to chunk
#pragma unroll
            for (int j = 0; j < L::SCORE_TILES; j++) {
                const int tile = first_tile + j * L::WAVES, row = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, col = tile - row * (row + 1) / 2, ot = REVERSE ? 3 - row : row, st = REVERSE ? 3 - col : col;
                if (tile >= 10) break;
                score[j] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (16 * (REVERSE ? st : ot) >= n) continue;
                rlt_f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int block = 0; block < KEY_BLOCKS; block++) if (FULL || 32 * block < a.key) x = multiply(row_operand(L::K, L::ROW, 16 * st + l, block), row_operand(L::Q, L::ROW, 16 * ot + l, block), x);
                if constexpr (SLOPE) {
#pragma unroll
                    for (int block = 0; block < L::COLUMNS / 32; block++) if (FULL || part0 + 32 * block < a.value) y = multiply(row_operand(L::V, L::COLUMN_ROW, 16 * st + l, block), row_operand(L::W, L::COLUMN_ROW, 16 * ot + l, block), y);
                }
                const int i = 16 * ot + l;
                const float* const weight = score_weights + (REVERSE ? 16 * (st - ot) + 4 * quarter - l : 16 * (ot - st) + l - 4 * quarter);
                if (grows) {
#pragma unroll
                    for (int r = 0; r < 4; r++) { const float w = weight[REVERSE ? r : -r]; x[r] = w != 0.0f && x[r] != 0.0f ? x[r] * w : 0.0f; }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++) { const float w = weight[REVERSE ? r : -r]; x[r] = w != 0.0f ? x[r] * w : 0.0f; }
                }
                if (resets) {
                    const uint64_t before = resets & ((2ull << i) - 1), after = i < 63 ? resets & ~((2ull << i) - 1) : 0;
                    const int low = REVERSE ? 0 : before ? 63 - __builtin_clzll(before) : 0, high = REVERSE && after ? __builtin_ctzll(after) - 1 : 63;      // steps of the episode of step i
#pragma unroll
                    for (int r = 0; r < 4; r++) { const int s = 16 * st + 4 * quarter + r; x[r] = s >= low && s <= high ? x[r] : 0.0f; }
                }
                if constexpr (SLOPE) {
#pragma unroll
                    for (int r = 0; r < 4; r++) { const int s = 16 * st + 4 * quarter + r; if (x[r] != 0.0f) total += (double)x[r] * ((float)(REVERSE ? s - i : i - s) * y[r]); }
                }
                score[j] = x;
                __builtin_amdgcn_sched_barrier(0);      // one tile in registers at a time
            }
            // what the state before the chunk gives: columns of the result are the steps, rows the value columns
            rlt_f32x4 out[TILES][4], out_slope[SLOPE ? TILES : 1][SLOPE ? 4 : 1];
#pragma unroll
            for (int tile = 0; tile < TILES; tile++)
#pragma unroll
                for (int ot = 0; ot < 4; ot++) {
                    out[tile][ot] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (SLOPE) out_slope[tile][ot] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            auto before = [&](auto tiles) {
                constexpr int STEP_TILES = decltype(tiles)::value;
#pragma unroll
            for (int block = 0; block < KEY_BLOCKS; block++) {
                if (!FULL && 32 * block >= a.key) break;
                Vector q[STEP_TILES];
#pragma unroll
                for (int ot = 0; ot < STEP_TILES; ot++) q[ot] = tiled_operand(L::Q, 16 * ot + l, block);
#pragma unroll
                for (int tile = 0; tile < TILES; tile++) {
                    const Cut<T> s(__builtin_shufflevector(state[tile][2 * block], state[tile][2 * block + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int p = 0; p < PARTS<T>; p++)
#pragma unroll
                        for (int ot = 0; ot < STEP_TILES; ot++) out[tile][ot] = multiply(s.part[p], q[ot], out[tile][ot]);
                    if constexpr (SLOPE) {
                        const Cut<T> d(__builtin_shufflevector(slope[tile][2 * block], slope[tile][2 * block + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                        for (int p = 0; p < PARTS<T>; p++)
#pragma unroll
                            for (int ot = 0; ot < STEP_TILES; ot++) out_slope[tile][ot] = multiply(d.part[p], q[ot], out_slope[tile][ot]);
                    }
                }
                if constexpr (SLOPE) __builtin_amdgcn_sched_barrier(0);      // one block's operands in registers at a time
            }
#pragma unroll
            for (int ot = 0; ot < STEP_TILES; ot++) {
                const int i = 16 * ot + l;
                const float weight = read_weights[i];
#pragma unroll
                for (int tile = 0; tile < TILES; tile++) {
                    if constexpr (SLOPE) {
                        const Quad with = *reinterpret_cast<const Quad*>(lds + L::W + i * L::COLUMN_ROW + inner0 + 16 * tile + 4 * quarter);
                        float d = 0.0f;
#pragma unroll
                        for (int r = 0; r < 4; r++) d = fmaf((float)with[r], fmaf((float)(i + 1), out[tile][ot][r], out_slope[tile][ot][r]), d);
                        if (weight != 0.0f) total += (double)weight * d;
                    }
                    if (resets) {      // a state of another episode need not be finite
#pragma unroll
                        for (int r = 0; r < 4; r++) out[tile][ot][r] = weight != 0.0f ? out[tile][ot][r] * weight : 0.0f;
                    } else out[tile][ot] *= weight;
                }
            }
            };
            if (!nothing && !idle) by_steps(n, before);
            if constexpr (L::OVER) rlt_lds_barrier();      // the queries have been read
#pragma unroll
            for (int j = 0; j < L::SCORE_TILES; j++) {
                const int tile = first_tile + j * L::WAVES, row = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, col = tile - row * (row + 1) / 2, ot = REVERSE ? 3 - row : row, st = REVERSE ? 3 - col : col;
                if (tile >= 10) break;
#pragma unroll
                for (int plane = 0; plane < L::PLANES; plane++) {
                    const Quad part = __builtin_convertvector(score[j], Quad);
                    *reinterpret_cast<Quad*>(lds + L::P + plane * CHUNK * L::SCORES + (16 * ot + l) * L::SCORES + 16 * st + 4 * quarter) = part;
                    if (plane + 1 < L::PLANES) score[j] -= __builtin_convertvector(part, rlt_f32x4);
                }
            }
            // the tiles on the wrong side of the diagonal that are multiplied all the same, as halves of blocks of 32
            for (int which = wave; which < 2 * L::PLANES; which += L::WAVES)
                *reinterpret_cast<Quad*>(lds + L::P + which / 2 * CHUNK * L::SCORES + (32 * (which % 2) + (REVERSE ? 16 : 0) + l) * L::SCORES + 32 * (which % 2) + (REVERSE ? 0 : 16) + 4 * quarter) = Quad{};
            float apart = 0.0f;
#pragma unroll
            for (int w = 0; w < L::WAVES; w++) apart += flags[L::WAVES + w];
            rlt_lds_barrier();
            if constexpr (SLOPE) { if (!done) fetch_chunk(next_t0, next_stop); }      // only here: the products with two states before leave no registers for it
            // what the chunk's own steps give
            auto within = [&](auto tiles) {
                constexpr int STEP_TILES = decltype(tiles)::value;
#pragma unroll
            for (int block = 0; block < (STEP_TILES + 1) / 2; block++) {
                Vector values[TILES];
#pragma unroll
                for (int tile = 0; tile < TILES; tile++) values[tile] = column_operand(L::V, L::COLUMN_ROW, TILES * wave + tile, block);
#pragma unroll
                for (int ot = 0; ot < STEP_TILES; ot++)
                    if (REVERSE ? 32 * block + 31 >= 16 * ot : 32 * block <= 16 * ot + 15) {
#pragma unroll
                        for (int plane = 0; plane < L::PLANES; plane++) {
                            const Vector scores = row_operand(L::P + plane * CHUNK * L::SCORES, L::SCORES, 16 * ot + l, block);
#pragma unroll
                            for (int tile = 0; tile < TILES; tile++) out[tile][ot] = multiply(values[tile], scores, out[tile][ot]);
                        }
                    }
            }
            };
            if (__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, apart)) == 0) { if (!idle) by_steps(n, within); }
            else if (!idle) {      // zero times a value that is not finite is not zero: one step after the other goes to the steps that see it
#pragma unroll 1
                for (int s = 0; s < n; s++)
#pragma unroll
                    for (int ot = 0; ot < 4; ot++) {
                        const int i = 16 * ot + l;
                        float weight = 0.0f;
#pragma unroll
                        for (int plane = 0; plane < L::PLANES; plane++) weight += (float)lds[L::P + plane * CHUNK * L::SCORES + i * L::SCORES + s];
#pragma unroll
                        for (int tile = 0; tile < TILES; tile++) {
                            const Quad v = *reinterpret_cast<const Quad*>(lds + L::V + s * L::COLUMN_ROW + inner0 + 16 * tile + 4 * quarter);
#pragma unroll
                            for (int r = 0; r < 4; r++) { const float x = fmaf(weight, (float)v[r], out[tile][ot][r]); out[tile][ot][r] = (REVERSE ? s >= i : s <= i) ? x : out[tile][ot][r]; }
                        }
                    }
            }
            typedef typename Operand<O>::Quad OutQuad;
            O* const to = lane_out + t0 * a.out.step;
#pragma unroll
            for (int ot = 0; ot < 4; ot++) {
                const int i = 16 * ot + l;
                if (t0 + i < stop) {
#pragma unroll
                    for (int tile = 0; tile < TILES; tile++) {
                        const int c0 = column0 + 16 * tile + 4 * quarter;
                        rlt_f32x4 x = out[tile][ot];
                        if (n < CHUNK && i >= n) x = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        O* const here = to + (int64_t)(16 * ot) * a.out.step + 16 * tile;
                        if (FULL) *reinterpret_cast<OutQuad*>(here) = __builtin_convertvector(x, OutQuad);
                        else if (c0 + 4 <= a.value) {
                            typedef O Anywhere __attribute__((ext_vector_type(4), aligned(sizeof(O))));
                            *reinterpret_cast<Anywhere*>(here) = __builtin_convertvector(x, Anywhere);
                        } else {
#pragma unroll
                            for (int r = 0; r < 3; r++) if (c0 + r < a.value) here[r] = (O)x[r];
                        }
                    }
                }
            }
        }
        // the state after the chunk
        if (n > 0 && !(done && last_unread) && !idle) {
            nothing = false;
            const float f = power(log2_decay, REVERSE ? n - 1 : n);
            counted += n; forgotten |= resets != 0;
#pragma unroll
            for (int tile = 0; tile < TILES; tile++)
#pragma unroll
                for (int k = 0; k < KEY_TILES; k++) {
                    if (resets) {
                        state[tile][k] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        if constexpr (SLOPE) slope[tile][k] = rlt_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    } else {
                        if constexpr (SLOPE) slope[tile][k] = f * (slope[tile][k] + (float)n * state[tile][k]);
                        state[tile][k] *= f;
                    }
                }
#pragma unroll
            for (int block = 0; block < 2; block++) {
                if (32 * block >= n) break;
                const rlt_f32x8 weight = *reinterpret_cast<const rlt_f32x8*>(added_weights + 32 * block + 8 * quarter);
                constexpr bool TOGETHER = !SLOPE && FULL;      // all key operands in registers, else one at a time, as far as there are keys
                Vector key[TOGETHER ? KEY_TILES : 1];
                if constexpr (TOGETHER) {
#pragma unroll
                    for (int k = 0; k < KEY_TILES; k++) key[k] = column_operand(L::K, L::ROW, k, block);
                }
#pragma unroll
                for (int tile = 0; tile < TILES; tile++) {
                    const Vector v = column_operand(L::V, L::COLUMN_ROW, TILES * wave + tile, block);
                    const rlt_f32x8 weighted = __builtin_convertvector(v, rlt_f32x8) * weight;
                    const Cut<T> x(weighted);
                    if constexpr (SLOPE) {
                        const rlt_f32x8 lagged = __builtin_convertvector(v, rlt_f32x8) * *reinterpret_cast<const rlt_f32x8*>(lagged_weights + 32 * block + 8 * quarter);
                        const Cut<T> y(lagged);
#pragma unroll
                        for (int k = 0; k < KEY_TILES; k++) {
                            if (!FULL && 16 * k >= a.key) break;
                            key[0] = column_operand(L::K, L::ROW, k, block);
#pragma unroll
                            for (int p = 0; p < PARTS<T>; p++) {
                                state[tile][k] = multiply(key[0], x.part[p], state[tile][k]);
                                slope[tile][k] = multiply(key[0], y.part[p], slope[tile][k]);
                            }
                        }
                    } else if constexpr (!TOGETHER) {
#pragma unroll
                        for (int k = 0; k < KEY_TILES; k++) {
                            if (16 * k >= a.key) break;
                            key[0] = column_operand(L::K, L::ROW, k, block);
#pragma unroll
                            for (int p = 0; p < PARTS<T>; p++) state[tile][k] = multiply(key[0], x.part[p], state[tile][k]);
                        }
                    } else {
#pragma unroll
                        for (int p = 0; p < PARTS<T>; p++) {
#pragma unroll
                            for (int k = 0; k < KEY_TILES; k++) state[tile][k] = multiply(key[k], x.part[p], state[tile][k]);
                        }
                    }
                }
                if constexpr (SLOPE) __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (REVERSE) {      // the power that all of them share: the cut operands keep their parts above the smallest numbers also where one step forgets nearly everything
                const float once = power(log2_decay, 1);
#pragma unroll
                for (int tile = 0; tile < TILES; tile++)
#pragma unroll
                    for (int k = 0; k < KEY_TILES; k++) state[tile][k] *= once;
            }
        }
        if (done) break;
        t0 = next_t0; stop = next_stop;
    }

    if (float* to = a.exit) {
        to += state_base;
        over_state([&](int tile, int k, int r, bool there, int i) { if (there) to[i] = state[tile][k][r]; });
    }
    if constexpr (SLOPE && STATE) {
        float* const to = a.exit_slope + state_base;
        over_state([&](int tile, int k, int r, bool there, int i) { if (there) to[i] = slope[tile][k][r]; });
    }
    if constexpr (STATE) { if (threadIdx.x == 0 && half == 0) a.factors[item] = make_float2(forgotten ? 0.0f : power(log2_decay, counted), (float)counted); }
    if constexpr (SLOPE && !STATE) {
        if (a.d_final && last) {
            read_state(a.d_final + (size_t)pair * a.key * a.value, [&](int tile, int k, rlt_f32x4 x) {
#pragma unroll
                for (int r = 0; r < 4; r++) total += (double)x[r] * slope[tile][k][r];      // zeros outside
            });
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
        asm volatile("" : "+v"(total));      // the last exchange stays ahead of the barrier
        double* const totals = (double*)added_weights;
        rlt_lds_barrier();
        if (lane == 0) totals[wave] = total;
        rlt_lds_barrier();
        if (threadIdx.x == 0) {
            double s = 0.0;
            for (int w = 0; w < L::WAVES; w++) s += totals[w];
            a.partial[item * L::SPLIT + half] = s;
        }
    }
}

// States that the segments start from, out of what each of them adds: element by element along the segments (REVERSE: from the last). locals become the entries. The values of AHEAD segments are asked for at a time.
template <bool SLOPES> __global__ __launch_bounds__(256) void scan_kernel(const float* __restrict__ initial, float* __restrict__ locals, float* __restrict__ slopes, const float2* __restrict__ factors,
                                                                          float* __restrict__ final, int elements, int segments, int reverse) {
    constexpr int AHEAD = 8;
    const int pair = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x;
    if (e >= elements) return;
    float carry = initial ? initial[(size_t)pair * elements + e] : 0.0f, carry_slope = 0.0f;
    const int added = final ? segments : segments - 1;      // segments whose own states are there
    for (int i0 = 0; i0 < segments; i0 += AHEAD) {
        float local[AHEAD], local_slope[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int i = min(i0 + j, added - 1);
            const size_t at = ((size_t)pair * segments + (reverse ? segments - 1 - i : i)) * elements + e;
            local[j] = locals[at];
            if (SLOPES) local_slope[j] = slopes[at];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (i0 + j < segments) {
                const size_t p = (size_t)pair * segments + (reverse ? segments - 1 - i0 - j : i0 + j), at = p * elements + e;
                const float2 f = i0 + j < added ? factors[p] : make_float2(0.0f, 0.0f);
                if (SLOPES) {
                    slopes[at] = carry_slope;
                    carry_slope = f.x == 0.0f ? local_slope[j] : fmaf(f.x, fmaf(f.y, carry, carry_slope), local_slope[j]);
                }
                locals[at] = carry;
                carry = f.x == 0.0f ? local[j] : fmaf(f.x, carry, local[j]);
            }
    }
    if (final) final[(size_t)pair * elements + e] = carry;
}

// sums over the rows of a batch and their segments (and the workgroups that share one), in a fixed order: a workgroup per head
__global__ __launch_bounds__(512) void decay_sum_kernel(const double* __restrict__ partial, int batch, int heads, int segments, float* __restrict__ out, int accumulate) {
    __shared__ double sums[8];
    const int h = blockIdx.x;
    double s = 0.0;
    for (int i = threadIdx.x; i < batch * segments; i += 512) s += partial[((size_t)(i / segments) * heads + h) * segments + i % segments];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) s += sums[w];
        out[h] = (float)(accumulate ? out[h] + s : s);
    }
}

// gradients of shared keys and values: the sums over the heads that read them. A workgroup takes the elements of some tokens at a time; those of keys and of values are two rows of the grid.
// V elements of a head at a time: four (16 bytes of each share) where the widths are multiples of four.
struct HeadSum { const float* parts; Part out; int width; };
template <typename T, int V> __global__ __launch_bounds__(256) void head_sum_kernel(HeadSum first, HeadSum second, size_t tokens, int batch, int kv_heads, int group) {
    typedef float vector __attribute__((ext_vector_type(V)));
    typedef T OutVector __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    const HeadSum& a = blockIdx.y ? second : first;
    const int width = a.width / V, elements = kv_heads * width, at_once = elements < 1024 ? 1024 / elements : 1;
    for (size_t token0 = (size_t)blockIdx.x * at_once; token0 < tokens; token0 += (size_t)gridDim.x * at_once) {
        const int there = tokens - token0 < (size_t)at_once ? (int)(tokens - token0) : at_once, t0 = (int)(token0 / batch), b0 = (int)(token0 % batch);
        for (int i = threadIdx.x; i < there * elements; i += 256) {
            const int token = i / elements, e = i - token * elements, h = e / width, c = (e - h * width) * V, steps = (b0 + token) / batch;
            const float* const parts = a.parts + (((token0 + token) * kv_heads + h) * group) * a.width + c;
            vector s = {};
            for (int g = 0; g < group; g++) s += *reinterpret_cast<const vector*>(parts + (size_t)g * a.width);
            *reinterpret_cast<OutVector*>(at<T>(a.out, t0 + steps, b0 + token - steps * batch, h) + c) = __builtin_convertvector(s, OutVector);
        }
    }
}

// One step of a row and head by THREADS threads, a wavefront or a workgroup: S = decay S + k^T v, out = scale q S, the state once in and once out (what bounds it). A thread has V columns of every G-th key, four keys' loads in flight;
// the sums over a column's keys are joined through LDS in the order of their threads. next_state may be state: each element is read and written by one thread. States of up to STEP_NARROW elements take a wavefront (4,096 rows x 4 heads of 32 x 32: 28 us,
// 85 with a workgroup each and no vectors), others a workgroup: 4,096 x 8 heads of 64 x 64: 185 us, 5.9 TB/s (202 by wavefronts); 1,024 x 4 of 128 x 128: 102 us (114); 64 x 4 of 64 x 64: 4.6 us (5.8).
// Columns that are no whole vectors are taken one by one: 4,000 x 4 heads of 50 x 37: 59 us, 4.1 TB/s.
template <typename T, int V, int THREADS> __global__ __launch_bounds__(256) void step_kernel(Walk a, unsigned pairs) {
    constexpr int AHEAD = 4;
    typedef float vector __attribute__((ext_vector_type(V)));
    __shared__ vector parts[256];
    const unsigned pair = blockIdx.x * (256 / THREADS) + (THREADS == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
    const bool work = pair < pairs;
    const int h = pair % a.heads, b = pair / a.heads, t = threadIdx.x % THREADS, columns = a.value / V, groups = THREADS / columns, g = t / columns, c = (t % columns) * V;
    vector out = {};
    if (work && a.lengths && a.lengths[b] <= 0) {      // a row without this step: its state stays, its output is zero
        const size_t base = ((size_t)b * a.heads + h) * a.key * a.value;
        for (int i = t; i < a.key * a.value; i += THREADS) a.exit[base + i] = a.entry ? a.entry[base + i] : 0.0f;
    } else if (work && g < groups) {
        const T* const q = at<T>(a.q, 0, b, h); const T* const k = at<T>(a.k, 0, b, h); const T* const values = at<T>(a.v, 0, b, h) + c;
        const size_t base = ((size_t)b * a.heads + h) * a.key * a.value + c;
        const float decay = expf(a.log_decay[h]);
        const bool forget = !a.entry || (a.reset && a.reset[b]);      // what a forgotten state holds reaches nothing, values that are not finite either
        vector v;
#pragma unroll
        for (int n = 0; n < V; n++) v[n] = (float)values[n];
        for (int i = g; i < a.key; i += AHEAD * groups) {
            vector s[AHEAD] = {};
            float ks[AHEAD], qs[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                const int at_key = i + j * groups, key = at_key < a.key ? at_key : i;
                ks[j] = (float)k[key]; qs[j] = (float)q[key];
                if (!forget) s[j] = *reinterpret_cast<const vector*>(a.entry + base + key * a.value);
            }
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                const int key = i + j * groups;
                if (key < a.key) {
#pragma unroll
                    for (int n = 0; n < V; n++) { s[j][n] = fmaf(ks[j], v[n], s[j][n] * decay); out[n] = fmaf(qs[j], s[j][n], out[n]); }
                    *reinterpret_cast<vector*>(a.exit + base + key * a.value) = s[j];
                }
            }
        }
    }
    parts[threadIdx.x] = out;
    rlt_lds_barrier();
    const float* const sums = reinterpret_cast<const float*>(parts + (threadIdx.x - t));
    for (int column = t; work && column < a.value; column += THREADS) {
        float s = 0.0f;
        for (int i = 0; i < groups && i < a.key; i++) s += sums[i * a.value + column];
        at<T>(a.out, 0, b, h)[column] = (T)(s * a.read_scale);
    }
}

template <typename T, int V = 16 / sizeof(T)> Part part(const rlt_head_view* v, int group, int width) {
    const bool vectors = reinterpret_cast<uintptr_t>(v->data) % (V * sizeof(T)) == 0 && v->step_stride % V == 0 && v->row_stride % V == 0 && v->head_stride % V == 0 && width % V == 0;
    return Part{v->data, v->step_stride, v->row_stride, v->head_stride, group, vectors};
}
bool described(const rlt_linear_attention* p) {
    return p && (p->type == RLT_TYPE_F32 || p->type == RLT_TYPE_BF16) && p->batch > 0 && p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->key_dim > 0 && p->value_dim > 0;
}
bool supported(const rlt_linear_attention* p) { return p->key_dim <= MAX_WIDTH && p->value_dim <= MAX_WIDTH && (int64_t)p->batch * p->heads <= INT32_MAX / 64; }
bool given(const rlt_head_view* v) { return v && v->data; }
size_t padded(size_t n) { return (n + 63) / 64 * 64; }

// The steps of a row and head are cut into segments where rows and heads alone leave compute units without work: their states then cost a pass over keys and values ahead of the walk, a quarter of a walk's time, and
// launches worth about four chunks. Measured (us, by segments): 8 rows x 4 heads of 64, 1,024 steps, fp32: 77 with 2, 44 with 4, 30 with 8 and 16; 8 heads of 64, 2,048 steps, bf16: 133 with 1, 22 with 16, 21 with 32;
// 4 x 16 heads of 128, 8,192 steps, bf16: 592 with 2, 317 with 4, 277 with 8, 309 with 16; forward and backward of 16 x 8 heads of 128, 256 steps, bf16: 111 with 1, 168 with 2, 197 with 4; of 37 x 6 heads of 24 x 41, 333 steps, fp32: 199 with 1, 190 to 222 with 2 to 6.
struct Segments { int count, steps; };
Segments segments_of(const rlt_linear_attention* p, int steps) {
    const int chunks = (steps + CHUNK - 1) / CHUNK;
    const double pairs = (double)p->batch * p->heads;
    int best = 1;
    double least = chunks;      // with one segment, in chunks' walks, while every row and head has a place on the chip
    if (pairs > 512) least *= pairs / 512;
    auto try_count = [&](int count) {
        if (count < 2 || count > chunks) return;
        const int per = (chunks + count - 1) / count;
        const double filled = pairs * ((chunks + per - 1) / per) / 512, cost = 1.25 * per * (filled > 1 ? filled : 1) + 4;
        if (cost < least) { least = cost; best = count; }
    };
    if (pairs < 512) {
        try_count((int)(512 / pairs));
        for (int count = 2; count <= 512 / pairs; count *= 2) try_count(count);
    }
    const int per = (chunks + best - 1) / best;
    return {(chunks + per - 1) / per, per * CHUNK};
}
// scratch memory, in floats: [states of the segments][their slopes][factors][partial sums][gradients of the heads that share keys and values]
struct Scratch { size_t states, slopes, factors, partial, shared, total; };
Scratch scratch_of(const rlt_linear_attention* p, int steps, bool backward) {
    const Segments g = segments_of(p, steps);
    const size_t pairs = (size_t)p->batch * p->heads, state = padded(pairs * g.count * p->key_dim * p->value_dim);
    Scratch s{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += padded(n); return here; };
    if (g.count > 1) {
        s.states = take(state);
        if (backward) s.slopes = take(state);
        s.factors = take(2 * pairs * g.count);
    }
    if (backward) {
        s.partial = take(4 * pairs * g.count);      // doubles, of up to two workgroups that share a head
        if (p->heads != p->kv_heads) s.shared = take(padded((size_t)steps * pairs * p->value_dim) + (size_t)steps * pairs * p->key_dim);
    }
    s.total = at;
    return s;
}

template <typename T, typename O, int D, bool REVERSE, bool SLOPE, bool STATE, bool FULL> int launch_walk(rlt_rocm_device* device, const Walk& a, const Walk* second) {
    typedef Layout<T, D, SLOPE, STATE> L;
    const auto kernel = walk_kernel<T, O, D, REVERSE, SLOPE, STATE, FULL>;
    const unsigned items = (unsigned)a.batch * a.heads * a.segments;
    RLT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)L::BYTES));
    hipLaunchKernelGGL(kernel, dim3(second ? (items + 7) / 8 * 16 : items * L::SPLIT), dim3(L::THREADS), L::BYTES, device->stream, Walks{a, second ? *second : a, (int)items, second != nullptr});
    return rlt_launch_status(device);
}
// FULL: heads of exactly D channels, all of whose tensors may be read and written in vectors
template <typename T, typename O, int D, bool REVERSE, bool SLOPE, bool STATE> int walk_width(rlt_rocm_device* device, const Walk& a, const Walk* second) {
    auto full = [&](const Walk& w) {
        auto near = [](const Part& p) { return p.step >= 0 && p.step < 1 << 22; };      // a chunk's offsets in bytes fit 32 bits without a sign; steps that go back in memory take 64-bit addresses
        if (!near(w.k) || !near(w.v) || (!STATE && !near(w.q)) || (SLOPE && !STATE && !near(w.with))) return false;
        return w.key == D && w.value == D && w.k.vectors && w.v.vectors && (STATE || (w.q.vectors && w.out.vectors)) && (!SLOPE || STATE || w.with.vectors);
    };
    return full(a) && (!second || full(*second)) ? launch_walk<T, O, D, REVERSE, SLOPE, STATE, true>(device, a, second) : launch_walk<T, O, D, REVERSE, SLOPE, STATE, false>(device, a, second);
}
template <typename T, typename O, bool REVERSE, bool SLOPE, bool STATE> int walk(rlt_rocm_device* device, const Walk& a, const Walk* second = nullptr) {
    const int width = a.key > a.value ? a.key : a.value;
    return width <= 32 ? walk_width<T, O, 32, REVERSE, SLOPE, STATE>(device, a, second) : width <= 64 ? walk_width<T, O, 64, REVERSE, SLOPE, STATE>(device, a, second)
                                                                                           : walk_width<T, O, 128, REVERSE, SLOPE, STATE>(device, a, second);
}
Walk walk_of(const rlt_linear_attention* p, const uint8_t* reset, const int32_t* lengths, int steps) {
    const Segments g = segments_of(p, steps);
    Walk a{};
    a.log_decay = p->log_decay; a.reset = reset; a.lengths = lengths; a.score_scale = a.read_scale = p->scale; a.added_scale = 1.0f;
    a.batch = p->batch; a.heads = p->heads; a.steps = steps; a.key = p->key_dim; a.value = p->value_dim; a.segments = g.count; a.segment_steps = g.steps;
    a.state_key = p->value_dim; a.state_value = 1;
    return a;
}
// states that the segments of `a` start from, in scratch memory
template <typename T, bool REVERSE, bool SLOPE> int segment_states(rlt_rocm_device* device, const Walk& a, const float* initial, float* final, float* states, float* slopes, float2* factors) {
    Walk s = a;
    s.entry = nullptr; s.exit = states; s.exit_slope = slopes; s.factors = factors; s.last_wanted = final != nullptr;
    int rc = walk<T, T, REVERSE, SLOPE, true>(device, s);
    if (rc) return rc;
    const int elements = a.key * a.value, pairs = a.batch * a.heads;
    hipLaunchKernelGGL(scan_kernel<SLOPE>, dim3((elements + 255) / 256, pairs), dim3(256), 0, device->stream, initial, states, SLOPE ? slopes : nullptr, factors, final, elements, a.segments, (int)REVERSE);
    return rlt_launch_status(device);
}

template <typename T> int launch_step(rlt_rocm_device* device, const Walk& a) {
    const unsigned pairs = (unsigned)a.heads * a.batch;
    const bool vectors = a.value % 4 == 0 && (reinterpret_cast<uintptr_t>(a.entry) | reinterpret_cast<uintptr_t>(a.exit)) % 16 == 0, narrow = a.key * a.value <= STEP_NARROW && (vectors || a.value <= 64);
    const unsigned at_once = narrow ? 4 : 1, blocks = (pairs + at_once - 1) / at_once;
    if (blocks > UINT32_MAX / 256) return RLT_E_UNSUPPORTED;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, device->stream, a, pairs); };
    if (vectors && narrow) go(step_kernel<T, 4, 64>); else if (vectors) go(step_kernel<T, 4, 256>);
    else if (narrow) go(step_kernel<T, 1, 64>); else go(step_kernel<T, 1, 256>);
    return rlt_launch_status(device);
}

// Whether a call's launches have fewer than 2^32 threads, which is what a dimension of a grid holds; asked before the first of them. `decays`: with the decays' gradient.
enum Call { FORWARD, BACKWARD };
template <typename T> bool launchable(const rlt_linear_attention* p, Call call, bool decays) {
    const uint64_t pairs = (uint64_t)p->batch * p->heads;
    auto of = [&](auto width) {
        constexpr int D = decltype(width)::value;
        typedef Layout<T, D, false, false> Plain;
        typedef Layout<T, D, true, false> Sloped;
        if (call == FORWARD) return pairs * Plain::THREADS;
        const uint64_t both = (pairs + 7) / 8 * 16 * Plain::THREADS, sloped = decays ? pairs * Sloped::SPLIT * Sloped::THREADS : 0, sums = decays ? (uint64_t)p->heads * 512 : 0;
        return both > sloped ? (both > sums ? both : sums) : (sloped > sums ? sloped : sums);
    };
    const int width = p->key_dim > p->value_dim ? p->key_dim : p->value_dim;
    return (width <= 32 ? of(std::integral_constant<int, 32>{}) : width <= 64 ? of(std::integral_constant<int, 64>{}) : of(std::integral_constant<int, 128>{})) <= UINT32_MAX;
}
bool launchable(const rlt_linear_attention* p, Call call, bool decays) { return p->type == RLT_TYPE_F32 ? launchable<float>(p, call, decays) : launchable<rlt_bf16>(p, call, decays); }

template <typename T> int forward(rlt_rocm_device* device, const rlt_linear_attention* p, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v, const rlt_head_view* output,
                                  const float* initial_state, float* final_state, const uint8_t* reset, const int32_t* lengths, int steps, float* workspace) {
    const int group = p->heads / p->kv_heads;
    const Scratch s = scratch_of(p, steps, false);
    Walk a = walk_of(p, reset, lengths, steps);
    a.q = part<T>(q, 1, p->key_dim); a.k = part<T>(k, group, p->key_dim); a.v = part<T>(v, group, p->value_dim); a.out = part<T, 4>(output, 1, p->value_dim);
    a.entry = initial_state; a.exit = final_state;
    if (steps == 1 && final_state) return launch_step<T>(device, a);      // a pass over the states (9,639 rows, one head of 118, fp32: 235 us; 551 as a walk of one step)
    if (a.segments > 1) {
        const int rc = segment_states<T, false, false>(device, a, initial_state, final_state, workspace + s.states, nullptr, (float2*)(workspace + s.factors));
        if (rc) return rc;
        a.entry = workspace + s.states; a.exit = nullptr;
    }
    return walk<T, T, false, false, false>(device, a);
}

template <typename T> int backward(rlt_rocm_device* device, const rlt_linear_attention* p, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v, const rlt_head_view* d_output,
                                   const rlt_head_view* d_q, const rlt_head_view* d_k, const rlt_head_view* d_v, const float* initial_state, const float* d_final_state, float* d_initial_state,
                                   float* d_log_decay, int accumulate, const uint8_t* reset, const int32_t* lengths, int steps, float* workspace) {
    const int group = p->heads / p->kv_heads;
    const Scratch s = scratch_of(p, steps, true);
    const Part Q = part<T>(q, 1, p->key_dim), K = part<T>(k, group, p->key_dim), V = part<T>(v, group, p->value_dim), G = part<T>(d_output, 1, p->value_dim);
    float* const states = workspace + s.states; float* const slopes = workspace + s.slopes; float2* const factors = (float2*)(workspace + s.factors);
    int rc;
    // d_q reads the state across: values are its keys
    Walk a = walk_of(p, reset, lengths, steps);
    const bool cut = a.segments > 1;
    if (cut) {
        a.k = K; a.v = V;
        rc = d_log_decay ? segment_states<T, false, true>(device, a, initial_state, nullptr, states, slopes, factors) : segment_states<T, false, false>(device, a, initial_state, nullptr, states, nullptr, factors);
        if (rc) return rc;
    }
    a.q = G; a.k = V; a.v = K; a.with = Q; a.out = part<T, 4>(d_q, 1, p->key_dim); a.key = p->value_dim; a.value = p->key_dim; a.state_key = 1; a.state_value = p->value_dim;
    a.entry = cut ? states : initial_state; a.entry_slope = cut ? slopes : nullptr; a.d_final = d_final_state; a.partial = (double*)(workspace + s.partial);
    rc = d_log_decay ? walk<T, T, false, true, false>(device, a) : walk<T, T, false, false, false>(device, a);
    if (rc) return rc;
    if (d_log_decay) hipLaunchKernelGGL(decay_sum_kernel, dim3(p->heads), dim3(512), 0, device->stream, a.partial, p->batch, p->heads, a.segments * (p->key_dim > 64 || p->value_dim > 64 ? Layout<T, 128, true, false>::SPLIT : 1), d_log_decay, accumulate);
    // the state's gradient, from the last step to the first; d_v reads it, d_k reads it across
    Walk r = walk_of(p, reset, lengths, steps);
    r.k = Q; r.v = G; r.read_scale = 1.0f; r.added_scale = p->scale;
    if (cut && (rc = segment_states<T, true, false>(device, r, d_final_state, d_initial_state, states, nullptr, factors))) return rc;
    r.entry = cut ? states : d_final_state;
    Walk w = r;
    r.q = K;
    if (!cut) r.exit = d_initial_state;
    w.q = V; w.k = G; w.v = Q; w.key = p->value_dim; w.value = p->key_dim; w.state_key = 1; w.state_value = p->value_dim;
    const bool in_place = r.exit && r.exit == r.entry;      // d_k's walk has read the state's gradient before d_v's overwrites it: one launch after the other
    if (group == 1) {
        r.out = part<T, 4>(d_v, 1, p->value_dim); w.out = part<T, 4>(d_k, 1, p->key_dim);
        if (in_place && (rc = walk<T, T, true, false, false>(device, w))) return rc;
        return walk<T, T, true, false, false>(device, r, in_place ? nullptr : &w);
    }
    // shared keys and values: every head's share in fp32, then the sums over the heads
    const size_t tokens = (size_t)steps * p->batch;
    auto shares = [&](float* base, int width) { return Part{base, (int64_t)p->batch * p->heads * width, (int64_t)p->heads * width, width, 1, width % 4 == 0}; };
    float* const shared_v = workspace + s.shared; float* const shared_k = shared_v + padded(tokens * p->heads * p->value_dim);
    r.out = shares(shared_v, p->value_dim); w.out = shares(shared_k, p->key_dim);
    if (in_place && (rc = walk<T, float, true, false, false>(device, w))) return rc;
    if ((rc = walk<T, float, true, false, false>(device, r, in_place ? nullptr : &w))) return rc;
    const HeadSum sum_v = {shared_v, part<T, 4>(d_v, 1, p->value_dim), p->value_dim}, sum_k = {shared_k, part<T, 4>(d_k, 1, p->key_dim), p->key_dim};
    if (p->value_dim % 4 == 0 && p->key_dim % 4 == 0) hipLaunchKernelGGL((head_sum_kernel<T, 4>), dim3(2048, 2), dim3(256), 0, device->stream, sum_v, sum_k, tokens, p->batch, p->kv_heads, group);
    else hipLaunchKernelGGL((head_sum_kernel<T, 1>), dim3(2048, 2), dim3(256), 0, device->stream, sum_v, sum_k, tokens, p->batch, p->kv_heads, group);
    return rlt_launch_status(device);
}

}  // namespace

extern "C" {

size_t rlt_rocm_linear_attention_workspace_bytes(const rlt_linear_attention* layer, int steps, int backward) {
    if (!described(layer) || !supported(layer) || steps <= 0 || steps > MAX_STEPS || !launchable(layer, backward ? BACKWARD : FORWARD, false)) return 0;
    return scratch_of(layer, steps, backward != 0).total * sizeof(float);
}

int rlt_rocm_linear_attention_forward(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                      const rlt_head_view* output, const float* initial_state, float* final_state, const uint8_t* reset, const int32_t* lengths, int steps,
                                      void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && steps > 0 && given(q) && given(k) && given(v) && given(output));
    if (!supported(layer) || steps > MAX_STEPS || (!(steps == 1 && final_state) && !launchable(layer, FORWARD, false))) return RLT_E_UNSUPPORTED;
    const size_t need = rlt_rocm_linear_attention_workspace_bytes(layer, steps, 0);
    RLT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0));
    return layer->type == RLT_TYPE_F32 ? forward<float>(device, layer, q, k, v, output, initial_state, final_state, reset, lengths, steps, (float*)workspace)
                                       : forward<rlt_bf16>(device, layer, q, k, v, output, initial_state, final_state, reset, lengths, steps, (float*)workspace);
}

int rlt_rocm_linear_attention_backward(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                       const rlt_head_view* d_output, const rlt_head_view* d_q, const rlt_head_view* d_k, const rlt_head_view* d_v,
                                       const float* initial_state, const float* d_final_state, float* d_initial_state, float* d_log_decay, int accumulate,
                                       const uint8_t* reset, const int32_t* lengths, int steps, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && steps > 0 && given(q) && given(k) && given(v) && given(d_output) && given(d_q) && given(d_k) && given(d_v));
    if (!supported(layer) || steps > MAX_STEPS || !launchable(layer, BACKWARD, d_log_decay != nullptr)) return RLT_E_UNSUPPORTED;
    const size_t need = rlt_rocm_linear_attention_workspace_bytes(layer, steps, 1);
    RLT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0));
    return layer->type == RLT_TYPE_F32 ? backward<float>(device, layer, q, k, v, d_output, d_q, d_k, d_v, initial_state, d_final_state, d_initial_state, d_log_decay, accumulate, reset, lengths, steps, (float*)workspace)
                                       : backward<rlt_bf16>(device, layer, q, k, v, d_output, d_q, d_k, d_v, initial_state, d_final_state, d_initial_state, d_log_decay, accumulate, reset, lengths, steps, (float*)workspace);
}

int rlt_rocm_linear_attention_step(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                   const rlt_head_view* output, const float* state, float* next_state, const uint8_t* reset) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && given(q) && given(k) && given(v) && given(output) && state && next_state);
    if (!supported(layer)) return RLT_E_UNSUPPORTED;
    const int group = layer->heads / layer->kv_heads;
    Walk a = walk_of(layer, reset, nullptr, 1);
    a.entry = state; a.exit = next_state;
    auto views = [&](auto type) {
        typedef decltype(type) T;
        a.q = part<T>(q, 1, layer->key_dim); a.k = part<T>(k, group, layer->key_dim); a.v = part<T>(v, group, layer->value_dim); a.out = part<T, 4>(output, 1, layer->value_dim);
        return launch_step<T>(device, a);
    };
    return layer->type == RLT_TYPE_F32 ? views(0.0f) : views((rlt_bf16)0.0f);
}

}  // extern "C"
