// Short causal convolution over the steps of a sequence, each channel with its own few weights: forward, backward and single steps.
#include "selective.h"
#include <type_traits>

namespace {

constexpr int MAX_STEPS = 1 << 30, MAX_ROWS = 1 << 24, MAX_CHANNELS = 1 << 22, MIN_WIDTH = 2, MAX_WIDTH = 8;

struct Convolution {
    const float* weights; const float* biases;
    rlt_part x, out, d_out, d_x;
    const float* initial; float* final; const float* d_final; float* d_initial;
    const uint8_t* reset; const int32_t* lengths;
    float* partial;               // [groups][width + 1][channels]: weights' gradients, the bias's behind them
    int batch, channels, silu, steps, segment_steps, segments, vectors;
    unsigned groups;              // threads that share a channel: all rows and segments, or as many as leave little to add up
};

// A thread has V channels of one row and the steps of one segment; the channels of a row are side by side over the threads.
struct Place { int row, segment, channel; bool there; };
template <int V> __device__ __forceinline__ Place place_of(const Convolution& a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, pair = i / a.vectors;
    return {(int)(pair % a.batch), (int)(pair / a.batch), (int)(i - pair * a.vectors) * V, pair < a.groups};
}
template <typename T> __device__ __forceinline__ T* at(const rlt_part& p, int step, int row, int channel) { return (T*)p.data + (int64_t)step * p.step + (int64_t)row * p.row + channel; }

// how many of the inputs before step t belong to its episode, at most W - 1, were there no reset at t itself
template <int W> __device__ __forceinline__ int age_of(const Convolution& a, int t, int row) {
    int age = W - 1;
    if (a.reset && t > 0) {
#pragma unroll
        for (int k = W - 2; k > 0; k--)
            if (t - k >= 0 && a.reset[(size_t)(t - k) * a.batch + row]) age = k;
    }
    return age;
}
// window[j]: the input of step t - 1 - j
template <typename T, int W, int V> __device__ __forceinline__ void load_window(const Convolution& a, int t, int row, int channel, float (&window)[W - 1][V]) {
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        const int s = t - 1 - j;
#pragma unroll
        for (int i = 0; i < V; i++) window[j][i] = 0.0f;
        if (s >= 0) rlt_load<V>(at<T>(a.x, s, row, channel), window[j]);
        else if (a.initial) {
            const float* const from = a.initial + ((size_t)row * (W - 1) + (W - 1 + s)) * a.channels + channel;
#pragma unroll
            for (int i = 0; i < V; i++) window[j][i] = from[i];
        }
    }
}
template <int W, int V> __device__ __forceinline__ void load_weights(const Convolution& a, int channel, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
#pragma unroll
        for (int j = 0; j < W; j++) w[j][i] = a.weights[(size_t)(channel + i) * W + W - 1 - j];      // w[j]: of the input j steps back
        bias[i] = a.biases ? a.biases[channel + i] : 0.0f;
    }
}
// sum over the taps that the episode has
template <int W, int V, bool RESETS> __device__ __forceinline__ void taps(const float (&w)[W][V], const float (&bias)[V], const float (&x)[V], const float (&window)[W - 1][V], int age, float (&z)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        z[i] = bias[i];
#pragma unroll
        for (int j = W - 1; j > 0; j--) z[i] = !RESETS || age >= j ? fmaf(w[j][i], window[j - 1][i], z[i]) : z[i];
        z[i] = fmaf(w[0][i], x[i], z[i]);
    }
}
// 1 / (1 + e^-z), and what it leaves to one. bfloat16 tensors do without what the rounding of the exponent drops, |z| 2^-25 of the sigmoid, a thousandth of their own rounding at z = -64; the instructions' own
// errors are 2^-23 of it (8,192 x 4 x 2,048: forward 60 us with them, 52 without, backward 101 and 91). The fp32 sums that such steps go into, gradients of weights and biases, are off by |z| 2^-25 of the slope, which is |z| e^z far below zero: 2^-25.9 of the
// output's gradient at the most, less than the sums round (2,048 steps x 4 rows x 512 channels: d_weights 1.33e-7 off 64 bits with them and without)
template <typename T> __device__ __forceinline__ void sigmoids(float z, float& s, float& other) {
    if constexpr (sizeof(T) == sizeof(float)) rlt_sigmoids(z, s, other);
    else {
        s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
        other = 1.0f - s;
    }
}
template <typename T, int V> __device__ __forceinline__ void activate(float (&z)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        float s, other;
        sigmoids<T>(z[i], s, other);
        z[i] *= s;
    }
}
// V elements as they lie in memory
template <typename T, int V> struct Raw {
    typedef T vector __attribute__((ext_vector_type(V)));
    vector v;
    __device__ __forceinline__ void load(const T* from) { if constexpr (V == 1) v = vector(*from); else v = *reinterpret_cast<const vector*>(from); }
    __device__ __forceinline__ void unpack(float (&to)[V]) const {
#pragma unroll
        for (int i = 0; i < V; i++) to[i] = (float)v[i];
    }
};
template <int W, int V> __device__ __forceinline__ void shift(float (&window)[W - 1][V], const float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
#pragma unroll
        for (int j = W - 2; j > 0; j--) window[j][i] = window[j - 1][i];
        window[0][i] = x[i];
    }
}
template <int W, int V> __device__ __forceinline__ void store_state(float* state, int channels, int row, int channel, const float (&window)[W - 1][V], int age) {
#pragma unroll
    for (int j = 0; j < W - 1; j++)
#pragma unroll
        for (int i = 0; i < V; i++) state[((size_t)row * (W - 1) + W - 2 - j) * channels + channel + i] = age > j ? window[j][i] : 0.0f;
}

// Memory bounds it: each input once (and the window ahead of a segment again), each output once. Eight steps' inputs are on their way while those of the eight before them are worked on
// (8,192 steps x 4 rows x 2,048 channels, bfloat16: 52 us, 5.2 TB/s).
template <typename T, int W, int V, bool RESETS> __global__ __launch_bounds__(256) void forward_kernel(Convolution a) {
    constexpr int U = 8;
    const Place p = place_of<V>(a);
    if (!p.there) return;
    const int first = p.segment * a.segment_steps, end = min(first + a.segment_steps, a.steps), length = a.lengths ? min(max(a.lengths[p.row], 0), a.steps) : a.steps, live = min(end, length);
    float w[W][V], bias[V], window[W - 1][V];
    load_weights<W, V>(a, p.channel, w, bias);
    int age = W - 1;
    if (first <= length) {
        if (RESETS) age = age_of<W>(a, first, p.row);
        load_window<T, W, V>(a, first, p.row, p.channel, window);
    }
    const T* from = at<T>(a.x, first, p.row, p.channel); T* to = at<T>(a.out, first, p.row, p.channel);
    const uint8_t* flags = RESETS ? a.reset + (size_t)first * a.batch + p.row : nullptr;
    auto step = [&](const Raw<T, V>& raw, bool begins) {
        float x[V], z[V];
        raw.unpack(x);
        if (RESETS && begins) age = 0;
        taps<W, V, RESETS>(w, bias, x, window, age, z);
        if (a.silu) activate<T, V>(z);
        rlt_store<V>(to, z);
        to += a.out.step;
        shift<W, V>(window, x);
        if (RESETS) age = min(age + 1, W - 1);
    };
    Raw<T, V> next[U];
    bool begins[U];
    auto ask = [&] {
#pragma unroll
        for (int u = 0; u < U; u++) {
            next[u].load(from);
            from += a.x.step;
            if (RESETS) { begins[u] = *flags; flags += a.batch; }
        }
    };
    int t = first;
    if (t + U <= live) ask();
    for (; t + U <= live; t += U) {
        Raw<T, V> x[U];
        bool now[U];
#pragma unroll
        for (int u = 0; u < U; u++) { x[u] = next[u]; if (RESETS) now[u] = begins[u]; }
        if (t + 2 * U <= live) ask();
#pragma unroll
        for (int u = 0; u < U; u++) step(x[u], RESETS && now[u]);
    }
    for (; t < live; t++) {
        Raw<T, V> x;
        x.load(from);
        from += a.x.step;
        bool now = false;
        if (RESETS) { now = *flags; flags += a.batch; }
        step(x, now);
    }
    if (a.final && (length > first ? length <= end : length == 0 && first == 0)) store_state<W, V>(a.final, a.channels, p.row, p.channel, window, age);
    float zeros[V];
#pragma unroll
    for (int i = 0; i < V; i++) zeros[i] = 0.0f;
    for (t = max(live, first); t < end; t++, to += a.out.step) rlt_store<V>(to, zeros);
}

// The state behind the last steps alone, where it takes the initial state's place: a launch behind the one that reads it. A thread reads what it writes over before it does.
template <typename T, int W> __global__ __launch_bounds__(256) void final_state_kernel(Convolution a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(i / a.channels), channel = (int)(i - (size_t)row * a.channels);
    if (row >= a.batch) return;
    const int length = a.lengths ? min(max(a.lengths[row], 0), a.steps) : a.steps;
    int age = age_of<W>(a, length, row);
    float window[W - 1][1];
    load_window<T, W, 1>(a, length, row, channel, window);
    store_state<W, 1>(a.final, a.channels, row, channel, window, age);
}

// One walk with the steps: step t's gradient before the activation needs the inputs up to t, and is added to those of the W inputs that it read; the oldest of them is then whole and is written. A segment goes W - 1 steps beyond
// its end for the sake of its last inputs. Memory bounds it: inputs and the output's gradient in, the input's gradient out (90 us where the forward pass takes 52, 4.5 TB/s).
template <typename T, int W, int V, bool RESETS> __global__ __launch_bounds__(256) void backward_kernel(Convolution a) {
    constexpr int U = 4;
    Place p = place_of<V>(a);
    if (!p.there) return;
    float w[W][V], bias[V], d_w[W][V], d_bias[V];
    load_weights<W, V>(a, p.channel, w, bias);
#pragma unroll
    for (int i = 0; i < V; i++) {
        d_bias[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) d_w[j][i] = 0.0f;
    }
    const size_t group = ((size_t)blockIdx.x * 256 + threadIdx.x) / a.vectors, pairs = (size_t)a.batch * a.segments;
    for (size_t pair = group; pair < pairs; pair += a.groups) {
        p.row = (int)(pair % a.batch); p.segment = (int)(pair / a.batch);
        const int first = p.segment * a.segment_steps, end = min(first + a.segment_steps, a.steps), length = a.lengths ? min(max(a.lengths[p.row], 0), a.steps) : a.steps;
        const int own = min(end, length), stop = min(end + W - 1, length);      // steps whose inputs are this segment's; steps that are looked at
        float window[W - 1][V], d[W - 1][V];
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int i = 0; i < V; i++) d[j][i] = 0.0f;
        int age = W - 1;
        if (first <= length) {
            if (RESETS) age = age_of<W>(a, first, p.row);
            load_window<T, W, V>(a, first, p.row, p.channel, window);
        }
        T* const d_x0 = at<T>(a.d_x, 0, p.row, p.channel);
        auto emit = [&](int s, const float (&v)[V]) {      // the gradient of the input of step s
            if (s >= first) { if (s < own) rlt_store<V>(d_x0 + (int64_t)s * a.d_x.step, v); }
            else if (s < 0 && first == 0 && a.d_initial) {
#pragma unroll
                for (int i = 0; i < V; i++) a.d_initial[((size_t)p.row * (W - 1) + W - 1 + s) * a.channels + p.channel + i] = v[i];
            }
        };
        // INNER: a step of the segment whose oldest input is one, too
        auto step = [&](int t, const Raw<T, V>& x_raw, const Raw<T, V>& d_raw, bool begins, auto inner) {
            constexpr bool INNER = decltype(inner)::value;
            float x[V], g[V], now[V];
            x_raw.unpack(x);
            d_raw.unpack(g);
            if (RESETS && begins) age = 0;
            if (a.silu) {
                float z[V];
                taps<W, V, RESETS>(w, bias, x, window, age, z);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    float s, other;
                    sigmoids<T>(z[i], s, other);
                    g[i] *= s * fmaf(z[i], other, 1.0f);
                }
            }
            if (INNER || t < end) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    d_bias[i] += g[i];
                    d_w[0][i] = fmaf(g[i], x[i], d_w[0][i]);
#pragma unroll
                    for (int j = 1; j < W; j++) d_w[j][i] = !RESETS || age >= j ? fmaf(g[i], window[j - 1][i], d_w[j][i]) : d_w[j][i];
                }
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                now[i] = w[0][i] * g[i];
#pragma unroll
                for (int j = 1; j < W; j++) d[j - 1][i] = !RESETS || age >= j ? fmaf(w[j][i], g[i], d[j - 1][i]) : d[j - 1][i];
            }
            if (INNER) rlt_store<V>(d_x0 + (int64_t)(t - (W - 1)) * a.d_x.step, d[W - 2]);
            else emit(t - (W - 1), d[W - 2]);
            shift<W, V>(d, now);
            shift<W, V>(window, x);
            if (RESETS) age = min(age + 1, W - 1);
        };
        const T* from = at<T>(a.x, first, p.row, p.channel); const T* d_from = at<T>(a.d_out, first, p.row, p.channel);
        const uint8_t* flags = RESETS ? a.reset + (size_t)first * a.batch + p.row : nullptr;
        auto one = [&](int t) {
            Raw<T, V> x, g;
            x.load(from); g.load(d_from);
            from += a.x.step; d_from += a.d_out.step;
            bool begins = false;
            if (RESETS) { begins = *flags; flags += a.batch; }
            step(t, x, g, begins, std::false_type{});
        };
        int t = first;
        for (; t < min(first + W - 1, stop); t++) one(t);
        Raw<T, V> next_x[U], next_d[U];
        bool next_begins[U];
        auto ask = [&] {
#pragma unroll
            for (int u = 0; u < U; u++) {
                next_x[u].load(from); next_d[u].load(d_from);
                from += a.x.step; d_from += a.d_out.step;
                if (RESETS) { next_begins[u] = *flags; flags += a.batch; }
            }
        };
        if (t + U <= own) ask();
        for (; t + U <= own; t += U) {
            Raw<T, V> x[U], g[U];
            bool begins[U];
#pragma unroll
            for (int u = 0; u < U; u++) { x[u] = next_x[u]; g[u] = next_d[u]; if (RESETS) begins[u] = next_begins[u]; }
            if (t + 2 * U <= own) ask();
#pragma unroll
            for (int u = 0; u < U; u++) step(t + u, x[u], g[u], RESETS && begins[u], std::true_type{});
        }
        for (; t < stop; t++) one(t);
        // a row that ends here: the gradient of the state behind it, then what waits
        if (length >= first && length < end + W - 1 && (length > 0 || first == 0)) {
            if (a.d_final) {
#pragma unroll
                for (int j = 1; j < W; j++)
#pragma unroll
                    for (int i = 0; i < V; i++)
                        if (!RESETS || age >= j) d[j - 1][i] += a.d_final[((size_t)p.row * (W - 1) + W - 1 - j) * a.channels + p.channel + i];
            }
#pragma unroll
            for (int j = W - 1; j > 0; j--) emit(length - j, d[j - 1]);
        }
        float zeros[V];
#pragma unroll
        for (int i = 0; i < V; i++) zeros[i] = 0.0f;
        for (t = max(own, first); t < end; t++) rlt_store<V>(d_x0 + (int64_t)t * a.d_x.step, zeros);
    }
    if (a.partial) {
        float* const to = a.partial + group * (W + 1) * a.channels + p.channel;
#pragma unroll
        for (int i = 0; i < V; i++) {
#pragma unroll
            for (int j = 0; j < W; j++) to[(size_t)(W - 1 - j) * a.channels + i] = d_w[j][i];
            to[(size_t)W * a.channels + i] = d_bias[i];
        }
    }
}

// sums over rows and segments
__global__ __launch_bounds__(1024) void join_kernel(const float* __restrict__ partial, int parts, int width, int channels, float* __restrict__ d_weights, float* __restrict__ d_biases, int accumulate) {
    const int column = blockIdx.x * RLT_JOIN_COLUMNS + threadIdx.x % RLT_JOIN_COLUMNS, columns = (width + 1) * channels;
    const float s = rlt_join_column(partial, parts, columns, column, column < columns);
    if (threadIdx.x < RLT_JOIN_COLUMNS && column < columns) {
        const int tap = column / channels, channel = column - tap * channels;
        float* const to = tap < width ? (d_weights ? d_weights + (size_t)channel * width + tap : nullptr) : (d_biases ? d_biases + channel : nullptr);
        if (to) *to = accumulate ? *to + s : s;
    }
}

// A pass over the states, which are read and written once: a thread has its channels of ROWS rows, whose loads are all on their way before the first of them is worked on, and their weights once (4,096 rows x 2,048 channels,
// width 4, bfloat16: 60 us; 75 with a row to a thread).
constexpr int STEP_ROWS = 4;
template <typename T, int W, int V> __global__ __launch_bounds__(256) void step_kernel(Convolution a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, rows = i / a.vectors;
    const int row0 = (int)rows * STEP_ROWS, channel = (int)(i - rows * a.vectors) * V;
    if (rows * STEP_ROWS >= (size_t)a.batch) return;
    float window[STEP_ROWS][W - 1][V], x[STEP_ROWS][V], w[W][V], bias[V];
    bool begins[STEP_ROWS];
#pragma unroll
    for (int r = 0; r < STEP_ROWS; r++) {
        const int row = min(row0 + r, a.batch - 1);
        rlt_load<V>(at<T>(a.x, 0, row, channel), x[r]);
        load_window<T, W, V>(a, 0, row, channel, window[r]);
        begins[r] = a.reset && a.reset[row];
    }
    load_weights<W, V>(a, channel, w, bias);
#pragma unroll
    for (int r = 0; r < STEP_ROWS; r++) {
        if (row0 + r >= a.batch) break;
        float z[V];
        const int age = begins[r] ? 0 : W - 1;
        taps<W, V, true>(w, bias, x[r], window[r], age, z);
        if (a.silu) activate<T, V>(z);
        rlt_store<V>(at<T>(a.out, 0, row0 + r, channel), z);
        shift<W, V>(window[r], x[r]);
        store_state<W, V>(a.final, a.channels, row0 + r, channel, window[r], min(age + 1, W - 1));
    }
}

bool described(const rlt_causal_convolution* p) {
    return p && (p->type == RLT_TYPE_F32 || p->type == RLT_TYPE_BF16) && p->batch > 0 && p->channels > 0 && p->width > 0;
}
bool supported(const rlt_causal_convolution* p) {
    return p->width >= MIN_WIDTH && p->width <= MAX_WIDTH && p->batch <= MAX_ROWS && p->channels <= MAX_CHANNELS && (int64_t)p->batch * p->channels <= INT32_MAX;
}
bool whole(const rlt_part& p, int64_t vector, int64_t size) { return !p.data || (reinterpret_cast<uintptr_t>(p.data) % 16 == 0 && p.step % vector == 0 && p.row % vector == 0 && 16 / size == vector); }

// Segments until the chip has two threads' worth of work for every lane, of 16 steps at the least.
struct Segments { int count, steps; unsigned groups; };
Segments segments_of(const rlt_causal_convolution* p, int steps) {
    const int64_t vectors = (int64_t)p->batch * ((p->channels * (p->type == RLT_TYPE_F32 ? 4 : 2) + 15) / 16), wanted = 131072;
    int64_t count = (wanted + vectors - 1) / vectors, most = (steps + 15) / 16;
    if (count > most) count = most;
    const int per = (int)((steps + count - 1) / count);
    count = (steps + per - 1) / per;
    // backward: threads go from one row and segment to the next where there are more of them than lanes, so that what is left to add up stays small
    const int64_t pairs = p->batch * count, groups = (wanted * p->batch + vectors - 1) / vectors;
    return {(int)count, per, (unsigned)(pairs < groups ? pairs : groups)};
}
Convolution convolution_of(const rlt_causal_convolution* p, const uint8_t* reset, const int32_t* lengths, int steps) {
    const Segments g = segments_of(p, steps);
    Convolution a{};
    a.weights = p->weights; a.biases = p->biases; a.reset = reset; a.lengths = lengths;
    a.batch = p->batch; a.channels = p->channels; a.silu = p->silu; a.steps = steps; a.segment_steps = g.steps; a.segments = g.count; a.groups = (unsigned)(p->batch * g.count);
    return a;
}
enum Pass { FORWARD, BACKWARD, STEP };
template <typename T, int W, int V, int PASS> int launch_vectors(rlt_rocm_device* device, Convolution a) {
    a.vectors = a.channels / V;
    const size_t blocks = ((size_t)a.vectors * (PASS == STEP ? (a.batch + STEP_ROWS - 1) / STEP_ROWS : a.groups) + 255) / 256;
    if (blocks > UINT32_MAX / 256) return RLT_E_UNSUPPORTED;
    const dim3 grid((unsigned)blocks), block(256);
    if constexpr (PASS == STEP) hipLaunchKernelGGL((step_kernel<T, W, V>), grid, block, 0, device->stream, a);
    else if constexpr (PASS == FORWARD) {
        if (a.reset) hipLaunchKernelGGL((forward_kernel<T, W, V, true>), grid, block, 0, device->stream, a);
        else hipLaunchKernelGGL((forward_kernel<T, W, V, false>), grid, block, 0, device->stream, a);
    } else {
        if (a.reset) hipLaunchKernelGGL((backward_kernel<T, W, V, true>), grid, block, 0, device->stream, a);
        else hipLaunchKernelGGL((backward_kernel<T, W, V, false>), grid, block, 0, device->stream, a);
    }
    return rlt_launch_status(device);
}
// Vectors of 16 bytes, in the backward pass of bfloat16 of 8 bytes: what it holds for eight channels leaves a SIMD two wavefronts.
template <typename T, int W> int launch_width(rlt_rocm_device* device, const Convolution& a, Pass pass) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = a.channels % V == 0 && whole(a.x, V, sizeof(T)) && whole(a.out, V, sizeof(T)) && whole(a.d_out, V, sizeof(T)) && whole(a.d_x, V, sizeof(T));
    if (pass == FORWARD) return vectors ? launch_vectors<T, W, V, FORWARD>(device, a) : launch_vectors<T, W, 1, FORWARD>(device, a);
    if (pass == BACKWARD) return vectors ? launch_vectors<T, W, 4, BACKWARD>(device, a) : launch_vectors<T, W, 1, BACKWARD>(device, a);
    return vectors ? launch_vectors<T, W, V, STEP>(device, a) : launch_vectors<T, W, 1, STEP>(device, a);
}
template <typename F> int by_width(int width, F&& f) {
    switch (width) {
        case 2: return f(std::integral_constant<int, 2>{}); case 3: return f(std::integral_constant<int, 3>{}); case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{}); case 6: return f(std::integral_constant<int, 6>{}); case 7: return f(std::integral_constant<int, 7>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}
int launch(rlt_rocm_device* device, const rlt_causal_convolution* p, const Convolution& a, Pass pass) {
    return by_width(p->width, [&](auto w) {
        constexpr int W = decltype(w)::value;
        return p->type == RLT_TYPE_F32 ? launch_width<float, W>(device, a, pass) : launch_width<rlt_bf16, W>(device, a, pass);
    });
}
int launch_final_state(rlt_rocm_device* device, const rlt_causal_convolution* p, const Convolution& a) {
    const unsigned blocks = (unsigned)(((size_t)a.batch * a.channels + 255) / 256);
    return by_width(p->width, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (p->type == RLT_TYPE_F32) hipLaunchKernelGGL((final_state_kernel<float, W>), dim3(blocks), dim3(256), 0, device->stream, a);
        else hipLaunchKernelGGL((final_state_kernel<rlt_bf16, W>), dim3(blocks), dim3(256), 0, device->stream, a);
        return rlt_launch_status(device);
    });
}
// whether a launch has fewer than 2^32 threads also where every thread has one channel
bool launchable(const rlt_causal_convolution* p, int steps) { return (uint64_t)p->batch * p->channels * segments_of(p, steps).count <= UINT32_MAX - 255; }

}  // namespace

extern "C" {

int rlt_rocm_causal_convolution_forward(rlt_rocm_device* device, const rlt_causal_convolution* layer, const rlt_head_view* x, const rlt_head_view* output, const float* initial_state,
                                        float* final_state, const uint8_t* reset, const int32_t* lengths, int steps) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->weights && steps > 0 && rlt_given(x) && rlt_given(output));
    if (!supported(layer) || steps > MAX_STEPS || !launchable(layer, steps)) return RLT_E_UNSUPPORTED;
    Convolution a = convolution_of(layer, reset, lengths, steps);
    a.x = rlt_part_of(x); a.out = rlt_part_of(output); a.initial = initial_state;
    const bool apart = final_state && final_state == initial_state && a.segments > 1;
    a.final = apart ? nullptr : final_state;
    const int rc = launch(device, layer, a, FORWARD);
    if (rc || !apart) return rc;
    a.final = final_state;
    return launch_final_state(device, layer, a);
}

size_t rlt_rocm_causal_convolution_workspace_bytes(const rlt_causal_convolution* layer, int steps) {
    if (!described(layer) || !supported(layer) || steps <= 0 || steps > MAX_STEPS || !launchable(layer, steps) || (!layer->d_weights && !layer->d_biases)) return 0;
    return (size_t)segments_of(layer, steps).groups * (layer->width + 1) * layer->channels * sizeof(float);
}

int rlt_rocm_causal_convolution_backward(rlt_rocm_device* device, const rlt_causal_convolution* layer, const rlt_head_view* x, const rlt_head_view* d_output, const rlt_head_view* d_x,
                                         const float* initial_state, const float* d_final_state, float* d_initial_state, int accumulate, const uint8_t* reset, const int32_t* lengths, int steps,
                                         void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->weights && steps > 0 && rlt_given(x) && rlt_given(d_output) && rlt_given(d_x));
    RLT_REQUIRE(!d_initial_state || (d_initial_state != d_final_state && d_initial_state != initial_state));
    if (!supported(layer) || steps > MAX_STEPS || !launchable(layer, steps)) return RLT_E_UNSUPPORTED;
    const size_t need = rlt_rocm_causal_convolution_workspace_bytes(layer, steps);
    RLT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0));
    Convolution a = convolution_of(layer, reset, lengths, steps);
    a.x = rlt_part_of(x); a.d_out = rlt_part_of(d_output); a.d_x = rlt_part_of(d_x); a.initial = initial_state; a.d_final = d_final_state; a.d_initial = d_initial_state;
    a.partial = need ? (float*)workspace : nullptr; a.groups = segments_of(layer, steps).groups;
    const int rc = launch(device, layer, a, BACKWARD);
    if (rc || !need) return rc;
    const size_t columns = (size_t)(layer->width + 1) * layer->channels;
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((columns + RLT_JOIN_COLUMNS - 1) / RLT_JOIN_COLUMNS)), dim3(1024), 0, device->stream, (const float*)workspace, (int)a.groups, layer->width, layer->channels, layer->d_weights,
                       layer->d_biases, accumulate);
    return rlt_launch_status(device);
}

int rlt_rocm_causal_convolution_step(rlt_rocm_device* device, const rlt_causal_convolution* layer, const rlt_head_view* x, const rlt_head_view* output, const float* state, float* next_state,
                                     const uint8_t* reset) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->weights && rlt_given(x) && rlt_given(output) && state && next_state);
    if (!supported(layer)) return RLT_E_UNSUPPORTED;
    Convolution a = convolution_of(layer, reset, nullptr, 1);
    a.x = rlt_part_of(x); a.out = rlt_part_of(output); a.initial = state; a.final = next_state;
    return launch(device, layer, a, STEP);
}

}  // extern "C"
