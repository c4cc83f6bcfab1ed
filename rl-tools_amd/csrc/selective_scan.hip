// Selective scan: a few states for each channel, whose decays, inputs and readings depend on the step; forward, backward and single steps.
#include "selective.h"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

constexpr int MAX_STEPS = 1 << 30, MAX_STATES = 32, MAX_CHANNELS = 1 << 20;      // channels: of all heads, whose gradients are summed in one launch
constexpr int64_t MAX_STRIDE = 1 << 27;      // elements between steps: three of them and a row of channels are an offset of 32 bits
constexpr int WAVES = 4, LANES = 64 * WAVES, TILE = 16 * WAVES;      // channels of a workgroup: four lanes share one, each with a quarter of its states
constexpr float NO_DELTA = -__builtin_huge_valf();      // what a delta of nothing comes of: a step that is not there leaves the state as it is
constexpr float LOG2_E = 1.44269504088896341f, LN_2 = 0.69314718055994531f;

// steps that a lane looks at together, and behind which the forward pass leaves the states for the backward pass; NPT states to a lane
template <int NPT> constexpr int CHUNK = NPT == 8 ? 8 : 16;
static int per_lane(int states) { return states <= 8 ? 2 : states <= 16 ? 4 : 8; }
static int chunk_of(int states) { return states <= 16 ? 16 : 8; }

struct Scan {
    const float* log_rates; const float* skip; const float* delta_biases;
    rlt_part x, delta, b, c, gate, out, d_out, d_x, d_delta, d_b, d_c, d_gate;
    const float* entry; float* exit;         // states (backward: their gradients) before the first step walked and behind the last: [pairs][channels][states], or where there are segments [pairs][segments][channels][4 NPT]
    float* sums;                  // of delta over a segment, [pairs][segments][channels]; below zero: the segment holds a reset, nothing passes it
    float* checkpoints;           // [pairs][chunks][channels][4 NPT]: states before each chunk
    float* d_shared;              // d_b, then d_c: [tiles][pairs][steps][4 NPT]
    float* d_rates; float* d_skips; float* d_biases;      // [row groups x segments][heads][channels][4 NPT] and [...][channels]
    const uint8_t* reset; const int32_t* lengths;
    int batch, heads, channels, states, steps, segments, segment_steps, tiles, chunks, row_groups;
    int entry_padded;             // entry is the segments'
};

template <typename T> __device__ __forceinline__ T* at(const rlt_part& p, int step, int row, int head) { return (T*)p.data + (int64_t)step * p.step + (int64_t)row * p.row + (int64_t)head * p.head; }

// The parts of a launch's arguments as they are needed, from where the launch left them: strides that a kernel needs once a row would otherwise hold scalar registers, of which there are too few, from its start to its end.
struct Arguments {
    const __attribute__((address_space(4))) char* at;
    __device__ __forceinline__ Arguments() {
        at = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(at));
    }
    __device__ __forceinline__ rlt_part part(size_t offset) const {
        const auto* const v = (const __attribute__((address_space(4))) int64_t*)(at + offset);
        return {(void*)v[0], v[1], v[2], v[3]};
    }
};
#define SCAN_PART(arguments, name) (arguments).part(offsetof(Scan, name))

// ---- exchanges between the four lanes of a channel
template <int CTRL> __device__ __forceinline__ float lanes(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)); }
template <int J> __device__ __forceinline__ float from_lane(float v) { return lanes<J * 0x55>(v); }
// lane j receives the sum over its channel's lanes of v[j]
__device__ __forceinline__ float sum_to_lane(const float (&v)[4], bool odd, bool upper) {
    const float a = (odd ? v[1] : v[0]) + lanes<0xB1>(odd ? v[0] : v[1]), b = (odd ? v[3] : v[2]) + lanes<0xB1>(odd ? v[2] : v[3]);
    return (upper ? b : a) + lanes<0x4E>(upper ? a : b);
}
__device__ __forceinline__ float sum_of_lanes(float v) {
    v += lanes<0xB1>(v);
    return v + lanes<0x4E>(v);
}
template <int FIRST, int LAST, typename F> __device__ __forceinline__ void each(F&& f) {
    if constexpr (FIRST < LAST) { f(std::integral_constant<int, FIRST>{}); each<FIRST + 1, LAST>(f); }
}
// v in the lanes of quad J of each row of sixteen, `old` in the others
template <int J> __device__ __forceinline__ float into_quad(float old, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), 0xE4, 0xF, 1 << J, false));
}
__device__ __forceinline__ float add_halves(float a, float b) {      // lanes 0 to 31: a's sum over both halves of the wavefront, the others: b's
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
}
__device__ __forceinline__ float add_rows(float a, float b) {        // even rows of sixteen lanes: a's sum over both of a half, odd rows: b's
    const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
}
// Sums over the sixteen channels of a wavefront. A lane ends up with those of NPT / 4 of its states (of one where NPT < 4): state k + (NPT / 4) * (lane bit 4) + (NPT / 2) * (lane bit 5) of the lane's NPT.
template <int NPT> __device__ __forceinline__ void sum_channels(const float (&v)[NPT], float (&s)[NPT > 4 ? NPT / 4 : 1]) {
    if constexpr (NPT == 2) {
        const float a = add_halves(v[0], v[1]);
        s[0] = add_rows(a, a);
    } else {
        float h[NPT / 2];
#pragma unroll
        for (int i = 0; i < NPT / 2; i++) h[i] = add_halves(v[i], v[i + NPT / 2]);
#pragma unroll
        for (int i = 0; i < NPT / 4; i++) s[i] = add_rows(h[i], h[i + NPT / 4]);
    }
#pragma unroll
    for (int i = 0; i < (NPT > 4 ? NPT / 4 : 1); i++) {
        s[i] += lanes<0x124>(s[i]);      // four and eight lanes round the row
        s[i] += lanes<0x128>(s[i]);
    }
}

// The elements' own functions. fp32 tensors take what the rounding of an exponent drops along (rlt_exp_negative) and a step of Newton's method behind a reciprocal; bfloat16 ones do without: delta is off by |raw| 2^-25 of itself, a thousandth
// of what the rounding of raw leaves (a prompt of 16,384 steps x 4,096 channels: 530 us, with them 563; 8,192 x 2 x 2,048 forward and backward 905, 951). What is fp32 there too, states and the parameters' gradients, stays as close to 64 bits as with
// fp32 tensors, whose sums and decays round by more (2,048 steps x 2 rows x 512 channels x 16 states: final state 1.3e-7 off, with them 1.1e-7, fp32 tensors 1.3e-7; d_log_rates 2.8e-7, 2.6e-7, 2.8e-7); only steps of far below e^-10 are off by more, 1e-6
// of themselves at raw = -32.
template <typename T> __device__ __forceinline__ float exp_negative(float t) { return sizeof(T) == sizeof(float) ? rlt_exp_negative(t) : __builtin_amdgcn_exp2f(t * LOG2_E); }
template <typename T> __device__ __forceinline__ float reciprocal(float d) { return sizeof(T) == sizeof(float) ? rlt_reciprocal(d) : __builtin_amdgcn_rcpf(d); }
// log(1 + e^v), and e = e^-|v|. With u = 1 + e as it is rounded, log(1 + e) = log(u) + (e - (u - 1)), whose last part is exact and all there is of it far below zero; the instruction's logarithm to base 2 is within
// 1.2e-7 of itself down to u's last bit (measured on all u in [1, 2)).
template <typename T> __device__ __forceinline__ float softplus(float v, float& e) {
    e = exp_negative<T>(-fabsf(v));
    const float u = 1.0f + e;
    return fmaxf(v, 0.0f) + fmaf(__builtin_amdgcn_logf(u), LN_2, e - (u - 1.0f));
}
// z / (1 + e^-z), and (PASSED) d times its slope
template <typename T> __device__ __forceinline__ float gate_factor(float z) {
    if constexpr (sizeof(T) == sizeof(float)) {
        float one, other;
        rlt_sigmoids(z, one, other);
        return z * one;
    } else return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -LOG2_E));
}
template <typename T> __device__ __forceinline__ float gate_factor(float z, float d, float& passed) {
    float one, other;
    if constexpr (sizeof(T) == sizeof(float)) rlt_sigmoids(z, one, other);
    else { one = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -LOG2_E)); other = 1.0f - one; }
    passed = d * one * fmaf(z, other, 1.0f);
    return z * one;
}

// ---- what a workgroup walks over
struct Place { int tile, head, row, segment, first, end, length, live; };      // steps [first, end) of the segment; the row's steps; end or length
__device__ __forceinline__ Place place_of(const Scan& a, unsigned item, int row_count) {
    Place p;
    p.tile = item % a.tiles; item /= a.tiles;
    p.head = item % a.heads; item /= a.heads;
    p.segment = item / row_count; p.row = item - p.segment * row_count;
    p.first = p.segment * a.segment_steps; p.end = min(p.first + a.segment_steps, a.steps);
    return p;
}
__device__ __forceinline__ void set_row(const Scan& a, Place& p, int row) {
    p.row = row;
    p.length = a.lengths ? min(max(a.lengths[row], 0), a.steps) : a.steps;
    p.live = min(p.end, p.length);
}
__device__ __forceinline__ int pair_of(const Scan& a, const Place& p) { return p.row * a.heads + p.head; }
__device__ __forceinline__ bool bit(unsigned mask, int i) {
    mask = __builtin_amdgcn_readfirstlane(mask);
    asm volatile("" : "+s"(mask));      // looked at where it is needed: sixteen answers held from a walk forward to the one back are 32 scalar registers
    return mask >> i & 1;
}
// What a chunk needs is asked for without a branch and without looking at it, so that all of it is under way at once and nothing waits before the chunk is worked on: what is not there is read from where something is, and taken out then.
// WHOLE: all of the chunk's steps are there, which is known of every chunk but a row's last.
// Resets: a lane holds step t + lane's; bit s of the answer: step t + s forgets its state.
template <int K> struct Resets {
    uint8_t own;
    template <bool WHOLE> __device__ __forceinline__ void ask(const Scan& a, const Place& p, int t) {
        own = 0;
        const int step = t + (int)(threadIdx.x & (K - 1));
        if (a.reset) own = a.reset[(size_t)(WHOLE ? step : min(step, p.live - 1)) * a.batch + p.row];
    }
    __device__ __forceinline__ unsigned get(const Place& p, int t) const {
        const int s = threadIdx.x & 63;
        return (unsigned)__ballot(s < K && t + s < p.live && own);
    }
};

// b and c of a chunk, zero beyond the row's length and the layer's states; a thread holds its elements while the chunk before is worked on
template <typename T, int NPT, int K = CHUNK<NPT>> struct Shared {
    static constexpr int N = 4 * NPT, PER = (K * N + LANES - 1) / LANES;
    T b[PER], c[PER];
    template <bool WHOLE, bool B, bool C> __device__ __forceinline__ void ask(const Scan& a, const Place& p, int t) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            int e = threadIdx.x + j * LANES;
            asm volatile("" : "+v"(e));      // addresses are worked out for each chunk rather than held from one to the next
            const int step = WHOLE ? t + e / N : min(t + e / N, p.live - 1), n = min(e % N, a.states - 1);
            if (K * N % LANES && e >= K * N) continue;
            if (B) b[j] = at<T>(a.b, step, p.row, p.head)[n];
            if (C) c[j] = at<T>(a.c, step, p.row, p.head)[n];
        }
    }
    template <bool WHOLE, bool B, bool C> __device__ __forceinline__ void put(const Scan& a, const Place& p, int t, float (*to)[K * N]) const {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int e = threadIdx.x + j * LANES;
            const bool there = (WHOLE || t + e / N < p.live) && e % N < a.states;
            if (K * N % LANES && e >= K * N) continue;
            if (B) to[0][e] = there ? (float)b[j] : 0.0f;
            if (C) to[1][e] = there ? (float)c[j] : 0.0f;
        }
    }
    __device__ __forceinline__ void cut(const Place& p, int t) {
#pragma unroll
        for (int j = 0; j < PER; j++) if (t + (int)(threadIdx.x + j * LANES) / N >= p.live) b[j] = c[j] = (T)0.0f;
    }
};
template <int NPT> __device__ __forceinline__ void read(const float* from, float (&to)[NPT]) {
    typedef float vector __attribute__((ext_vector_type(NPT < 4 ? NPT : 4)));
#pragma unroll
    for (int i = 0; i < NPT; i += NPT < 4 ? NPT : 4) {
        const vector v = *reinterpret_cast<const vector*>(from + i);
#pragma unroll
        for (int j = 0; j < (NPT < 4 ? NPT : 4); j++) to[i + j] = v[j];
    }
}
template <int NPT> __device__ __forceinline__ void read_global(const __attribute__((address_space(1))) char* from, float (&to)[NPT]) {
    typedef float vector __attribute__((ext_vector_type(NPT < 4 ? NPT : 4)));
#pragma unroll
    for (int i = 0; i < NPT; i += NPT < 4 ? NPT : 4) {
        const vector v = *(const __attribute__((address_space(1))) vector*)(from + i * sizeof(float));
#pragma unroll
        for (int j = 0; j < (NPT < 4 ? NPT : 4); j++) to[i + j] = v[j];
    }
}
template <int NPT> __device__ __forceinline__ void write(float* to, const float (&from)[NPT]) {
    typedef float vector __attribute__((ext_vector_type(NPT < 4 ? NPT : 4)));
#pragma unroll
    for (int i = 0; i < NPT; i += NPT < 4 ? NPT : 4) {
        vector v;
#pragma unroll
        for (int j = 0; j < (NPT < 4 ? NPT : 4); j++) v[j] = from[i + j];
        *reinterpret_cast<vector*>(to + i) = v;
    }
}
// A tensor of channels as a wavefront reads and writes it: lane l has the element of its channel in step t + 4 i + l % 4, at an address that all lanes share and an offset of its own, of 32 bits (MAX_STRIDE).
#define GLOBAL __attribute__((address_space(1)))
template <typename T> struct Lanes {
    GLOBAL char* base; int stride; unsigned offset;      // of step 0; bytes to the next step; a lane's own
    __device__ __forceinline__ Lanes(const rlt_part& part, const Place& p, int channel) {
        stride = (int)(part.step * (int64_t)sizeof(T));
        const int lowest = stride < 0 ? 3 * stride : 0;      // steps that go back in memory: from the last of four on
        base = (GLOBAL char*)part.data + ((int64_t)p.row * part.row + (int64_t)p.head * part.head) * (int64_t)sizeof(T) + lowest;
        offset = (unsigned)((int)(threadIdx.x & 3) * stride - lowest) + (unsigned)channel * (unsigned)sizeof(T);
    }
    template <bool WHOLE, int OWN> __device__ __forceinline__ void ask(int t, int live, T (&v)[OWN]) const {
        const GLOBAL char* from = base + (int64_t)t * stride;
        if (WHOLE || t + 4 * OWN <= live) {
#pragma unroll
            for (int i = 0; i < OWN; i++) { v[i] = *(const GLOBAL T*)(from + offset); from += 4 * (int64_t)stride; }
        } else {
            const int last = live - 1 - t, last_four = last & ~3;      // lanes beyond the last step read the last one's
            const unsigned cut = offset - (unsigned)(max(last_four + (int)(threadIdx.x & 3) - last, 0) * stride);
#pragma unroll
            for (int i = 0; i < OWN; i++) v[i] = *(const GLOBAL T*)(from + (int64_t)min(4 * i, last_four) * stride + (4 * i < last_four ? offset : cut));
        }
    }
    __device__ __forceinline__ void put(int t, float v) const { *(GLOBAL T*)(base + (int64_t)t * stride + offset) = (T)v; }      // t: a multiple of four steps into a chunk
};
// a channel's states in the caller's memory: a lane's together, from any element on, but for what is left to the last lane that has any
template <int NPT> __device__ __forceinline__ void load_states(const float* from, int n0, int states, float (&h)[NPT]) {
    constexpr int V = NPT < 4 ? NPT : 4;
    typedef float vector __attribute__((ext_vector_type(V), aligned(4)));
    if (n0 + NPT <= states) {
#pragma unroll
        for (int n = 0; n < NPT; n += V) {
            const vector v = *reinterpret_cast<const vector*>(from + n0 + n);
#pragma unroll
            for (int i = 0; i < V; i++) h[n + i] = v[i];
        }
    } else {
#pragma unroll
        for (int n = 0; n < NPT; n++) h[n] = n0 + n < states ? from[n0 + n] : 0.0f;
    }
}
template <int NPT> __device__ __forceinline__ void store_states(float* to, int n0, int states, const float (&h)[NPT]) {
    constexpr int V = NPT < 4 ? NPT : 4;
    typedef float vector __attribute__((ext_vector_type(V), aligned(4)));
    if (n0 + NPT <= states) {
#pragma unroll
        for (int n = 0; n < NPT; n += V) {
            vector v;
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = h[n + i];
            *reinterpret_cast<vector*>(to + n0 + n) = v;
        }
    } else {
#pragma unroll
        for (int n = 0; n < NPT; n++) if (n0 + n < states) to[n0 + n] = h[n];
    }
}
// exp(log_rate), 1e30 at the most: a delta of zero, of a step that is not there, decays nothing then, whatever the rate (infinity times zero would be no number)
__device__ __forceinline__ float rate_of(float log_rate) {
    const float r = expf(log_rate);
    return r > 1e30f ? 1e30f : r;
}
// logarithms of the decays to base 2 for a delta of one; nothing where there is no state
template <int NPT> __device__ __forceinline__ void load_rates(const Scan& a, int head, int channel, int n0, float (&rate)[NPT]) {
    const float* const from = a.log_rates + ((size_t)head * a.channels + channel) * a.states;
#pragma unroll
    for (int n = 0; n < NPT; n++) rate[n] = n0 + n < a.states ? -rate_of(from[n0 + n]) * LOG2_E : 0.0f;
}

// Forward over a segment. STATES: only what the segment adds to the state, for states that segments start from. The vector units bound it, 83 % busy with four wavefronts to a SIMD (16,384 steps x 4,096 channels x 16 states, bfloat16: 350 us,
// 3.1e12 steps of a state a second; STATES 237, 78 % busy).
template <typename T, int NPT, bool STATES> __global__ __launch_bounds__(LANES) void forward_kernel(Scan a) {
    constexpr int K = CHUNK<NPT>, OWN = K / 4, N = 4 * NPT;
    __shared__ float shared[2][2][K * N];
    Place p = place_of(a, blockIdx.x, a.batch);
    set_row(a, p, p.row);
    const int lane = threadIdx.x & 63, nq = lane & 3, n0 = nq * NPT, own_channel = p.tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1);
    const bool there = own_channel < a.channels, all_there = (p.tile + 1) * TILE <= a.channels, gated = a.gate.data != nullptr, odd = nq & 1, upper = nq & 2;
    const size_t pair = pair_of(a, p), at_channel = (size_t)p.head * a.channels + channel;
    T x[OWN], raw[OWN], gate[OWN];
    Resets<K> resets;
    Shared<T, NPT, K> next;
    const Arguments arguments;
    const Lanes<T> x_lanes(SCAN_PART(arguments, x), p, channel), delta_lanes(SCAN_PART(arguments, delta), p, channel), gate_lanes(SCAN_PART(arguments, gate), p, channel), out_lanes(SCAN_PART(arguments, out), p, channel);
    auto ask_chunk = [&](int t) {
        x_lanes.template ask<false>(t, p.live, x);
        delta_lanes.template ask<false>(t, p.live, raw);
        if (!STATES && gated) gate_lanes.template ask<false>(t, p.live, gate);
        next.template ask<false, true, !STATES>(a, p, t);
        resets.template ask<false>(a, p, t);
    };
    if (p.first < p.live) ask_chunk(p.first);
    float rate[NPT], h[NPT];
    if (STATES || !a.entry) {
#pragma unroll
        for (int n = 0; n < NPT; n++) h[n] = 0.0f;
    } else if (a.entry_padded) read<NPT>(a.entry + ((pair * a.segments + p.segment) * a.channels + channel) * N + n0, h);
    else load_states<NPT>(a.entry + (pair * a.channels + channel) * a.states, n0, a.states, h);
    const float bias = a.delta_biases ? a.delta_biases[at_channel] : 0.0f, skip = a.skip ? a.skip[at_channel] : 0.0f;
    load_rates<NPT>(a, p.head, channel, n0, rate);
    float sum = 0.0f;
    bool forgotten = false;

    int turn = 0;
    for (int t = p.first; t < p.live; t += K, turn ^= 1) {
        float xs[OWN], delta[OWN], added[OWN], gates[OWN];
        if (!all_there || t + K > p.live) {
#pragma unroll
            for (int i = 0; i < OWN; i++) if (!there || t + 4 * i + nq >= p.live) { x[i] = gate[i] = (T)0.0f; raw[i] = (T)NO_DELTA; }
        }
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            float e;
            xs[i] = (float)x[i];
            delta[i] = softplus<T>((float)raw[i] + bias, e);
            added[i] = delta[i] * xs[i];
            if (!STATES) gates[i] = gated ? (float)gate[i] : 0.0f;
        }
        const unsigned forget = resets.get(p, t);
        next.template put<false, true, !STATES>(a, p, t, shared[turn]);
        if (t + K < p.live) ask_chunk(t + K);
        rlt_lds_barrier();
        const float* const bs = shared[turn][0] + n0; const float* const cs = shared[turn][1] + n0;
        if (!STATES && a.checkpoints && there) write<NPT>(a.checkpoints + ((pair * a.chunks + t / K) * a.channels + channel) * N + n0, h);
        float y[OWN];
        auto walk = [&](auto with_resets, auto whole) {
#pragma unroll
            for (int i = 0; i < OWN; i++) {
                if (!decltype(whole)::value && t + 4 * i >= p.live) { y[i] = 0.0f; continue; }
                float part[4];
                auto step = [&](auto which) {
                    constexpr int j = decltype(which)::value;
                    const float d = from_lane<j>(delta[i]), u = from_lane<j>(added[i]);
                    float b[NPT], c[NPT];
                    read<NPT>(bs + (4 * i + j) * N, b);
                    if (!STATES) read<NPT>(cs + (4 * i + j) * N, c);
                    if (decltype(with_resets)::value && (forget >> (4 * i + j) & 1)) {
#pragma unroll
                        for (int n = 0; n < NPT; n++) h[n] = 0.0f;
                        if (STATES) forgotten = true;
                    }
                    part[j] = 0.0f;
#pragma unroll
                    for (int n = 0; n < NPT; n++) {
                        h[n] = fmaf(__builtin_amdgcn_exp2f(d * rate[n]), h[n], u * b[n]);
                        if (!STATES) part[j] = fmaf(c[n], h[n], part[j]);
                    }
                };
                step(std::integral_constant<int, 0>{}); step(std::integral_constant<int, 1>{}); step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 3>{});
                if (!STATES) y[i] = sum_to_lane(part, odd, upper);
                else sum += delta[i];
            }
        };
        if (t + K > p.live) walk(std::true_type{}, std::false_type{});
        else if (forget) walk(std::true_type{}, std::true_type{});
        else walk(std::false_type{}, std::true_type{});
        if (!STATES) {
#pragma unroll
            for (int i = 0; i < OWN; i++) {
                const int s = t + 4 * i + nq;
                float v = fmaf(skip, xs[i], y[i]);
                if (gated) v *= gate_factor<T>(gates[i]);
                if (there && s < p.end) out_lanes.put(t + 4 * i, s < p.live ? v : 0.0f);      // (nothing read times a state that is infinite is no zero)
            }
        }
    }
    if constexpr (STATES) {
        if (!there) return;
        write<NPT>(a.exit + ((pair * a.segments + p.segment) * a.channels + channel) * N + n0, h);
        sum = sum_of_lanes(sum);
        if (nq == 0) a.sums[(pair * a.segments + p.segment) * a.channels + channel] = forgotten ? -1.0f : sum;
    } else {
        if (!there) return;
        if (a.exit && p.segment == a.segments - 1) store_states<NPT>(a.exit + (pair * a.channels + channel) * a.states, n0, a.states, h);
        // steps behind the last chunk that holds any of the row's
        const int walked = p.live > p.first ? p.first + (p.live - p.first + K - 1) / K * K : p.first;
        for (int s = walked; s + nq < p.end; s += 4) out_lanes.put(s, 0.0f);
    }
}

// Forward over sequences of K steps at most, four or eight: a workgroup goes from one row to the next, whose inputs and state are on their way while it works (8 steps x 4,096 rows x 1,024 channels, bfloat16: 240 us, a workgroup for each row 458;
// one step x 4,096 rows x 256 channels 40 and 54; two rows on their way: no faster).
template <typename T, int NPT, int K> __global__ __launch_bounds__(LANES) void short_forward_kernel(Scan a) {
    constexpr int OWN = K / 4, N = 4 * NPT;
    __shared__ float shared[2][2][K * N];
    Place p = place_of(a, blockIdx.x, a.row_groups);
    const int group = p.row, nq = threadIdx.x & 3, n0 = nq * NPT, own_channel = p.tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1);
    const bool there = own_channel < a.channels, gated = a.gate.data != nullptr, odd = nq & 1, upper = nq & 2;
    const size_t at_channel = (size_t)p.head * a.channels + channel;
    T x[OWN], raw[OWN], gate[OWN];
    Resets<K> resets;
    Shared<T, NPT, K> next;
    float entry[NPT];
    int live;
    auto ask = [&](int row) {
        const Arguments arguments;
        set_row(a, p, row);
        live = p.live;
        p.live = max(live, 1);      // (a row without steps reads its first one all the same, and looks at none)
        const Lanes<T> x_lanes(SCAN_PART(arguments, x), p, channel), delta_lanes(SCAN_PART(arguments, delta), p, channel), gate_lanes(SCAN_PART(arguments, gate), p, channel);
        x_lanes.template ask<false>(0, p.live, x);
        delta_lanes.template ask<false>(0, p.live, raw);
        if (gated) gate_lanes.template ask<false>(0, p.live, gate);
        next.template ask<false, true, true>(a, p, 0);
        resets.template ask<false>(a, p, 0);
        if (a.entry) load_states<NPT>(a.entry + ((size_t)pair_of(a, p) * a.channels + channel) * a.states, n0, a.states, entry);
        p.live = live;
    };
#pragma unroll
    for (int n = 0; n < NPT; n++) entry[n] = 0.0f;
    ask(group);
    const float bias = a.delta_biases ? a.delta_biases[at_channel] : 0.0f, skip = a.skip ? a.skip[at_channel] : 0.0f;
    float rate[NPT];
    load_rates<NPT>(a, p.head, channel, n0, rate);
    int turn = 0;
    for (int row = group; row < a.batch; row += a.row_groups, turn ^= 1) {
        const size_t pair = (size_t)row * a.heads + p.head;
        const int steps = live;
        float h[NPT], xs[OWN], delta[OWN], added[OWN], z[OWN];
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const bool whole = there && 4 * i + nq < steps;
            float e;
            xs[i] = whole ? (float)x[i] : 0.0f;
            delta[i] = softplus<T>(whole ? (float)raw[i] + bias : NO_DELTA, e);
            added[i] = delta[i] * xs[i];
            z[i] = gated && whole ? (float)gate[i] : 0.0f;
        }
        const unsigned forget = resets.get(p, 0);
        next.template put<false, true, true>(a, p, 0, shared[turn]);
#pragma unroll
        for (int n = 0; n < NPT; n++) h[n] = entry[n];
        const Arguments arguments;
        const Lanes<T> out_lanes(SCAN_PART(arguments, out), p, channel);
        ask(min(row + a.row_groups, a.batch - 1));
        rlt_lds_barrier();
        if (a.checkpoints && there && steps > 0) write<NPT>(a.checkpoints + (pair * a.channels + channel) * N + n0, h);
        float part[OWN][4];
        each<0, K>([&](auto which) {
            constexpr int j = decltype(which)::value;
            part[j / 4][j % 4] = 0.0f;
            if (j < steps) {
                const float d = from_lane<j % 4>(delta[j / 4]), u = from_lane<j % 4>(added[j / 4]);
                float b[NPT], c[NPT];
                read<NPT>(shared[turn][0] + n0 + j * N, b);
                read<NPT>(shared[turn][1] + n0 + j * N, c);
                const bool begins = forget >> j & 1;
#pragma unroll
                for (int n = 0; n < NPT; n++) {
                    h[n] = fmaf(__builtin_amdgcn_exp2f(d * rate[n]), begins ? 0.0f : h[n], u * b[n]);
                    part[j / 4][j % 4] = fmaf(c[n], h[n], part[j / 4][j % 4]);
                }
            }
        });
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            float v = fmaf(skip, xs[i], sum_to_lane(part[i], odd, upper));
            if (gated) v *= gate_factor<T>(z[i]);
            if (there && 4 * i + nq < a.steps) out_lanes.put(4 * i, v);
        }
        if (there && a.exit) store_states<NPT>(a.exit + (pair * a.channels + channel) * a.states, n0, a.states, h);
    }
}

// States that the segments start from, out of what each of them adds: element by element along the segments (REVERSE: from the last). locals become the entries.
template <bool REVERSE> __global__ __launch_bounds__(256) void join_segments_kernel(Scan a, const float* __restrict__ initial, float* __restrict__ locals, int padded) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, per_pair = (size_t)a.channels * padded, pair = i / per_pair;
    if (pair >= (size_t)a.batch * a.heads) return;
    const int e = (int)(i - pair * per_pair), channel = e / padded, n = e - channel * padded;
    const bool there = n < a.states;
    const size_t at_channel = (pair % a.heads) * a.channels + channel;
    const float rate = there ? -rate_of(a.log_rates[at_channel * a.states + n]) * LOG2_E : 0.0f;
    float carry = initial && there ? initial[(pair * a.channels + channel) * a.states + n] : 0.0f;
    constexpr int AHEAD = 8;      // segments whose shares are asked for before the first of them is used
    for (int k0 = 0; k0 < a.segments; k0 += AHEAD) {
        float local[AHEAD], sum[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int k = min(k0 + j, a.segments - 2), s = REVERSE ? a.segments - 1 - k : k;      // (the last segment adds to nothing)
            local[j] = locals[(pair * a.segments + s) * per_pair + e];
            sum[j] = a.sums[(pair * a.segments + s) * a.channels + channel];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            if (k0 + j >= a.segments) break;
            const int s = REVERSE ? a.segments - 1 - (k0 + j) : k0 + j;
            locals[(pair * a.segments + s) * per_pair + e] = carry;
            carry = sum[j] < 0.0f ? local[j] : fmaf(__builtin_amdgcn_exp2f(sum[j] * rate), carry, local[j]);
        }
    }
}

// Backward over a segment: from the last chunk to the first, the chunk's states again from its checkpoint, then its steps from the last to the first with the state's gradient G:
//     G_t = c_t g_t + a_{t+1} G_{t+1},   g = d_output times the gate's factor;   d_c = sum over channels of g h,   d_b = sum over channels of delta x G,
//     d_x = delta (G . b) + skip g,   d_delta = x (G . b) + rates . q,   d_rates += delta q   with q = G a h_{t-1}.
// The vector units bound it, 78 % busy with two wavefronts to a SIMD, whose registers hold a chunk's states and decays (8,192 steps x 2 rows x 2,048 channels x 16 states, bfloat16: 510 to 543 us, 1.0e12 steps of a state a second). What a row or a
// chunk needs once goes to scratch memory, 12 to 68 bytes a lane with more than eight states; the steps read none of it. Steps that fill up a row's last chunk are taken out by selection: a branch around each sends a chunk's states to scratch memory
// (944 bytes a lane, 3,455 us for both passes where they take 899).
template <typename T, int NPT, bool ONE_TILE> __global__ __launch_bounds__(LANES, 2) void backward_kernel(Scan a) {
    constexpr int K = CHUNK<NPT>, OWN = K / 4, N = 4 * NPT, KEPT = NPT > 4 ? NPT / 4 : 1, PER = (K * N + LANES - 1) / LANES;
    __shared__ float shared[2][2][K * N];
    __shared__ float slabs[2][WAVES][2][K * N];
    Place p = place_of(a, blockIdx.x, a.row_groups);
    const int group = p.row, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nq = lane & 3, quad = lane >> 2 & 3, n0 = nq * NPT, own_channel = p.tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1);
    const int kept_state = n0 + (NPT >= 4 ? (lane >> 4 & 1) * (NPT / 4) : 0) + (lane >> 5) * (NPT / 2);      // the first state whose sums over channels this lane is left with
    const bool there = own_channel < a.channels, all_there = (p.tile + 1) * TILE <= a.channels, odd = nq & 1, upper = nq & 2;
    const size_t at_channel = (size_t)p.head * a.channels + channel;
    float rate[NPT], d_rate[NPT];
    load_rates<NPT>(a, p.head, channel, n0, rate);
#pragma unroll
    for (int n = 0; n < NPT; n++) d_rate[n] = 0.0f;
    const float bias = a.delta_biases ? a.delta_biases[at_channel] : 0.0f, skip = a.skip ? a.skip[at_channel] : 0.0f;
    float d_skip = 0.0f, d_bias = 0.0f;
    const bool gated = a.gate.data != nullptr;
    const unsigned at_checkpoint = (unsigned)(channel * N + n0) * sizeof(float);
    int turn = 0;
    for (int row = group; row < a.batch; row += a.row_groups) {
        set_row(a, p, row);
        const size_t pair = pair_of(a, p);
        float carry[NPT];
        if (!a.entry) {
#pragma unroll
            for (int n = 0; n < NPT; n++) carry[n] = 0.0f;
        } else if (a.entry_padded) read<NPT>(a.entry + ((pair * a.segments + p.segment) * a.channels + channel) * N + n0, carry);
        else load_states<NPT>(a.entry + (pair * a.channels + channel) * a.states, n0, a.states, carry);
        const Arguments arguments;
        const Lanes<T> x_lanes(SCAN_PART(arguments, x), p, channel), delta_lanes(SCAN_PART(arguments, delta), p, channel), gate_lanes(SCAN_PART(arguments, gate), p, channel), d_out_lanes(SCAN_PART(arguments, d_out), p, channel),
            d_x_lanes(SCAN_PART(arguments, d_x), p, channel), d_delta_lanes(SCAN_PART(arguments, d_delta), p, channel), d_gate_lanes(SCAN_PART(arguments, d_gate), p, channel);
        GLOBAL float* const d_shared = ONE_TILE ? nullptr : (GLOBAL float*)a.d_shared + ((size_t)p.tile * 2 * a.batch * a.heads + pair) * a.steps * N;
        auto store_shared = [&](int t, int e, float d_b, float d_c) {      // of step t + e / N
            if constexpr (ONE_TILE) {
                if (e % N < a.states) {
                    at<T>(a.d_b, t + e / N, p.row, p.head)[e % N] = (T)d_b;
                    at<T>(a.d_c, t + e / N, p.row, p.head)[e % N] = (T)d_c;
                }
            } else {
                GLOBAL float* const to = d_shared + (size_t)t * N;
                to[e] = d_b;
                (to + (size_t)a.batch * a.heads * a.steps * N)[e] = d_c;
            }
        };
        const int chunks = p.live > p.first ? (p.live - p.first + K - 1) / K : 0;
        // steps behind the last chunk that holds any of the row's
        for (int t = p.first + chunks * K; t < p.end; t += K) {
#pragma unroll 1
            for (int i = 0; i < OWN; i++)
                if (there && t + 4 * i + nq < p.end) {
                    d_x_lanes.put(t + 4 * i, 0.0f);
                    d_delta_lanes.put(t + 4 * i, 0.0f);
                    if (gated) d_gate_lanes.put(t + 4 * i, 0.0f);
                }
            for (int e = threadIdx.x; e < K * N; e += LANES) if (t + e / N < p.end) store_shared(t, e, 0.0f, 0.0f);
        }
        T x[OWN], raw[OWN], gate[OWN], d_out[OWN];
        Shared<T, NPT, K> next;
        Resets<K> resets;
        float first_state[NPT];
        auto ask_chunk = [&](int t, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            x_lanes.template ask<WHOLE>(t, p.live, x);
            delta_lanes.template ask<WHOLE>(t, p.live, raw);
            d_out_lanes.template ask<WHOLE>(t, p.live, d_out);
            if (gated) gate_lanes.template ask<WHOLE>(t, p.live, gate);
            next.template ask<WHOLE, true, true>(a, p, t);
            resets.template ask<WHOLE>(a, p, t);
            read_global<NPT>((const GLOBAL char*)a.checkpoints + (pair * a.chunks + t / K) * a.channels * (N * sizeof(float)) + at_checkpoint, first_state);
        };
        if (chunks) {
            const int t = p.first + (chunks - 1) * K;
            ask_chunk(t, std::false_type{});
            if (t + K > p.live) {
                next.cut(p, t);
#pragma unroll
                for (int i = 0; i < OWN; i++) if (t + 4 * i + nq >= p.live) { x[i] = gate[i] = d_out[i] = (T)0.0f; raw[i] = (T)NO_DELTA; }
            }
        }
        for (int k = chunks - 1; k >= 0; k--, turn ^= 1) {
            const int t = p.first + k * K;
            float xs[OWN], delta[OWN], added[OWN], slope[OWN], d[OWN], by_gate[OWN];      // by_gate: the gate's gradient but for what it multiplies
            float h[K][NPT], decay[K][NPT], before[NPT];
            const unsigned forget = resets.get(p, t), passed = forget | (t + K > p.live ? ~0u << (p.live - t) : 0u);      // steps that add nothing to the rates' gradients: of another episode before them, or not there
            next.template put<true, true, true>(a, p, t, shared[turn]);
            if (!all_there && !there) {      // (lanes beyond the channels have another's state, which may be infinite)
#pragma unroll
                for (int i = 0; i < OWN; i++) { x[i] = gate[i] = d_out[i] = (T)0.0f; raw[i] = (T)NO_DELTA; }
#pragma unroll
                for (int n = 0; n < NPT; n++) first_state[n] = carry[n] = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < NPT; n++) before[n] = first_state[n];
#pragma unroll
            for (int i = 0; i < OWN; i++) {
                float e;
                const float v = (float)raw[i] + bias;
                xs[i] = (float)x[i];
                delta[i] = softplus<T>(v, e);
                const float large = reciprocal<T>(1.0f + e);
                slope[i] = v >= 0.0f ? large : e * large;      // of softplus
                added[i] = delta[i] * xs[i];
                d[i] = (float)d_out[i];
                by_gate[i] = 0.0f;
                if (gated) d[i] *= gate_factor<T>((float)gate[i], (float)d_out[i], by_gate[i]);
            }
            rlt_lds_barrier();
            const float* const bs = shared[turn][0] + n0; const float* const cs = shared[turn][1] + n0;
            auto walk = [&](auto with_resets) {
                constexpr bool RESETS = decltype(with_resets)::value;
#pragma unroll
                for (int i = 0; i < OWN; i++) {
                    auto step = [&](auto which) {
                        constexpr int j = decltype(which)::value;
                        const int s = 4 * i + j;
                        __builtin_amdgcn_sched_barrier(0);
                        const float dt = from_lane<j>(delta[i]), u = from_lane<j>(added[i]);
                        const bool begins = RESETS && bit(forget, s);
                        float b[NPT];
                        read<NPT>(bs + s * N, b);
#pragma unroll
                        for (int n = 0; n < NPT; n++) {
                            decay[s][n] = __builtin_amdgcn_exp2f(dt * rate[n]);
                            const float old = s ? h[s ? s - 1 : 0][n] : before[n];
                            h[s][n] = begins ? u * b[n] : fmaf(decay[s][n], old, u * b[n]);
                        }
                    };
                    step(std::integral_constant<int, 0>{}); step(std::integral_constant<int, 1>{}); step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 3>{});
                }
                asm volatile("" ::: "memory");      // b is read again rather than held from the walk forward; what other lanes hold is fetched again too
#pragma unroll
                for (int i = 0; i < OWN; i++) asm volatile("" : "+v"(delta[i]), "+v"(added[i]));
#pragma unroll
                for (int i = OWN - 1; i >= 0; i--) {
                    if (i == 0 && k > 0) ask_chunk(t - K, std::true_type{});      // the registers of states that are behind take what the next chunk needs
                    float mixed_part[4], through_part[4], exponent_part[4], kept_b[KEPT], kept_c[KEPT];
#pragma unroll
                    for (int m = 0; m < KEPT; m++) kept_b[m] = kept_c[m] = 0.0f;
                    auto step = [&](auto which) {
                        constexpr int j = decltype(which)::value;
                        const int s = 4 * i + j;
                        __builtin_amdgcn_sched_barrier(0);
                        const float dt = from_lane<j>(delta[i]), u = from_lane<j>(added[i]), g = from_lane<j>(d[i]);
                        const bool begins = RESETS && bit(forget, s), adds_nothing = RESETS && bit(passed, s);
                        float b[NPT], c[NPT], d_b[NPT], d_c[NPT];
                        read<NPT>(bs + s * N, b);
                        read<NPT>(cs + s * N, c);
                        mixed_part[j] = through_part[j] = exponent_part[j] = 0.0f;
#pragma unroll
                        for (int n = 0; n < NPT; n++) {
                            const float G = fmaf(c[n], g, carry[n]);
                            d_c[n] = g * h[s][n];
                            d_b[n] = u * G;
                            mixed_part[j] = fmaf(c[n], h[s][n], mixed_part[j]);
                            through_part[j] = fmaf(b[n], G, through_part[j]);
                            carry[n] = begins ? 0.0f : decay[s][n] * G;
                            const float old = s ? h[s ? s - 1 : 0][n] : before[n], q = adds_nothing ? 0.0f : carry[n] * old;
                            exponent_part[j] = fmaf(rate[n], q, exponent_part[j]);
                            d_rate[n] = fmaf(dt, q, d_rate[n]);
                        }
                        float sum_b[KEPT], sum_c[KEPT];
                        sum_channels<NPT>(d_b, sum_b);
                        sum_channels<NPT>(d_c, sum_c);
#pragma unroll
                        for (int m = 0; m < KEPT; m++) { kept_b[m] = into_quad<j>(kept_b[m], sum_b[m]); kept_c[m] = into_quad<j>(kept_c[m], sum_c[m]); }
                    };
                    step(std::integral_constant<int, 3>{}); step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 1>{}); step(std::integral_constant<int, 0>{});
                    const float mixed = sum_to_lane(mixed_part, odd, upper), through = sum_to_lane(through_part, odd, upper), exponent = sum_to_lane(exponent_part, odd, upper);
                    const bool live = !RESETS || t + 4 * i + nq < p.live;      // (nothing times a state or a gradient that is infinite is no zero)
                    const float d_delta = live ? fmaf(exponent, LN_2, through * xs[i]) * slope[i] : 0.0f;
                    d_skip = fmaf(d[i], xs[i], d_skip);
                    d_bias += d_delta;
                    if (there && t + 4 * i + nq < p.end) {
                        d_x_lanes.put(t + 4 * i, live ? fmaf(through, delta[i], skip * d[i]) : 0.0f);
                        d_delta_lanes.put(t + 4 * i, d_delta);
                        if (gated) d_gate_lanes.put(t + 4 * i, live ? by_gate[i] * fmaf(skip, xs[i], mixed) : 0.0f);
                    }
                    if (RESETS && t + 4 * i + quad >= p.live) {
#pragma unroll
                        for (int m = 0; m < KEPT; m++) kept_b[m] = kept_c[m] = 0.0f;
                    }
#pragma unroll
                    for (int m = 0; m < KEPT; m++) { slabs[turn][wave][0][(4 * i + quad) * N + kept_state + m] = kept_b[m]; slabs[turn][wave][1][(4 * i + quad) * N + kept_state + m] = kept_c[m]; }
                }
            };
            if (passed) walk(std::true_type{}); else walk(std::false_type{});
            rlt_lds_barrier();
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int e = threadIdx.x + j * LANES;
                if (e < K * N && t + e / N < p.end) {
                    float d_b = 0.0f, d_c = 0.0f;
#pragma unroll
                    for (int w = 0; w < WAVES; w++) { d_b += slabs[turn][w][0][e]; d_c += slabs[turn][w][1][e]; }
                    store_shared(t, e, d_b, d_c);
                }
            }
        }
        if (there && a.exit && p.segment == 0) store_states<NPT>(a.exit + (pair * a.channels + channel) * a.states, n0, a.states, carry);
    }
    if (!there) return;
    const size_t part = (size_t)p.segment * a.row_groups + group, of_channel = (part * a.heads + p.head) * a.channels + channel;
    if (a.d_rates) write<NPT>(a.d_rates + of_channel * N + n0, d_rate);
    d_skip = sum_of_lanes(d_skip); d_bias = sum_of_lanes(d_bias);
    if (nq == 0 && a.d_skips) a.d_skips[of_channel] = d_skip;
    if (nq == 0 && a.d_biases) a.d_biases[of_channel] = d_bias;
}

// Backward over sequences of K steps at most, as backward_kernel, from one row to the next like short_forward_kernel; nothing is computed for steps that are not there (both passes, 8 steps x 1,024 rows x 1,024 channels, fp32: 280 us, by whole
// chunks 433; one step x 8,192 rows x 4 heads of 256: 700 and 1,760). Registers for three wavefronts a SIMD where the states of its steps leave them (eight steps of more than
// sixteen states send 8 to 12 a lane to scratch memory, 36 to 52 bytes).
template <typename T, int NPT, bool ONE_TILE, int K> __global__ __launch_bounds__(LANES, NPT * K > 16 ? 2 : 3) void short_backward_kernel(Scan a) {
    constexpr int OWN = K / 4, N = 4 * NPT, KEPT = NPT > 4 ? NPT / 4 : 1;
    static_assert(K * N <= LANES, "");
    __shared__ float shared[2][2][K * N];
    __shared__ float slabs[2][WAVES][2][K * N];
    Place p = place_of(a, blockIdx.x, a.row_groups);
    const int group = p.row, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nq = lane & 3, quad = lane >> 2 & 3, n0 = nq * NPT, own_channel = p.tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1);
    const int kept_state = n0 + (NPT >= 4 ? (lane >> 4 & 1) * (NPT / 4) : 0) + (lane >> 5) * (NPT / 2);
    const bool there = own_channel < a.channels, gated = a.gate.data != nullptr, odd = nq & 1, upper = nq & 2;
    const size_t at_channel = (size_t)p.head * a.channels + channel;
    T x[OWN], raw[OWN], gate[OWN], d_out[OWN];
    Resets<K> resets;
    Shared<T, NPT, K> next;
    float first_state[NPT], entry[NPT];
    int live;
    auto ask = [&](int row) {
        const Arguments arguments;
        set_row(a, p, row);
        live = p.live;
        p.live = max(live, 1);      // (a row without steps reads its first one all the same, and looks at none)
        const Lanes<T> x_lanes(SCAN_PART(arguments, x), p, channel), delta_lanes(SCAN_PART(arguments, delta), p, channel), gate_lanes(SCAN_PART(arguments, gate), p, channel), d_out_lanes(SCAN_PART(arguments, d_out), p, channel);
        x_lanes.template ask<false>(0, p.live, x);
        delta_lanes.template ask<false>(0, p.live, raw);
        d_out_lanes.template ask<false>(0, p.live, d_out);
        if (gated) gate_lanes.template ask<false>(0, p.live, gate);
        next.template ask<false, true, true>(a, p, 0);
        resets.template ask<false>(a, p, 0);
        const size_t pair = pair_of(a, p);
        read_global<NPT>((const GLOBAL char*)a.checkpoints + pair * a.channels * (N * sizeof(float)) + (unsigned)(channel * N + n0) * sizeof(float), first_state);
        if (a.entry) load_states<NPT>(a.entry + (pair * a.channels + channel) * a.states, n0, a.states, entry);
        p.live = live;
    };
#pragma unroll
    for (int n = 0; n < NPT; n++) entry[n] = 0.0f;
    ask(group);
    const float bias = a.delta_biases ? a.delta_biases[at_channel] : 0.0f, skip = a.skip ? a.skip[at_channel] : 0.0f;
    float rate[NPT], d_rate[NPT], d_skip = 0.0f, d_bias = 0.0f;
    load_rates<NPT>(a, p.head, channel, n0, rate);
#pragma unroll
    for (int n = 0; n < NPT; n++) d_rate[n] = 0.0f;
    const unsigned own = there ? ~0u : 0u;
    int turn = 0;
    for (int row = group; row < a.batch; row += a.row_groups, turn ^= 1) {
        const size_t pair = (size_t)row * a.heads + p.head;
        const int steps = live;
        float by_gate[OWN], h[K][NPT], decay[K][NPT], before[NPT], carry[NPT], xs[OWN], delta[OWN], added[OWN], slope[OWN], d[OWN];
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const bool whole = there && 4 * i + nq < steps;
            float e;
            const float v = whole ? (float)raw[i] + bias : NO_DELTA;
            xs[i] = whole ? (float)x[i] : 0.0f;
            delta[i] = softplus<T>(v, e);
            const float large = reciprocal<T>(1.0f + e);
            slope[i] = v >= 0.0f ? large : e * large;
            added[i] = delta[i] * xs[i];
            d[i] = whole ? (float)d_out[i] : 0.0f;
            by_gate[i] = 0.0f;
            if (gated) {
                const float g = d[i];
                d[i] *= gate_factor<T>(whole ? (float)gate[i] : 0.0f, g, by_gate[i]);
            }
        }
        const unsigned forget = resets.get(p, 0);
        next.template put<false, true, true>(a, p, 0, shared[turn]);
#pragma unroll
        for (int n = 0; n < NPT; n++) {      // (lanes beyond the channels have another's state, which may be infinite: none)
            before[n] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, first_state[n]) & own);
            carry[n] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, entry[n]) & own);
        }
        const Arguments arguments;
        const Lanes<T> d_x_lanes(SCAN_PART(arguments, d_x), p, channel), d_delta_lanes(SCAN_PART(arguments, d_delta), p, channel), d_gate_lanes(SCAN_PART(arguments, d_gate), p, channel);
        ask(min(row + a.row_groups, a.batch - 1));
        rlt_lds_barrier();
        each<0, K>([&](auto which) {
            constexpr int j = decltype(which)::value;
            if (j < steps) {
                const float dt = from_lane<j % 4>(delta[j / 4]), u = from_lane<j % 4>(added[j / 4]);
                const bool begins = forget >> j & 1;
                float b[NPT];
                read<NPT>(shared[turn][0] + n0 + j * N, b);
#pragma unroll
                for (int n = 0; n < NPT; n++) {
                    decay[j][n] = __builtin_amdgcn_exp2f(dt * rate[n]);
                    h[j][n] = begins ? u * b[n] : fmaf(decay[j][n], j ? h[j ? j - 1 : 0][n] : before[n], u * b[n]);
                }
            }
        });
        each<0, OWN>([&](auto group_of_four) {
            constexpr int i = OWN - 1 - decltype(group_of_four)::value;
            float mixed_part[4], through_part[4], exponent_part[4], kept_b[KEPT], kept_c[KEPT];
#pragma unroll
            for (int m = 0; m < KEPT; m++) kept_b[m] = kept_c[m] = 0.0f;
            each<0, 4>([&](auto which) {
                constexpr int j = 3 - decltype(which)::value, s = 4 * i + j;
                mixed_part[j] = through_part[j] = exponent_part[j] = 0.0f;
                if (s < steps) {
                    const float dt = from_lane<j>(delta[i]), u = from_lane<j>(added[i]), g = from_lane<j>(d[i]);
                    const bool begins = forget >> s & 1;
                    float b[NPT], c[NPT], d_b[NPT], d_c[NPT];
                    read<NPT>(shared[turn][0] + n0 + s * N, b);
                    read<NPT>(shared[turn][1] + n0 + s * N, c);
#pragma unroll
                    for (int n = 0; n < NPT; n++) {
                        const float G = fmaf(c[n], g, carry[n]);
                        d_c[n] = g * h[s][n];
                        d_b[n] = u * G;
                        mixed_part[j] = fmaf(c[n], h[s][n], mixed_part[j]);
                        through_part[j] = fmaf(b[n], G, through_part[j]);
                        carry[n] = begins ? 0.0f : decay[s][n] * G;
                        const float old = s ? h[s ? s - 1 : 0][n] : before[n], q = begins ? 0.0f : carry[n] * old;
                        exponent_part[j] = fmaf(rate[n], q, exponent_part[j]);
                        d_rate[n] = fmaf(dt, q, d_rate[n]);
                    }
                    float sum_b[KEPT], sum_c[KEPT];
                    sum_channels<NPT>(d_b, sum_b);
                    sum_channels<NPT>(d_c, sum_c);
#pragma unroll
                    for (int m = 0; m < KEPT; m++) { kept_b[m] = into_quad<j>(kept_b[m], sum_b[m]); kept_c[m] = into_quad<j>(kept_c[m], sum_c[m]); }
                }
            });
            const float mixed = sum_to_lane(mixed_part, odd, upper), through = sum_to_lane(through_part, odd, upper), exponent = sum_to_lane(exponent_part, odd, upper);
            const float d_delta = fmaf(exponent, LN_2, through * xs[i]) * slope[i];
            d_skip = fmaf(d[i], xs[i], d_skip);
            d_bias += d_delta;
            if (there && 4 * i + nq < a.steps) {
                d_x_lanes.put(4 * i, fmaf(through, delta[i], skip * d[i]));
                d_delta_lanes.put(4 * i, d_delta);
                if (gated) d_gate_lanes.put(4 * i, by_gate[i] * fmaf(skip, xs[i], mixed));
            }
#pragma unroll
            for (int m = 0; m < KEPT; m++) { slabs[turn][wave][0][(4 * i + quad) * N + kept_state + m] = kept_b[m]; slabs[turn][wave][1][(4 * i + quad) * N + kept_state + m] = kept_c[m]; }
        });
        rlt_lds_barrier();
        const int element = threadIdx.x, step = element / N, n = element % N;
        if (step < a.steps && element < K * N) {
            float d_b = 0.0f, d_c = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) { d_b += slabs[turn][w][0][element]; d_c += slabs[turn][w][1][element]; }
            if constexpr (ONE_TILE) {
                if (n < a.states) {
                    at<T>(a.d_b, step, row, p.head)[n] = (T)d_b;
                    at<T>(a.d_c, step, row, p.head)[n] = (T)d_c;
                }
            } else {
                float* const to = a.d_shared + ((size_t)p.tile * 2 * a.batch * a.heads + pair) * a.steps * N + element;
                to[0] = d_b;
                to[(size_t)a.batch * a.heads * a.steps * N] = d_c;
            }
        }
        if (there && a.exit) store_states<NPT>(a.exit + (pair * a.channels + channel) * a.states, n0, a.states, carry);
    }
    if (!there) return;
    const size_t of_channel = ((size_t)group * a.heads + p.head) * a.channels + channel;
    if (a.d_rates) write<NPT>(a.d_rates + of_channel * N + n0, d_rate);
    d_skip = sum_of_lanes(d_skip); d_bias = sum_of_lanes(d_bias);
    if (nq == 0 && a.d_skips) a.d_skips[of_channel] = d_skip;
    if (nq == 0 && a.d_biases) a.d_biases[of_channel] = d_bias;
}

// What a segment adds to the state's gradient that reaches it from its end, for the gradients that segments start from.
template <typename T, int NPT> __global__ __launch_bounds__(LANES) void backward_states_kernel(Scan a) {
    constexpr int K = CHUNK<NPT>, OWN = K / 4, N = 4 * NPT;
    __shared__ float shared[2][2][K * N];
    Place p = place_of(a, blockIdx.x + (unsigned)a.tiles * a.heads * a.batch, a.batch);      // the first segment's states reach none
    set_row(a, p, p.row);
    const int lane = threadIdx.x & 63, nq = lane & 3, n0 = nq * NPT, own_channel = p.tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1);
    const bool there = own_channel < a.channels, all_there = (p.tile + 1) * TILE <= a.channels, gated = a.gate.data != nullptr;
    const size_t pair = pair_of(a, p);
    float rate[NPT], carry[NPT], sum = 0.0f;
    load_rates<NPT>(a, p.head, channel, n0, rate);
    const float bias = a.delta_biases ? a.delta_biases[(size_t)p.head * a.channels + channel] : 0.0f;
    bool forgotten = false;
#pragma unroll
    for (int n = 0; n < NPT; n++) carry[n] = 0.0f;
    T raw[OWN], gate[OWN], d_out[OWN];
    Resets<K> resets;
    Shared<T, NPT> next;
    const Arguments arguments;
    const Lanes<T> delta_lanes(SCAN_PART(arguments, delta), p, channel), gate_lanes(SCAN_PART(arguments, gate), p, channel), d_out_lanes(SCAN_PART(arguments, d_out), p, channel);
    auto ask_chunk = [&](int t) {
        delta_lanes.template ask<false>(t, p.live, raw);
        d_out_lanes.template ask<false>(t, p.live, d_out);
        if (gated) gate_lanes.template ask<false>(t, p.live, gate);
        next.template ask<false, false, true>(a, p, t);
        resets.template ask<false>(a, p, t);
    };
    const int chunks = p.live > p.first ? (p.live - p.first + K - 1) / K : 0;
    if (chunks) ask_chunk(p.first + (chunks - 1) * K);
    int turn = 0;
    for (int k = chunks - 1; k >= 0; k--, turn ^= 1) {
        const int t = p.first + k * K;
        float delta[OWN], d[OWN];
        if (!all_there || t + K > p.live) {
#pragma unroll
            for (int i = 0; i < OWN; i++) if (!there || t + 4 * i + nq >= p.live) { gate[i] = d_out[i] = (T)0.0f; raw[i] = (T)NO_DELTA; }
        }
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            float e;
            delta[i] = softplus<T>((float)raw[i] + bias, e);
            d[i] = (float)d_out[i];
            if (gated) d[i] *= gate_factor<T>((float)gate[i]);
            sum += delta[i];
        }
        const unsigned forget = resets.get(p, t);
        next.template put<false, false, true>(a, p, t, shared[turn]);
        if (k > 0) ask_chunk(t - K);
        rlt_lds_barrier();
        const float* const cs = shared[turn][1] + n0;
#pragma unroll
        for (int i = OWN - 1; i >= 0; i--) {
            auto step = [&](auto which) {
                constexpr int j = decltype(which)::value;
                const float dt = from_lane<j>(delta[i]), g = from_lane<j>(d[i]);
                float c[NPT];
                read<NPT>(cs + (4 * i + j) * N, c);
#pragma unroll
                for (int n = 0; n < NPT; n++) carry[n] = __builtin_amdgcn_exp2f(dt * rate[n]) * fmaf(c[n], g, carry[n]);
                if (forget >> (4 * i + j) & 1) {
                    forgotten = true;
#pragma unroll
                    for (int n = 0; n < NPT; n++) carry[n] = 0.0f;
                }
            };
            step(std::integral_constant<int, 3>{}); step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 1>{}); step(std::integral_constant<int, 0>{});
        }
    }
    if (!there) return;
    write<NPT>(a.exit + ((pair * a.segments + p.segment) * a.channels + channel) * N + n0, carry);
    sum = sum_of_lanes(sum);
    if (nq == 0) a.sums[(pair * a.segments + p.segment) * a.channels + channel] = forgotten ? -1.0f : sum;
}

// The sums behind the backward pass, in one launch (8,192 steps x 2 rows x 2,048 channels: 25 us; in two 29). The first workgroups: the parameters' gradients out of the workgroups' shares, sixteen elements of one of the three each. The others: d_b and d_c out of the tiles' shares.
template <typename T> __global__ __launch_bounds__(1024) void sum_kernel(Scan a, int parts, int padded, unsigned of_parameters, float* __restrict__ d_log_rates, float* __restrict__ d_skip, float* __restrict__ d_delta_biases, int accumulate) {
    if (blockIdx.x >= of_parameters) {
        const size_t size = (size_t)a.batch * a.heads * a.steps * padded;
        for (size_t i = (size_t)(blockIdx.x - of_parameters) * 1024 + threadIdx.x; i < 2 * size; i += (size_t)(gridDim.x - of_parameters) * 1024) {
            const bool second = i >= size;
            const size_t e = second ? i - size : i, line = e / padded, pair = line / a.steps;
            const int n = (int)(e - line * padded), step = (int)(line - pair * a.steps), row = (int)(pair / a.heads), head = (int)(pair - (size_t)row * a.heads);
            if (n >= a.states) continue;
            float s = 0.0f;
            for (int tile = 0; tile < a.tiles; tile += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = a.d_shared[(size_t)min(tile + j, a.tiles - 1) * 2 * size + i];
#pragma unroll
                for (int j = 0; j < 8; j++) s += tile + j < a.tiles ? v[j] : 0.0f;
            }
            at<T>(second ? a.d_c : a.d_b, step, row, head)[n] = (T)s;
        }
        return;
    }
    const size_t channels = (size_t)a.heads * a.channels, rates = channels * padded;
    const unsigned of_rates = (unsigned)((rates + RLT_JOIN_COLUMNS - 1) / RLT_JOIN_COLUMNS), of_channels = (unsigned)((channels + RLT_JOIN_COLUMNS - 1) / RLT_JOIN_COLUMNS);
    const int which = blockIdx.x < of_rates ? 0 : blockIdx.x < of_rates + of_channels ? 1 : 2;
    const size_t columns = which ? channels : rates, i = (size_t)(blockIdx.x - (which ? of_rates : 0) - (which == 2 ? of_channels : 0)) * RLT_JOIN_COLUMNS + threadIdx.x % RLT_JOIN_COLUMNS;
    const float* const from = which == 0 ? a.d_rates : which == 1 ? a.d_skips : a.d_biases;
    if (!from) return;
    float s = rlt_join_column(from, parts, columns, i, i < columns);
    if (threadIdx.x >= RLT_JOIN_COLUMNS || i >= columns) return;
    float* to = which == 1 ? d_skip + i : d_delta_biases + i;
    if (which == 0) {
        const size_t channel = i / padded;
        const int n = (int)(i - channel * padded);
        if (n >= a.states) return;
        to = d_log_rates + channel * a.states + n;
        s *= -rate_of(a.log_rates[channel * a.states + n]);
    }
    *to = accumulate ? *to + s : s;
}

// One step of four rows: a pass over the states, which are read and written once, and what bounds it (4,096 rows x 1,024 channels x 16 states, bfloat16: 105 us, 5.5 TB/s). Four lanes share a channel, each with a quarter of its states of every row
// and all that depends on the step alone of one of them. VECTORS: a lane's NPT states are read and written together, from any element on, which the memory instructions allow; the last lanes' states end with the channel's, so that some are another
// lane's too: both compute and write the same, and one of them counts.
template <typename T, int NPT, bool VECTORS> __global__ __launch_bounds__(LANES) void step_kernel(Scan a) {
    constexpr int V = NPT < 4 ? NPT : 4;
    typedef float vector __attribute__((ext_vector_type(V), aligned(4)));
    const int nq = threadIdx.x & 3, own_n0 = nq * NPT, n0 = VECTORS ? min(own_n0, a.states - NPT) : own_n0;
    unsigned item = blockIdx.x;
    const int tile = item % a.tiles; item /= a.tiles;
    const int head = item % a.heads, row0 = item / a.heads * 4, own_channel = tile * TILE + (int)(threadIdx.x >> 2), channel = min(own_channel, a.channels - 1), own_row = min(row0 + nq, a.batch - 1);
    const bool there = own_channel < a.channels;
    const size_t at_channel = (size_t)head * a.channels + channel;
    float h[4][NPT], rate[NPT], sum[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = min(row0 + r, a.batch - 1);
        const float* const from = a.entry + (((size_t)row * a.heads + head) * a.channels + channel) * a.states;
        if constexpr (VECTORS) {
#pragma unroll
            for (int n = 0; n < NPT; n += V) {
                const vector v = *reinterpret_cast<const vector*>(from + n0 + n);
#pragma unroll
                for (int i = 0; i < V; i++) h[r][n + i] = v[i];
            }
        } else load_states<NPT>(from, n0, a.states, h[r]);
    }
    const float x = (float)at<T>(a.x, 0, own_row, head)[channel], raw = (float)at<T>(a.delta, 0, own_row, head)[channel], z = a.gate.data ? (float)at<T>(a.gate, 0, own_row, head)[channel] : 0.0f;
    const bool forget = a.reset && a.reset[own_row];
    load_rates<NPT>(a, head, channel, n0, rate);
    float e;
    const float delta = softplus<T>(raw + (a.delta_biases ? a.delta_biases[at_channel] : 0.0f), e), u = delta * x, forgets = forget ? 1.0f : 0.0f;
    each<0, 4>([&](auto which) {
        constexpr int r = decltype(which)::value;
        const int row = min(row0 + r, a.batch - 1);
        const float d = from_lane<r>(delta), added = from_lane<r>(u);
        const bool begins = from_lane<r>(forgets) != 0.0f;
        const T* const b = at<T>(a.b, 0, row, head); const T* const c = at<T>(a.c, 0, row, head);
        sum[r] = 0.0f;
#pragma unroll
        for (int n = 0; n < NPT; n++) {
            const bool in = VECTORS || n0 + n < a.states;
            const float bn = in ? (float)b[n0 + n] : 0.0f, cn = in ? (float)c[n0 + n] : 0.0f;
            h[r][n] = fmaf(__builtin_amdgcn_exp2f(d * rate[n]), begins ? 0.0f : h[r][n], added * bn);
            const float counted = fmaf(cn, h[r][n], sum[r]);
            sum[r] = !VECTORS || n0 + n >= own_n0 ? counted : sum[r];
        }
        float* const to = a.exit + (((size_t)row * a.heads + head) * a.channels + channel) * a.states;
        if (there && row0 + r < a.batch) {
            if constexpr (VECTORS) {
#pragma unroll
                for (int n = 0; n < NPT; n += V) {
                    vector v;
#pragma unroll
                    for (int i = 0; i < V; i++) v[i] = h[r][n + i];
                    *reinterpret_cast<vector*>(to + n0 + n) = v;
                }
            } else store_states<NPT>(to, n0, a.states, h[r]);
        }
    });
    float v = sum_to_lane(sum, nq & 1, nq & 2);
    if (a.skip) v = fmaf(a.skip[at_channel], x, v);
    if (a.gate.data) v *= gate_factor<T>(z);
    if (there && row0 + nq < a.batch) at<T>(a.out, 0, own_row, head)[channel] = (T)v;
}

bool described(const rlt_selective_scan* p) {
    return p && (p->type == RLT_TYPE_F32 || p->type == RLT_TYPE_BF16) && p->batch > 0 && p->heads > 0 && p->channels > 0 && p->states > 0;
}
int tiles_of(const rlt_selective_scan* p) { return (p->channels + TILE - 1) / TILE; }

// Steps are cut into segments, the same for both passes, where rows, heads and channels alone leave the chip without work: up to four wavefronts to a SIMD, where they have fewer than two (a pass more over the steps is not worth less: 104 steps x 37 rows x 1,024 channels,
// forward and backward, 125 us whole, 146 in three segments). A chunk takes the passes over a segment some 6 us, and a segment the launches that chain them 0.6, one after the other: their sum is least, and flat, around four times the root of the
// chunks (16,000 steps x 1 row x 64 channels: 172 us in 126 segments, 205 in 250, 620 in 1,000; 203 steps x 4 rows x 256 channels: 44 in 13, 75 in three).
struct Segments { int count, steps, row_groups; };
Segments segments_of(const rlt_selective_scan* p, int steps) {
    const int chunk = chunk_of(p->states), chunks = (steps + chunk - 1) / chunk;
    const int64_t blocks = (int64_t)p->batch * p->heads * tiles_of(p), most = std::min((int64_t)(4.0 * std::sqrt((double)chunks)), (int64_t)chunks);
    const int64_t count = std::max(std::min(blocks >= 512 ? 1 : (1024 + blocks - 1) / blocks, most), (int64_t)1);
    const int per = (int)((chunks + count - 1) / count);
    Segments g = {(chunks + per - 1) / per, per * chunk, 0};
    int64_t groups = 2048 / ((int64_t)p->heads * tiles_of(p) * g.count);      // rows are walked one after the other where there are more than fill the chip
    g.row_groups = (int)(groups < 1 ? 1 : groups < p->batch ? groups : p->batch);
    return g;
}
bool supported(const rlt_selective_scan* p, int steps) {
    if (p->states > MAX_STATES || steps > MAX_STEPS) return false;
    const __int128 pairs = (__int128)p->batch * p->heads, limit = (__int128)1 << 31;
    if (pairs * p->channels * MAX_STATES > limit || pairs * steps > limit || (int64_t)p->heads * p->channels > MAX_CHANNELS) return false;
    const __int128 blocks = pairs * tiles_of(p) * segments_of(p, steps).count;
    return blocks * LANES <= UINT32_MAX;
}
size_t padded(size_t n) { return (n + 63) / 64 * 64; }
// scratch memory, in floats
struct Scratch { size_t states, sums, shared, rates, skips, biases, total; };
Scratch scratch_of(const rlt_selective_scan* p, int steps, bool backward) {
    const Segments g = segments_of(p, steps);
    const size_t channels = (size_t)p->batch * p->heads * p->channels, wide = 4 * per_lane(p->states), parts = (size_t)g.row_groups * g.count * p->heads * p->channels;
    Scratch s{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += padded(n); return here; };
    if (g.count > 1) { s.states = take(channels * g.count * wide); s.sums = take(channels * g.count); }
    if (backward) {
        if (tiles_of(p) > 1) s.shared = take((size_t)tiles_of(p) * 2 * steps * p->batch * p->heads * wide);
        s.rates = take(parts * wide); s.skips = take(parts); s.biases = take(parts);
    }
    s.total = at;
    return s;
}
Scan scan_of(const rlt_selective_scan* p, const rlt_head_view* x, const rlt_head_view* delta, const rlt_head_view* b, const rlt_head_view* c, const rlt_head_view* gate, const uint8_t* reset,
             const int32_t* lengths, int steps) {
    const Segments g = segments_of(p, steps);
    Scan a{};
    a.log_rates = p->log_rates; a.skip = p->skip; a.delta_biases = p->delta_biases;
    a.x = rlt_part_of(x); a.delta = rlt_part_of(delta); a.b = rlt_part_of(b); a.c = rlt_part_of(c); a.gate = rlt_part_of(gate);
    a.reset = reset; a.lengths = lengths; a.batch = p->batch; a.heads = p->heads; a.channels = p->channels; a.states = p->states; a.steps = steps;
    a.segments = g.count; a.segment_steps = g.steps; a.row_groups = g.row_groups; a.tiles = tiles_of(p); a.chunks = (steps + chunk_of(p->states) - 1) / chunk_of(p->states);
    return a;
}
template <typename F> int by_kind(const rlt_selective_scan* p, F&& f) {
    auto typed = [&](auto type) {
        const int n = per_lane(p->states);
        return n == 2 ? f(type, std::integral_constant<int, 2>{}) : n == 4 ? f(type, std::integral_constant<int, 4>{}) : f(type, std::integral_constant<int, 8>{});
    };
    return p->type == RLT_TYPE_F32 ? typed(0.0f) : typed((rlt_bf16)0.0f);
}
unsigned blocks_of(const Scan& a, int rows) { return (unsigned)a.tiles * a.heads * a.segments * rows; }
template <bool REVERSE> int join_segments(rlt_rocm_device* device, const Scan& a, const float* initial, float* states, int wide) {
    const size_t blocks = ((size_t)a.batch * a.heads * a.channels * wide + 255) / 256;
    hipLaunchKernelGGL(join_segments_kernel<REVERSE>, dim3((unsigned)blocks), dim3(256), 0, device->stream, a, initial, states, wide);
    return rlt_launch_status(device);
}
template <typename... V> bool near(const V*... views) { return ((!views || (views->step_stride >= -MAX_STRIDE && views->step_stride <= MAX_STRIDE)) && ...); }
bool given(const rlt_selective_scan* p, const rlt_head_view* x, const rlt_head_view* delta, const rlt_head_view* b, const rlt_head_view* c, const rlt_head_view* gate) {
    return described(p) && p->log_rates && rlt_given(x) && rlt_given(delta) && rlt_given(b) && rlt_given(c) && (!gate || gate->data);
}

}  // namespace

extern "C" {

size_t rlt_rocm_selective_scan_workspace_bytes(const rlt_selective_scan* layer, int steps, int backward) {
    if (!described(layer) || steps <= 0 || !supported(layer, steps)) return 0;
    return scratch_of(layer, steps, backward != 0).total * sizeof(float);
}
size_t rlt_rocm_selective_scan_checkpoint_bytes(const rlt_selective_scan* layer, int steps) {
    if (!described(layer) || steps <= 0 || !supported(layer, steps)) return 0;
    const int chunk = chunk_of(layer->states);
    return (size_t)layer->batch * layer->heads * ((steps + chunk - 1) / chunk) * layer->channels * 4 * per_lane(layer->states) * sizeof(float);
}

int rlt_rocm_selective_scan_forward(rlt_rocm_device* device, const rlt_selective_scan* layer, const rlt_head_view* x, const rlt_head_view* delta, const rlt_head_view* b, const rlt_head_view* c,
                                    const rlt_head_view* gate, const rlt_head_view* output, const float* initial_state, float* final_state, const uint8_t* reset, const int32_t* lengths, int steps,
                                    void* checkpoints, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(given(layer, x, delta, b, c, gate) && rlt_given(output) && steps > 0 && reinterpret_cast<uintptr_t>(checkpoints) % 16 == 0);
    if (!supported(layer, steps) || !near(x, delta, b, c, gate, output)) return RLT_E_UNSUPPORTED;
    const Scratch s = scratch_of(layer, steps, false);
    RLT_REQUIRE(s.total == 0 || (workspace && workspace_bytes >= s.total * sizeof(float) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0));
    Scan a = scan_of(layer, x, delta, b, c, gate, reset, lengths, steps);
    a.out = rlt_part_of(output); a.checkpoints = (float*)checkpoints; a.entry = initial_state; a.exit = final_state;
    return by_kind(layer, [&](auto type, auto n) {
        typedef decltype(type) T;
        constexpr int NPT = decltype(n)::value;
        if (a.segments > 1) {
            Scan f = a;
            float* const states = (float*)workspace + s.states;
            f.sums = (float*)workspace + s.sums; f.exit = states;
            hipLaunchKernelGGL((forward_kernel<T, NPT, true>), dim3(blocks_of(a, a.batch) / a.segments * (a.segments - 1)), dim3(LANES), 0, device->stream, f);      // (nothing starts from what the last segment adds)
            int rc = rlt_launch_status(device);
            if (rc || (rc = join_segments<false>(device, f, initial_state, states, 4 * NPT))) return rc;
            a.entry = states; a.entry_padded = 1;
        }
        const dim3 blocks(blocks_of(a, a.batch));
        if (steps <= 4) hipLaunchKernelGGL((short_forward_kernel<T, NPT, 4>), dim3(blocks_of(a, a.row_groups)), dim3(LANES), 0, device->stream, a);
        else if (steps <= 8) hipLaunchKernelGGL((short_forward_kernel<T, NPT, 8>), dim3(blocks_of(a, a.row_groups)), dim3(LANES), 0, device->stream, a);
        else hipLaunchKernelGGL((forward_kernel<T, NPT, false>), blocks, dim3(LANES), 0, device->stream, a);
        return rlt_launch_status(device);
    });
}

int rlt_rocm_selective_scan_backward(rlt_rocm_device* device, const rlt_selective_scan* layer, const rlt_head_view* x, const rlt_head_view* delta, const rlt_head_view* b, const rlt_head_view* c,
                                     const rlt_head_view* gate, const rlt_head_view* d_output, const rlt_head_view* d_x, const rlt_head_view* d_delta, const rlt_head_view* d_b, const rlt_head_view* d_c,
                                     const rlt_head_view* d_gate, const float* d_final_state, float* d_initial_state, int accumulate, const uint8_t* reset, const int32_t* lengths, int steps,
                                     const void* checkpoints, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(given(layer, x, delta, b, c, gate) && rlt_given(d_output) && rlt_given(d_x) && rlt_given(d_delta) && rlt_given(d_b) && rlt_given(d_c) && (!gate || rlt_given(d_gate)) && steps > 0);
    RLT_REQUIRE(checkpoints && reinterpret_cast<uintptr_t>(checkpoints) % 16 == 0);
    if (!supported(layer, steps) || !near(x, delta, b, c, gate, d_output, d_x, d_delta, d_b, d_c, gate ? d_gate : nullptr)) return RLT_E_UNSUPPORTED;
    const Scratch s = scratch_of(layer, steps, true);
    RLT_REQUIRE(workspace && workspace_bytes >= s.total * sizeof(float) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
    float* const w = (float*)workspace;
    Scan a = scan_of(layer, x, delta, b, c, gate, reset, lengths, steps);
    a.d_out = rlt_part_of(d_output); a.d_x = rlt_part_of(d_x); a.d_delta = rlt_part_of(d_delta); a.d_b = rlt_part_of(d_b); a.d_c = rlt_part_of(d_c); a.d_gate = rlt_part_of(d_gate);
    a.checkpoints = (float*)const_cast<void*>(checkpoints); a.entry = d_final_state; a.exit = d_initial_state;
    a.d_shared = w + s.shared; a.d_rates = layer->d_log_rates ? w + s.rates : nullptr; a.d_skips = layer->d_skip ? w + s.skips : nullptr; a.d_biases = layer->d_delta_biases ? w + s.biases : nullptr;
    return by_kind(layer, [&](auto type, auto n) {
        typedef decltype(type) T;
        constexpr int NPT = decltype(n)::value;
        int rc;
        if (a.segments > 1) {
            Scan f = a;
            f.sums = w + s.sums; f.exit = w + s.states;
            hipLaunchKernelGGL((backward_states_kernel<T, NPT>), dim3(blocks_of(a, a.batch) / a.segments * (a.segments - 1)), dim3(LANES), 0, device->stream, f);      // (nothing goes on from the first segment)
            if ((rc = rlt_launch_status(device)) || (rc = join_segments<true>(device, f, d_final_state, f.exit, 4 * NPT))) return rc;
            a.entry = f.exit; a.entry_padded = 1;
        }
        const dim3 blocks(blocks_of(a, a.row_groups));
        auto walk = [&](auto one_tile) {
            constexpr bool ONE_TILE = decltype(one_tile)::value;
            if (steps <= 4) hipLaunchKernelGGL((short_backward_kernel<T, NPT, ONE_TILE, 4>), blocks, dim3(LANES), 0, device->stream, a);
            else if (steps <= 8) hipLaunchKernelGGL((short_backward_kernel<T, NPT, ONE_TILE, 8>), blocks, dim3(LANES), 0, device->stream, a);
            else hipLaunchKernelGGL((backward_kernel<T, NPT, ONE_TILE>), blocks, dim3(LANES), 0, device->stream, a);
        };
        if (a.tiles == 1) walk(std::true_type{});
        else walk(std::false_type{});
        if ((rc = rlt_launch_status(device))) return rc;
        const size_t channels = (size_t)layer->heads * layer->channels, shared = a.tiles > 1 ? (size_t)2 * a.batch * a.heads * steps * 4 * NPT : 0;
        auto blocks_for = [](size_t columns) { return (columns + RLT_JOIN_COLUMNS - 1) / RLT_JOIN_COLUMNS; };
        const size_t of_parameters = a.d_rates || a.d_skips || a.d_biases ? blocks_for(channels * 4 * NPT) + 2 * blocks_for(channels) : 0, of_shared = std::min((shared + 1023) / 1024, (size_t)4096);
        if (of_parameters + of_shared == 0) return 0;
        hipLaunchKernelGGL(sum_kernel<T>, dim3((unsigned)(of_parameters + of_shared)), dim3(1024), 0, device->stream, a, a.row_groups * a.segments, 4 * NPT, (unsigned)of_parameters, layer->d_log_rates, layer->d_skip,
                           layer->d_delta_biases, accumulate);
        return rlt_launch_status(device);
    });
}

int rlt_rocm_selective_scan_step(rlt_rocm_device* device, const rlt_selective_scan* layer, const rlt_head_view* x, const rlt_head_view* delta, const rlt_head_view* b, const rlt_head_view* c,
                                 const rlt_head_view* gate, const rlt_head_view* output, const float* state, float* next_state, const uint8_t* reset) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(given(layer, x, delta, b, c, gate) && rlt_given(output) && state && next_state);
    if (!supported(layer, 1)) return RLT_E_UNSUPPORTED;
    Scan a = scan_of(layer, x, delta, b, c, gate, reset, nullptr, 1);
    a.out = rlt_part_of(output); a.entry = state; a.exit = next_state;
    return by_kind(layer, [&](auto type, auto n) {
        typedef decltype(type) T;
        constexpr int NPT = decltype(n)::value;
        const dim3 blocks((unsigned)a.tiles * a.heads * ((a.batch + 3) / 4));
        if (a.states >= NPT) hipLaunchKernelGGL((step_kernel<T, NPT, true>), blocks, dim3(LANES), 0, device->stream, a);
        else hipLaunchKernelGGL((step_kernel<T, NPT, false>), blocks, dim3(LANES), 0, device->stream, a);
        return rlt_launch_status(device);
    });
}

}  // extern "C"
