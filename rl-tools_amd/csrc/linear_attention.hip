// Linear attention with a decay for each head: sequences forward and backward, and single steps on a kept state.
#include "typed.h"

namespace {

constexpr int MAX_WIDTH = 128;

// a tensor as the kernels see it: heads / group of it
struct Part { const void* data; int64_t step, row, head; int group; };
struct Walk {
    Part q, k, v;                 // what reads the state, and the two factors of what is added to it
    Part out;                     // written
    const float* log_decay; const float* initial; float* final;
    const uint8_t* reset; const int32_t* lengths;
    float scale_out, scale_added;
    int batch, heads, steps, key, value;
};

template <typename T> __device__ __forceinline__ T* at(const Part& p, int t, int b, int h) {
    return (T*)p.data + ((int64_t)t * p.step + (int64_t)b * p.row + (int64_t)(h / p.group) * p.head);
}

// One workgroup per row and head walks the steps; thread c holds column c of the state. Forward: the state decays, takes k^T v in and is read by q. REVERSE: it takes k^T v in, is read and decays.
// TRANSPOSED: the state lies in memory as [value x key].
template <typename T, typename O, bool REVERSE, bool TRANSPOSED> __global__ __launch_bounds__(MAX_WIDTH) void walk_kernel(Walk a) {
    __shared__ float q[MAX_WIDTH], k[MAX_WIDTH];
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, c = threadIdx.x;
    const float decay = expf(a.log_decay[h]);
    const size_t base = ((size_t)b * a.heads + h) * a.key * a.value;
    float state[MAX_WIDTH];
#pragma unroll
    for (int i = 0; i < MAX_WIDTH; i++) state[i] = a.initial && c < a.value && i < a.key ? a.initial[base + (TRANSPOSED ? c * a.key + i : i * a.value + c)] : 0.0f;
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.steps) : a.steps;
    for (int s = 0; s < a.steps; s++) {
        const int t = REVERSE ? a.steps - 1 - s : s;
        if (t >= length) {
            if (a.out.data && c < a.value) at<O>(a.out, t, b, h)[c] = (O)0.0f;
            continue;
        }
        __syncthreads();
        q[c] = c < a.key ? (float)at<T>(a.q, t, b, h)[c] : 0.0f;
        k[c] = c < a.key ? (float)at<T>(a.k, t, b, h)[c] * a.scale_added : 0.0f;
        const float v = c < a.value ? (float)at<T>(a.v, t, b, h)[c] : 0.0f;
        __syncthreads();
        const bool forget = a.reset && a.reset[(size_t)t * a.batch + b];
        float out = 0.0f;
#pragma unroll
        for (int i = 0; i < MAX_WIDTH; i++) {
            if (!REVERSE) state[i] = forget ? 0.0f : state[i] * decay;
            state[i] = fmaf(k[i], v, state[i]);
            out = fmaf(q[i], state[i], out);
            if (REVERSE) state[i] = forget ? 0.0f : state[i] * decay;
        }
        if (a.out.data && c < a.value) at<O>(a.out, t, b, h)[c] = (O)(out * a.scale_out);
    }
    if (a.final)
#pragma unroll
        for (int i = 0; i < MAX_WIDTH; i++)
            if (c < a.value && i < a.key) a.final[base + (TRANSPOSED ? c * a.key + i : i * a.value + c)] = state[i];
}

// Derivative by the decay's logarithm, of one row and head: the state's own derivative goes along with it.
template <typename T> __global__ __launch_bounds__(MAX_WIDTH) void slope_kernel(Walk a, Part d_out, const float* d_final, float* partial) {
    __shared__ float q[MAX_WIDTH], k[MAX_WIDTH], sum[2];
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, c = threadIdx.x;
    const float decay = expf(a.log_decay[h]);
    const size_t base = ((size_t)b * a.heads + h) * a.key * a.value;
    float state[MAX_WIDTH], slope[MAX_WIDTH];
#pragma unroll
    for (int i = 0; i < MAX_WIDTH; i++) { state[i] = a.initial && c < a.value && i < a.key ? a.initial[base + i * a.value + c] : 0.0f; slope[i] = 0.0f; }
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.steps) : a.steps;
    float total = 0.0f;
    for (int t = 0; t < length; t++) {
        __syncthreads();
        q[c] = c < a.key ? (float)at<T>(a.q, t, b, h)[c] : 0.0f;
        k[c] = c < a.key ? (float)at<T>(a.k, t, b, h)[c] : 0.0f;
        const float v = c < a.value ? (float)at<T>(a.v, t, b, h)[c] : 0.0f, d = c < a.value ? (float)at<T>(d_out, t, b, h)[c] * a.scale_out : 0.0f;
        __syncthreads();
        const bool forget = a.reset && a.reset[(size_t)t * a.batch + b];
        float out = 0.0f;
#pragma unroll
        for (int i = 0; i < MAX_WIDTH; i++) {
            slope[i] = forget ? 0.0f : decay * (slope[i] + state[i]);
            state[i] = fmaf(k[i], v, forget ? 0.0f : state[i] * decay);
            out = fmaf(q[i], slope[i], out);
        }
        total = fmaf(out, d, total);
    }
    if (d_final)
#pragma unroll
        for (int i = 0; i < MAX_WIDTH; i++)
            if (c < a.value && i < a.key) total = fmaf(d_final[base + i * a.value + c], slope[i], total);
    total = rlt_wave_sum(total);
    if ((c & 63) == 0) sum[c >> 6] = total;
    __syncthreads();
    if (c == 0) partial[(size_t)b * a.heads + h] = sum[0] + sum[1];
}

// sums over the rows of a batch, in their order
__global__ __launch_bounds__(64) void decay_sum_kernel(const float* __restrict__ partial, int batch, int heads, float* __restrict__ out, int accumulate) {
    const int h = blockIdx.x;
    float s = 0.0f;
    for (int b = threadIdx.x; b < batch; b += 64) s += partial[(size_t)b * heads + h];
    s = rlt_wave_sum(s);
    if (threadIdx.x == 0) out[h] = accumulate ? out[h] + s : s;
}

// gradients of shared keys and values: the sum over the heads that read them
template <typename T> __global__ __launch_bounds__(128) void head_sum_kernel(const float* __restrict__ parts, Part out, int steps, int batch, int kv_heads, int group, int width) {
    const size_t total = (size_t)steps * batch * kv_heads * width;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const int c = (int)(i % width);
        const size_t r = i / width;
        const int h = (int)(r % kv_heads);
        const size_t tb = r / kv_heads;
        float s = 0.0f;
        for (int g = 0; g < group; g++) s += parts[((tb * kv_heads + h) * group + g) * width + c];
        at<T>(out, (int)(tb / batch), (int)(tb % batch), h)[c] = (T)s;
    }
}

// One step: a workgroup per row and head
template <typename T> __global__ __launch_bounds__(128) void step_kernel(Walk a) {
    __shared__ float q[MAX_WIDTH], k[MAX_WIDTH];
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, c = threadIdx.x;
    const float decay = expf(a.log_decay[h]);
    const size_t base = ((size_t)b * a.heads + h) * a.key * a.value;
    q[c] = c < a.key ? (float)at<T>(a.q, 0, b, h)[c] : 0.0f;
    k[c] = c < a.key ? (float)at<T>(a.k, 0, b, h)[c] : 0.0f;
    const float v = c < a.value ? (float)at<T>(a.v, 0, b, h)[c] : 0.0f;
    __syncthreads();
    const bool forget = a.reset && a.reset[b];
    if (c >= a.value) return;
    float out = 0.0f;
    for (int i = 0; i < a.key; i++) {
        const float s = fmaf(k[i], v, forget ? 0.0f : a.initial[base + i * a.value + c] * decay);
        a.final[base + i * a.value + c] = s;
        out = fmaf(q[i], s, out);
    }
    at<T>(a.out, 0, b, h)[c] = (T)(out * a.scale_out);
}

Part part(const rlt_head_view* v, int group) { return Part{v->data, v->step_stride, v->row_stride, v->head_stride, group}; }
bool described(const rlt_linear_attention* p) {
    return p && (p->type == RLT_TYPE_F32 || p->type == RLT_TYPE_BF16) && p->batch > 0 && p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->key_dim > 0 && p->value_dim > 0;
}
bool supported(const rlt_linear_attention* p) { return p->key_dim <= MAX_WIDTH && p->value_dim <= MAX_WIDTH && (int64_t)p->batch * p->heads <= INT32_MAX; }
bool given(const rlt_head_view* v) { return v && v->data; }

Walk walk_of(const rlt_linear_attention* p, const uint8_t* reset, const int32_t* lengths, int steps) {
    Walk a{};
    a.log_decay = p->log_decay; a.reset = reset; a.lengths = lengths; a.scale_out = a.scale_added = 1.0f;
    a.batch = p->batch; a.heads = p->heads; a.steps = steps; a.key = p->key_dim; a.value = p->value_dim;
    return a;
}
template <typename T, typename O, bool REVERSE, bool TRANSPOSED> void walk(rlt_rocm_device* device, const Walk& a) {
    hipLaunchKernelGGL((walk_kernel<T, O, REVERSE, TRANSPOSED>), dim3((unsigned)a.heads * a.batch), dim3(MAX_WIDTH), 0, device->stream, a);
}

template <typename T> int backward(rlt_rocm_device* device, const rlt_linear_attention* p, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v, const rlt_head_view* d_output,
                                   const rlt_head_view* d_q, const rlt_head_view* d_k, const rlt_head_view* d_v, const float* initial_state, const float* d_final_state, float* d_initial_state,
                                   float* d_log_decay, int accumulate, const uint8_t* reset, const int32_t* lengths, int steps, void* workspace) {
    const int group = p->heads / p->kv_heads;
    const Part Q = part(q, 1), K = part(k, group), V = part(v, group), D = part(d_output, 1);
    float* partial = (float*)workspace;
    float* shared = partial + (((size_t)p->batch * p->heads + 63) / 64) * 64;
    Walk a = walk_of(p, reset, lengths, steps);      // d_q = scale * d_output S^T: the state, read across
    a.q = D; a.k = V; a.v = K; a.out = part(d_q, 1); a.key = p->value_dim; a.value = p->key_dim; a.scale_out = p->scale; a.initial = initial_state;
    walk<T, T, false, true>(device, a);
    auto reverse = [&](const Part& reader, const Part& x, const Part& y, const rlt_head_view* to, bool transposed) {
        Walk r = walk_of(p, reset, lengths, steps);
        const int width = transposed ? p->key_dim : p->value_dim;
        r.q = reader; r.k = x; r.v = y; r.scale_added = p->scale; r.initial = d_final_state; r.key = transposed ? p->value_dim : p->key_dim; r.value = width;
        if (!transposed) r.final = d_initial_state;
        r.out = group == 1 ? part(to, 1) : Part{shared, (int64_t)p->batch * p->heads * width, (int64_t)p->heads * width, width, 1};
        if (group == 1) { if (transposed) walk<T, T, true, true>(device, r); else walk<T, T, true, false>(device, r); }
        else {
            if (transposed) walk<T, float, true, true>(device, r); else walk<T, float, true, false>(device, r);
            hipLaunchKernelGGL((head_sum_kernel<T>), dim3(2048), dim3(128), 0, device->stream, shared, part(to, 1), steps, p->batch, p->kv_heads, group, width);
        }
    };
    reverse(K, Q, D, d_v, false);
    reverse(V, D, Q, d_k, true);
    if (d_log_decay) {
        Walk s = walk_of(p, reset, lengths, steps);
        s.q = Q; s.k = K; s.v = V; s.initial = initial_state; s.scale_out = p->scale;
        hipLaunchKernelGGL((slope_kernel<T>), dim3((unsigned)p->heads * p->batch), dim3(MAX_WIDTH), 0, device->stream, s, D, d_final_state, partial);
        hipLaunchKernelGGL(decay_sum_kernel, dim3(p->heads), dim3(64), 0, device->stream, partial, p->batch, p->heads, d_log_decay, accumulate);
    }
    return rlt_launch_status(device);
}

}  // namespace

extern "C" {

size_t rlt_rocm_linear_attention_workspace_bytes(const rlt_linear_attention* layer, int steps, int backward) {
    if (!described(layer) || steps <= 0 || !backward) return 0;
    const size_t partial = (((size_t)layer->batch * layer->heads + 63) / 64) * 64;
    const size_t shared = layer->heads == layer->kv_heads ? 0 : (size_t)steps * layer->batch * layer->heads * (layer->key_dim > layer->value_dim ? layer->key_dim : layer->value_dim);
    return (partial + shared) * sizeof(float);
}

int rlt_rocm_linear_attention_forward(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                      const rlt_head_view* output, const float* initial_state, float* final_state, const uint8_t* reset, const int32_t* lengths, int steps,
                                      void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && steps > 0 && given(q) && given(k) && given(v) && given(output));
    const size_t need = rlt_rocm_linear_attention_workspace_bytes(layer, steps, 0);
    RLT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need));
    if (!supported(layer)) return RLT_E_UNSUPPORTED;
    const int group = layer->heads / layer->kv_heads;
    Walk a = walk_of(layer, reset, lengths, steps);
    a.q = part(q, 1); a.k = part(k, group); a.v = part(v, group); a.out = part(output, 1); a.scale_out = layer->scale; a.initial = initial_state; a.final = final_state;
    if (layer->type == RLT_TYPE_F32) walk<float, float, false, false>(device, a); else walk<rlt_bf16, rlt_bf16, false, false>(device, a);
    return rlt_launch_status(device);
}

int rlt_rocm_linear_attention_backward(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                       const rlt_head_view* d_output, const rlt_head_view* d_q, const rlt_head_view* d_k, const rlt_head_view* d_v,
                                       const float* initial_state, const float* d_final_state, float* d_initial_state, float* d_log_decay, int accumulate,
                                       const uint8_t* reset, const int32_t* lengths, int steps, void* workspace, size_t workspace_bytes) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && steps > 0 && given(q) && given(k) && given(v) && given(d_output) && given(d_q) && given(d_k) && given(d_v));
    const size_t need = rlt_rocm_linear_attention_workspace_bytes(layer, steps, 1);
    RLT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need));
    if (!supported(layer)) return RLT_E_UNSUPPORTED;
    return layer->type == RLT_TYPE_F32 ? backward<float>(device, layer, q, k, v, d_output, d_q, d_k, d_v, initial_state, d_final_state, d_initial_state, d_log_decay, accumulate, reset, lengths, steps, workspace)
                                       : backward<rlt_bf16>(device, layer, q, k, v, d_output, d_q, d_k, d_v, initial_state, d_final_state, d_initial_state, d_log_decay, accumulate, reset, lengths, steps, workspace);
}

int rlt_rocm_linear_attention_step(rlt_rocm_device* device, const rlt_linear_attention* layer, const rlt_head_view* q, const rlt_head_view* k, const rlt_head_view* v,
                                   const rlt_head_view* output, const float* state, float* next_state, const uint8_t* reset) {
    if (!device) return RLT_E_NOT_INITIALISED;
    RLT_REQUIRE(described(layer) && layer->log_decay && given(q) && given(k) && given(v) && given(output) && state && next_state);
    if (!supported(layer)) return RLT_E_UNSUPPORTED;
    const int group = layer->heads / layer->kv_heads;
    Walk a = walk_of(layer, reset, nullptr, 1);
    a.q = part(q, 1); a.k = part(k, group); a.v = part(v, group); a.out = part(output, 1); a.scale_out = layer->scale; a.initial = state; a.final = next_state;
    if (layer->type == RLT_TYPE_F32) hipLaunchKernelGGL((step_kernel<float>), dim3((unsigned)a.heads * a.batch), dim3(MAX_WIDTH), 0, device->stream, a);
    else hipLaunchKernelGGL((step_kernel<rlt_bf16>), dim3((unsigned)a.heads * a.batch), dim3(MAX_WIDTH), 0, device->stream, a);
    return rlt_launch_status(device);
}

}  // extern "C"
