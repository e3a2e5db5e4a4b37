// Penalties for repeated tokens, biases and grammar masks on the logits of a
// batch, and the greedy id of each row (qwn_hip_ext_logits_process_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_types.h"

#include <algorithm>

namespace {

using namespace qwn;

constexpr int kThreads = 256;
constexpr uint32_t kSlice = 4096;          // tokens of the vocabulary a workgroup takes
constexpr uint32_t kSeen = 0x80000000u;    // in the history; the bits below count the generated ones
constexpr uint32_t kNone = 0xffffffffu;

struct LogitsArgs {
    const void *logits;
    void *out;
    const int32_t *history, *history_starts, *prompt_counts;
    const float *repetition, *presence, *frequency;
    const int32_t *bias_tokens, *bias_starts;
    const float *bias_values;
    const uint32_t *mask;
    const int32_t *mask_index;
    uint64_t *keys;  // [rows][parts], or null
    uint32_t vocab, in_stride, out_stride, history_capacity, bias_capacity, mask_rows, mask_stride, parts;
};

// Largest value first, then the smaller token; NaN and -inf never win.
__device__ __forceinline__ uint64_t greedy_key(float v, uint32_t token) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 is 0
    const uint32_t ord = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<uint64_t>(ord) << 32) | (kNone - token);
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
    for (int off = kWaveSize / 2; off > 0; off >>= 1) key = max(key, static_cast<uint64_t>(__shfl_xor(key, off)));
    return key;
}

// A list's part of row r, none where its ends do not lie in the list.
__device__ __forceinline__ void range_of(const int32_t *starts, uint32_t r, uint32_t capacity, uint32_t &from, uint32_t &to) {
    const int32_t a = starts[r], b = starts[r + 1];
    const bool ok = a >= 0 && b >= a && static_cast<uint32_t>(b) <= capacity;
    from = ok ? static_cast<uint32_t>(a) : 0u;
    to = ok ? static_cast<uint32_t>(b) : 0u;
}

// grid (slices of the vocabulary, rows).  A workgroup counts the row's
// history and finds its biases among its own tokens in LDS (integer adds and
// minima: their order does not matter), then passes over its slice of the
// logits once.  The row's lists are read by every slice, from L2.  Touched
// logits are computed in 64 bits and rounded once.
template <typename T>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ __attribute__((aligned(16))) uint32_t counts[kSlice];
    __shared__ __attribute__((aligned(16))) uint32_t owner[kSlice];  // the first of the token's biases in the list
    __shared__ uint32_t again[kSlice / 32];                            // tokens with more than one
    __shared__ uint64_t red[kThreads / kWaveSize];
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * kSlice, v1 = min(a.vocab, v0 + kSlice), tid = threadIdx.x;
    uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.history) range_of(a.history_starts, r, a.history_capacity, h0, h1);
    if (a.bias_tokens) range_of(a.bias_starts, r, a.bias_capacity, b0, b1);
    const bool lists = h1 > h0 || b1 > b0;
    if (lists) {
        for (uint32_t i = tid; i < kSlice / 4; i += kThreads) {
            reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0, 0, 0, 0);
            reinterpret_cast<uint4 *>(owner)[i] = make_uint4(kNone, kNone, kNone, kNone);
        }
        for (uint32_t i = tid; i < kSlice / 32; i += kThreads) again[i] = 0;
        __syncthreads();
        const int32_t prompt = a.prompt_counts ? a.prompt_counts[r] : 0;
        for (uint32_t i = h0 + tid; i < h1; i += kThreads) {
            const uint32_t t = static_cast<uint32_t>(a.history[i]);
            if (t < v0 || t >= v1) continue;
            atomicOr(&counts[t - v0], kSeen);
            if (static_cast<int32_t>(i - h0) >= prompt) atomicAdd(&counts[t - v0], 1u);
        }
        for (uint32_t i = b0 + tid; i < b1; i += kThreads) {
            const uint32_t t = static_cast<uint32_t>(a.bias_tokens[i]);
            if (t < v0 || t >= v1) continue;
            if (atomicMin(&owner[t - v0], i) != kNone) atomicOr(&again[(t - v0) / 32], 1u << ((t - v0) % 32));
        }
        __syncthreads();
    }
    const double rep = a.repetition ? a.repetition[r] : 1.0f, pres = a.presence ? a.presence[r] : 0.0f,
                 freq = a.frequency ? a.frequency[r] : 0.0f;
    const uint32_t *mask = nullptr;
    if (a.mask) {
        const int32_t m = a.mask_index ? a.mask_index[r] : static_cast<int32_t>(r);
        if (m >= 0 && static_cast<uint32_t>(m) < a.mask_rows) mask = a.mask + static_cast<size_t>(m) * a.mask_stride;
    }
    const T *in = static_cast<const T *>(a.logits) + static_cast<size_t>(r) * a.in_stride;
    T *out = static_cast<T *>(a.out) + static_cast<size_t>(r) * a.out_stride;
    // the value of token v0 + k: x, after the row's lists
    auto touched = [&](float x, uint32_t k) {
        const uint32_t n = counts[k], o = owner[k];
        if (n == 0 && o == kNone) return from_float<T>(x);
        double y = x;
        if (n & kSeen) y = y > 0.0 ? y / rep : y * rep;
        const uint32_t made = n & ~kSeen;
        if (made) y = y - static_cast<double>(made) * freq - pres;
        if (o != kNone) {
            double bias = a.bias_values[o];
            if ((again[k / 32] >> (k % 32)) & 1u)  // all of them, in the list's order
                for (uint32_t i = o + 1; i < b1; ++i)
                    if (static_cast<uint32_t>(a.bias_tokens[i]) == v0 + k) bias += a.bias_values[i];
            y += bias;
        }
        if constexpr (sizeof(T) == 4) return static_cast<float>(y);
        return from_float<T>(static_cast<float>(y));
    };
    uint64_t best = 0;
    auto one = [&](T raw, uint32_t v) {
        T y = lists ? touched(to_float(raw), v - v0) : raw;
        if (mask && !((mask[v / 32] >> (v % 32)) & 1u)) y = from_float<T>(-INFINITY);
        if (a.keys) best = max(best, greedy_key(to_float(y), v));
        return y;
    };
    for (uint32_t v = v0 + tid * VEC; v < v1; v += kThreads * VEC) {
        if (v + VEC <= v1) {
            const Vec<T, VEC> x = load_vec<T, VEC>(in + v);
            Vec<T, VEC> y;
#pragma unroll
            for (int i = 0; i < VEC; ++i) y.v[i] = one(x.v[i], v + i);
            store_vec<T, VEC>(out + v, y);
        } else {
            for (uint32_t i = v; i < v1; ++i) out[i] = one(in[i], i);
        }
    }
    if (!a.keys) return;
    best = wave_max_key(best);
    if (tid % kWaveSize == 0) red[tid / kWaveSize] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / kWaveSize; ++w) best = max(best, red[w]);
        a.keys[static_cast<size_t>(r) * a.parts + blockIdx.x] = best;
    }
}

// The winning token of each row's slices, -1 where nothing is left.
__global__ __launch_bounds__(kWaveSize) void logits_ids_kernel(const uint64_t *__restrict__ keys, uint32_t parts, int32_t *ids) {
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < parts; i += kWaveSize) best = max(best, keys[static_cast<size_t>(blockIdx.x) * parts + i]);
    best = wave_max_key(best);
    if (threadIdx.x == 0) ids[blockIdx.x] = best ? static_cast<int32_t>(kNone - static_cast<uint32_t>(best)) : -1;
}

uint32_t parts_of(uint32_t vocab) { return (vocab + kSlice - 1) / kSlice; }

template <typename T>
hipError_t launch_logits(const LogitsArgs &a, uint32_t rows, int32_t *ids, hipStream_t stream) {
    hipLaunchKernelGGL(logits_kernel<T>, dim3(a.parts, rows), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !ids) return e;
    hipLaunchKernelGGL(logits_ids_kernel, dim3(rows), dim3(kWaveSize), 0, stream, a.keys, a.parts, ids);
    return hipGetLastError();
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API uint64_t qwn_hip_ext_logits_workspace_bytes(uint32_t rows, uint32_t vocab) {
    return static_cast<uint64_t>(rows) * parts_of(vocab) * sizeof(uint64_t);
}

QWN_CUDA_ABI_API int qwn_hip_ext_logits_process_device(QwnCudaContextHandle *handle, const QwnHipLogitsRequest *r,
                                                       void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || !r || !header_ok(*r) || r->rows == 0 || r->rows > 65535 || r->vocab == 0 || r->vocab > 0x7fffffffu ||
        !r->logits || !r->out || r->dtype > QWN_HIP_DTYPE_BF16) {
        set_error("invalid logits request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    LogitsArgs a{};
    a.in_stride = stride_or(r->in_stride, r->vocab);
    a.out_stride = stride_or(r->out_stride, r->vocab);
    a.mask_stride = stride_or(r->mask_stride, (r->vocab + 31) / 32);
    if (a.in_stride < r->vocab || a.out_stride < r->vocab || (r->logits == r->out && a.in_stride != a.out_stride)) {
        set_error("logits request: a row stride is shorter than its row, or differs in place");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if ((r->history && (!r->history_starts || r->history_capacity > 0x7fffffffu)) ||
        (r->bias_tokens && (!r->bias_values || !r->bias_starts || r->bias_capacity > 0x7fffffffu)) ||
        (r->mask && (a.mask_stride < (r->vocab + 31) / 32 || r->mask_rows == 0 || (!r->mask_index && r->mask_rows < r->rows))) ||
        (r->ids && (!r->workspace || (reinterpret_cast<uintptr_t>(r->workspace) & 7u)))) {
        set_error("invalid logits request: a history, biases, mask or workspace without what it needs");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("logits device", device.error());
    a.logits = r->logits;
    a.out = r->out;
    a.history = r->history;
    a.history_starts = r->history_starts;
    a.prompt_counts = r->prompt_counts;
    a.repetition = r->repetition;
    a.presence = r->presence;
    a.frequency = r->frequency;
    a.bias_tokens = r->bias_tokens;
    a.bias_starts = r->bias_starts;
    a.bias_values = r->bias_values;
    a.mask = r->mask;
    a.mask_index = r->mask_index;
    a.keys = r->ids ? static_cast<uint64_t *>(r->workspace) : nullptr;
    a.vocab = r->vocab;
    a.history_capacity = r->history_capacity;
    a.bias_capacity = r->bias_capacity;
    a.mask_rows = r->mask_rows;
    a.parts = parts_of(r->vocab);
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_logits<float>(a, r->rows, r->ids, s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_logits<f16>(a, r->rows, r->ids, s)
                                                         : launch_logits<bf16>(a, r->rows, r->ids, s);
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("logits launch", e);
}

}  // extern "C"
