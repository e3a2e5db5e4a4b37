// Penalties for repeated tokens, biases and grammar masks on the logits of a
// batch, and the greedy id of each row (qwn_hip_ext_logits_process_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_types.h"

#include <algorithm>

namespace {

using namespace qwn;

constexpr int kThreads = 256;
constexpr uint32_t kSlice = 2048;          // tokens of the vocabulary a workgroup takes
// of a token: in the history, with a bias, with several; the bits below count
// the generated ones
constexpr uint32_t kSeen = 1u << 31, kBias = 1u << 30, kBiases = 1u << 29;
constexpr uint32_t kMostHistory = kBiases - 1;
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

// Four entries of a list from i on, `none` past its end.
template <typename E>
__device__ __forceinline__ Vec<E, 4> load_entries(const E *list, uint32_t i, uint32_t to, E none) {
    if (i + 4 <= to) return load_vec<E, 4>(list + i);
    Vec<E, 4> t;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) t.v[e] = i + e < to ? list[i + e] : none;
    return t;
}

// The biases of a token that has several, if `index` is its first entry: the
// wave reads the list 64 entries a step and adds them in its order.
__device__ __forceinline__ void add_biases(const LogitsArgs &a, uint32_t b0, uint32_t b1, uint32_t token, uint32_t index,
                                           double *biases, uint32_t v0) {
    const uint32_t lane = threadIdx.x % kWaveSize;
    double sum = 0.0;
    bool any = false;
    for (uint32_t j0 = b0; j0 < b1; j0 += kWaveSize) {
        const uint32_t j = j0 + lane;
        const bool mine = j < b1 && static_cast<uint32_t>(a.bias_tokens[j]) == token;
        const float v = mine ? a.bias_values[j] : 0.0f;
        for (uint64_t left = __ballot(mine); left; left &= left - 1) {
            const int l = __ffsll(static_cast<unsigned long long>(left)) - 1;
            if (!any && j0 + l != index) return;  // another entry is the first
            any = true;
            sum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
        }
    }
    if (lane == 0) biases[token - v0] = sum;
}

// grid (slices of the vocabulary, rows).  The beginnings of the row's lists (1024
// tokens and biases; 4096 tokens are no faster, 26 us for 24) and a workgroup's
// slice of the logits are loaded into registers, in this order; while the logits come, the history is
// counted and the biases are found among the slice's tokens in LDS (integer adds
// and ors: their order does not matter).  Every slice reads the row's lists, from L2.  Touched
// logits are computed in 64 bits and rounded once.
template <typename T>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr int N = kSlice / (kThreads * VEC);  // vectors of a thread
    __shared__ __attribute__((aligned(16))) uint32_t counts[kSlice];
    __shared__ double biases[kSlice];             // where kBias is set
    __shared__ uint64_t red[kThreads / kWaveSize];
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * kSlice, v1 = min(a.vocab, v0 + kSlice), tid = threadIdx.x;
    const T *in = static_cast<const T *>(a.logits) + static_cast<size_t>(r) * a.in_stride;
    T *out = static_cast<T *>(a.out) + static_cast<size_t>(r) * a.out_stride;
    uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.history) range_of(a.history_starts, r, a.history_capacity, h0, h1);
    if (a.bias_tokens) range_of(a.bias_starts, r, a.bias_capacity, b0, b1);
    const int32_t m = a.mask_index ? a.mask_index[r] : static_cast<int32_t>(r);
    const uint32_t *mask = a.mask && m >= 0 && static_cast<uint32_t>(m) < a.mask_rows ? a.mask + static_cast<size_t>(m) * a.mask_stride : nullptr;
    const uint32_t prompt = a.prompt_counts ? static_cast<uint32_t>(max(0, a.prompt_counts[r])) : 0u;
    const double rep = a.repetition ? a.repetition[r] : 1.0f, pres = a.presence ? a.presence[r] : 0.0f,
                 freq = a.frequency ? a.frequency[r] : 0.0f;
    const bool lists = h1 > h0 || b1 > b0;
    Vec<int32_t, 4> hist, tokens;
    Vec<float, 4> values;
    if (lists) {
        tokens = load_entries(a.bias_tokens, b0 + 4 * tid, b1, -1);
        values = load_entries(a.bias_values, b0 + 4 * tid, b1, 0.0f);
        hist = load_entries(a.history, h0 + 4 * tid, h1, -1);
    }
    Vec<T, VEC> x[N];
    uint32_t allowed[N];  // the words that hold a vector's tokens: VEC divides 32
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t v = v0 + (tid + kThreads * k) * VEC;
        allowed[k] = mask && v < v1 ? mask[v / 32] : 0xffffffffu;
        if (v + VEC <= v1) x[k] = load_vec<T, VEC>(in + v);
    }
    if (lists) {
        for (uint32_t i = tid; i < kSlice / 4; i += kThreads) reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0, 0, 0, 0);
        lds_barrier();
        auto count = [&](uint32_t i, const Vec<int32_t, 4> &t4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t t = static_cast<uint32_t>(t4.v[e]);
                if (t < v0 || t >= v1) continue;
                atomicOr(&counts[t - v0], kSeen);
                if (i + e - h0 >= prompt) atomicAdd(&counts[t - v0], 1u);
            }
        };
        auto find = [&](const Vec<int32_t, 4> &t4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t t = static_cast<uint32_t>(t4.v[e]);
                if (t < v0 || t >= v1) continue;
                if (atomicOr(&counts[t - v0], kBias) & kBias) atomicOr(&counts[t - v0], kBiases);
            }
        };
        // what comes once is put down; what comes several times is added up by the
        // wave that has the token's first entry, in the list's order
        auto put = [&](uint32_t i, const Vec<int32_t, 4> &t4, const Vec<float, 4> &v4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t t = static_cast<uint32_t>(t4.v[e]);
                const bool here = t >= v0 && t < v1, many = here && (counts[t - v0] & kBiases);
                if (here && !many) biases[t - v0] = v4.v[e];
                for (uint64_t left = __ballot(many); left; left &= left - 1) {
                    const int lane = __ffsll(static_cast<unsigned long long>(left)) - 1;
                    add_biases(a, b0, b1, __builtin_amdgcn_readlane(static_cast<int>(t), lane),
                               __builtin_amdgcn_readlane(static_cast<int>(i + e), lane), biases, v0);
                }
            }
        };
        find(tokens);
        for (uint32_t i = b0 + 4 * (tid + kThreads); i < b1; i += 4 * kThreads) find(load_entries(a.bias_tokens, i, b1, -1));
        count(h0 + 4 * tid, hist);
        for (uint32_t i = h0 + 4 * (tid + kThreads); i < h1; i += 4 * kThreads) count(i, load_entries(a.history, i, h1, -1));
        lds_barrier();
        if (b1 > b0) {
            put(b0 + 4 * tid, tokens, values);
            for (uint32_t i0 = b0 + 4 * kThreads; i0 < b1; i0 += 4 * kThreads) {
                const uint32_t i = i0 + 4 * tid;
                put(i, load_entries(a.bias_tokens, i, b1, -1), load_entries(a.bias_values, i, b1, 0.0f));
            }
            lds_barrier();
        }
    }
    const double inv_rep = 1.0 / rep;
    // the value of token v0 + k, with the row's lists' `n`: x after them
    auto touched = [&](float x, uint32_t k, uint32_t n) {
        double y = x;
        if (n & kSeen) y *= y > 0.0 ? inv_rep : rep;
        const uint32_t made = n & kMostHistory;
        if (made) y = y - static_cast<double>(made) * freq - pres;
        if (n & kBias) y += biases[k];
        return from_float<T>(static_cast<float>(y));
    };
    float best = -INFINITY;  // of the thread's tokens, in ascending order: NaN and -inf never win
    uint32_t best_at = kNone;
    auto finish = [&](T y, uint32_t v, uint32_t word) {
        if (!((word >> (v % 32)) & 1u)) y = from_float<T>(-INFINITY);
        const float f = to_float(y);
        if (f > best) best = f, best_at = v;
        return y;
    };
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t v = v0 + (tid + kThreads * k) * VEC;
        if (v + VEC <= v1) {
            if (lists) {
#pragma unroll
                for (int i0 = 0; i0 < VEC; i0 += 4) {
                    const uint4 n = *reinterpret_cast<const uint4 *>(counts + (v - v0 + i0));
                    if (n.x | n.y | n.z | n.w) {
                        const uint32_t n4[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n4[i]) x[k].v[i0 + i] = touched(to_float(x[k].v[i0 + i]), v - v0 + i0 + i, n4[i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[k].v[i] = finish(x[k].v[i], v + i, allowed[k]);
            store_vec<T, VEC>(out + v, x[k]);
        } else {
            for (uint32_t i = v; i < v1; ++i) {
                T y = in[i];
                if (lists && counts[i - v0]) y = touched(to_float(y), i - v0, counts[i - v0]);
                out[i] = finish(y, i, allowed[k]);
            }
        }
    }
    if (!a.keys) return;
    const uint64_t key = wave_max_key(greedy_key(best, best_at));
    if (tid % kWaveSize == 0) red[tid / kWaveSize] = key;
    lds_barrier();
    if (tid == 0) {
        uint64_t top = red[0];
        for (int w = 1; w < kThreads / kWaveSize; ++w) top = max(top, red[w]);
        a.keys[static_cast<size_t>(r) * a.parts + blockIdx.x] = top;
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
    if ((r->history && (!r->history_starts || r->history_capacity > kMostHistory)) ||
        (r->bias_tokens && (!r->bias_values || !r->bias_starts || r->bias_capacity > 0x7fffffffu)) ||
        (r->mask && (a.mask_stride < (r->vocab + 31) / 32 || r->mask_rows == 0 || (!r->mask_index && r->mask_rows < r->rows))) ||
        (r->ids && (!r->workspace || (reinterpret_cast<uintptr_t>(r->workspace) & 7u)))) {
        set_error("invalid logits request: a history, biases, mask or workspace without what it needs");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t size = dtype_bytes(r->dtype), rows = r->rows;
    const Rows in = row_block(r->logits, rows, r->vocab, a.in_stride, size), out = row_block(r->out, rows, r->vocab, a.out_stride, size);
    const auto list = [](bool used, const void *p, uint64_t n) { return list_of_bytes(used ? p : nullptr, 4 * n); };
    const bool history = r->history, biases = r->bias_tokens;
    const Rows ids = list(true, r->ids, rows),
               work = list_of_bytes(r->ids ? r->workspace : nullptr, qwn_hip_ext_logits_workspace_bytes(r->rows, r->vocab)),
               mask = row_block(r->mask, r->mask_rows, (r->vocab + 31) / 32, a.mask_stride, 4);
    const auto written = [&](const Rows &w) {
        return overlaps_any(w, {list(true, r->history, r->history_capacity), list(history, r->history_starts, rows + 1),
                                list(true, r->prompt_counts, rows), list(true, r->repetition, rows), list(true, r->presence, rows),
                                list(true, r->frequency, rows), list(true, r->bias_tokens, r->bias_capacity),
                                list(biases, r->bias_values, r->bias_capacity), list(biases, r->bias_starts, rows + 1), mask,
                                list(r->mask, r->mask_index, rows)});
    };
    if ((!in_place(out, in) && overlap(out, in)) || overlaps_any(ids, {in, out, work}) || overlaps_any(work, {in, out}) || written(out) ||
        written(ids) || written(work)) {
        set_error("logits request: an output or the workspace overlaps an input or another output");
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
