// Rotary positions with several axes on queries and keys, each head normed
// first where weights are given (qwn_hip_ext_rotary_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace qwn;

constexpr uint32_t kPairsMost = 128;
constexpr uint32_t kTokensMost = 4;     // of a workgroup
constexpr uint32_t kThreadsMost = 512;

struct RotaryArgs {
    const void *in[2];       // queries, keys
    void *out[2];
    const float *norm[2];
    const int32_t *positions;
    uint32_t heads[2], in_stride[2], out_stride[2];
    uint32_t tokens, head_dim, rope, position_stride, lanes;  // lanes: of a head, a power of two
    float eps;
    uint8_t axis[kPairsMost];
    double freq[kPairsMost];
};

// N elements [c, c + N) of a row, zeros from `end` on.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_part(const T *row, uint32_t c, uint32_t end) {
    constexpr int VEC = 16 / sizeof(T);
    Vec<T, N> x;
    if (c + N <= end) {
#pragma unroll
        for (int h = 0; h < N; h += VEC) {
            const Vec<T, VEC> v = load_vec<T, VEC>(row + c + h);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x.v[h + i] = v.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x.v[i] = c + i < end ? row[c + i] : from_float<T>(0.0f);
    }
    return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_part(T *row, uint32_t c, uint32_t end, const double y[N]) {
    constexpr int VEC = 16 / sizeof(T);
    if (c + N <= end) {
#pragma unroll
        for (int h = 0; h < N; h += VEC) {
            Vec<T, VEC> v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v.v[i] = from_float<T>(static_cast<float>(y[h + i]));
            store_vec<T, VEC>(row + c + h, v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < end) row[c + i] = from_float<T>(static_cast<float>(y[i]));
    }
}

// A task is 8 pairs of a head (both channels of a pair in one thread: results
// may be in place), or 16 of the channels behind the rotated ones; a head's
// tasks lie in `lanes` lanes next to each other, which add up its squares.  A
// workgroup takes up to 4 tokens, whose angles are computed once, in 64 bits (at
// position 100000 an fp32 angle would be off by hundredths), while the first
// loads are in flight.  64-bit arithmetic runs at the fp32 rate here and the bytes
// bound the pass, so values are rounded once.
template <typename T>
__global__ __launch_bounds__(kThreadsMost) void rotary_kernel(RotaryArgs a, uint32_t per_group) {
    __shared__ double2 cs[kTokensMost][kPairsMost];
    const uint32_t half = a.rope / 2, pair_tasks = (half + 7) / 8, D = a.head_dim;
    const uint32_t heads = a.heads[0] + a.heads[1];
    const uint32_t token0 = blockIdx.x * per_group, tokens = min(per_group, a.tokens - token0);
    const uint32_t tasks = tokens * heads * a.lanes, nt = blockDim.x;
    struct Task {
        uint32_t token, head, kind, lane;
    };
    auto task_of = [&](uint32_t i) {
        Task t;
        t.lane = i % a.lanes;
        const uint32_t j = i / a.lanes;
        t.token = j / heads;
        t.head = j % heads;
        t.kind = t.head >= a.heads[0];
        if (t.kind) t.head -= a.heads[0];
        return t;
    };
    // the 16 channels of a task: the pairs' first and second ones, or one run of channels in two halves
    auto first_of = [&](const Task &t) { return t.lane < pair_tasks ? t.lane * 8 : a.rope + (t.lane - pair_tasks) * 16; };
    auto load = [&](uint32_t i, Vec<T, 8> &x, Vec<T, 8> &y) {
        const Task t = task_of(i);
        const T *row = static_cast<const T *>(a.in[t.kind]) + static_cast<size_t>(token0 + t.token) * a.in_stride[t.kind] +
                       static_cast<size_t>(t.head) * D;
        const uint32_t c = first_of(t);
        if (t.lane < pair_tasks) {
            x = load_part<T, 8>(row, c, half);
            y = load_part<T, 8>(row + half, c, half);
        } else {
            x = load_part<T, 8>(row, c, D);
            y = load_part<T, 8>(row, c + 8, D);
        }
    };
    Vec<T, 8> x, y;
    if (threadIdx.x < tasks) load(threadIdx.x, x, y);
    for (uint32_t i = threadIdx.x; i < tokens * half; i += nt) {
        const uint32_t t = i / half, f = i % half;
        const double p = a.positions[static_cast<size_t>(a.axis[f]) * a.position_stride + token0 + t];
        double2 v;
        sincos(p * a.freq[f], &v.y, &v.x);
        cs[t][f] = v;
    }
    lds_barrier();
    // whole waves go on, as lanes exchange
    for (uint32_t i0 = 0; i0 < tasks; i0 += nt) {
        const uint32_t i = i0 + threadIdx.x;
        if (i0 > 0 && i < tasks) load(i, x, y);
        const Task t = task_of(min(i, tasks - 1));
        const bool pair = t.lane < pair_tasks, real = i < tasks;
        const uint32_t c = first_of(t);
        double u[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = to_float(x.v[e]), v[e] = to_float(y.v[e]);
        if (a.norm[0] || a.norm[1]) {
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += u[e] * u[e] + v[e] * v[e];
            for (uint32_t off = 1; off < a.lanes; off <<= 1) sum += __shfl_xor(sum, static_cast<int>(off));
            if (const float *w = a.norm[t.kind]) {
                const double inv = 1.0 / sqrt(sum / static_cast<double>(D) + static_cast<double>(a.eps));
                const Vec<float, 8> wu = load_part<float, 8>(w, c, pair ? half : D);
                const Vec<float, 8> wv = pair ? load_part<float, 8>(w + half, c, half) : load_part<float, 8>(w, c + 8, D);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] *= inv * wu.v[e], v[e] *= inv * wv.v[e];
            }
        }
        if (!real) continue;
        T *row = static_cast<T *>(a.out[t.kind]) + static_cast<size_t>(token0 + t.token) * a.out_stride[t.kind] +
                 static_cast<size_t>(t.head) * D;
        if (pair) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double2 r = cs[t.token][min(c + e, half - 1)];
                const double p = u[e] * r.x - v[e] * r.y;
                v[e] = u[e] * r.y + v[e] * r.x;
                u[e] = p;
            }
            store_part<T, 8>(row, c, half, u);
            store_part<T, 8>(row + half, c, half, v);
        } else {
            store_part<T, 8>(row, c, D, u);
            store_part<T, 8>(row, c + 8, D, v);
        }
    }
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API int qwn_hip_ext_rotary_device(QwnCudaContextHandle *handle, const QwnHipRotaryRequest *r, void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || !r || !header_ok(*r) || r->tokens == 0 || r->tokens > 0x7fffffffu || r->dtype > QWN_HIP_DTYPE_BF16 ||
        (r->query_heads == 0 && r->key_heads == 0) || r->query_heads > 65535 || r->key_heads > 65535 || r->head_dim == 0 ||
        (r->query_heads && (!r->query || !r->query_out)) || (r->key_heads && (!r->key || !r->key_out)) ||
        (r->rope_dims && !r->positions)) {
        set_error("invalid rotary request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (r->head_dim > 256 || r->rope_dims % 2 || r->rope_dims > r->head_dim ||
        (r->rope_dims && !(r->rope_theta > 0.0f && std::isfinite(r->rope_theta)))) {
        set_error("unsupported rotary request: head_dim %u, rope_dims %u", r->head_dim, r->rope_dims);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    RotaryArgs a{};
    const uint32_t half = r->rope_dims / 2;
    uint64_t pairs = 0, axes = 0;
    for (uint32_t x = 0; x < QWN_HIP_ROTARY_AXES; ++x) {
        pairs += r->sections[x];
        if (r->sections[x]) axes = x + 1;
    }
    a.position_stride = stride_or(r->position_stride, r->tokens);
    if (pairs != half || a.position_stride < r->tokens) {
        set_error("invalid rotary request: the axes' sections are not rope_dims / 2 pairs, or positions are too few");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const void *in[2] = {r->query_heads ? r->query : nullptr, r->key_heads ? r->key : nullptr};
    void *out[2] = {r->query_heads ? r->query_out : nullptr, r->key_heads ? r->key_out : nullptr};
    const float *norm[2] = {r->query_heads ? r->query_norm : nullptr, r->key_heads ? r->key_norm : nullptr};
    const uint32_t heads[2] = {r->query_heads, r->key_heads};
    const uint32_t strides[2] = {r->query_stride, r->key_stride}, out_strides[2] = {r->query_out_stride, r->key_out_stride};
    const uint64_t size = dtype_bytes(r->dtype), tokens = r->tokens;
    Rows from[2], to[2];
    for (int k = 0; k < 2; ++k) {
        const uint32_t channels = heads[k] * r->head_dim;
        a.in[k] = in[k];
        a.out[k] = out[k];
        a.norm[k] = norm[k];
        a.heads[k] = heads[k];
        a.in_stride[k] = stride_or(strides[k], channels);
        a.out_stride[k] = stride_or(out_strides[k], channels);
        if (a.in_stride[k] < channels || a.out_stride[k] < channels || (in[k] && in[k] == out[k] && a.in_stride[k] != a.out_stride[k])) {
            set_error("rotary request: a row stride is shorter than its row, or differs in place");
            return QWN_CUDA_STATUS_INVALID_ARGUMENT;
        }
        from[k] = row_block(in[k], tokens, channels, a.in_stride[k], size);
        to[k] = row_block(out[k], tokens, channels, a.out_stride[k], size);
    }
    const Rows positions = row_block(half ? r->positions : nullptr, axes, tokens, a.position_stride, 4);
    for (int k = 0; k < 2; ++k) {
        if ((!in_place(to[k], from[k]) && overlap(to[k], from[k])) ||
            overlaps_any(to[k], {from[1 - k], to[1 - k], positions, list_of_bytes(norm[0], 4ull * r->head_dim),
                                 list_of_bytes(norm[1], 4ull * r->head_dim)})) {
            set_error("rotary request: an output overlaps an input or the other output");
            return QWN_CUDA_STATUS_INVALID_ARGUMENT;
        }
    }
    // pairs to axes: a section after the other, or in turn past those that have theirs
    uint32_t left[QWN_HIP_ROTARY_AXES];
    std::copy(r->sections, r->sections + QWN_HIP_ROTARY_AXES, left);
    for (uint32_t i = 0, x = 0; i < half; ++i) {
        while (left[x] == 0) x = (x + 1) % QWN_HIP_ROTARY_AXES;
        a.axis[i] = static_cast<uint8_t>(x);
        --left[x];
        if (r->in_turn) x = (x + 1) % QWN_HIP_ROTARY_AXES;
        a.freq[i] = std::pow(static_cast<double>(r->rope_theta), -2.0 * i / static_cast<double>(r->rope_dims));
    }
    a.positions = r->positions;
    a.tokens = r->tokens;
    a.head_dim = r->head_dim;
    a.rope = r->rope_dims;
    a.eps = r->eps;
    const uint32_t lanes = (half + 7) / 8 + (r->head_dim - r->rope_dims + 15) / 16;  // at most 17
    for (a.lanes = 1; a.lanes < lanes;) a.lanes *= 2;
    // a token of a workgroup, or, where they fill the GPU all the same, 4
    const uint32_t per_group = r->tokens >= 1024 * kTokensMost ? kTokensMost : 1;
    const uint64_t tasks = static_cast<uint64_t>(heads[0] + heads[1]) * a.lanes * per_group;
    const uint32_t threads = static_cast<uint32_t>(std::min<uint64_t>(kThreadsMost, (tasks + kWaveSize - 1) / kWaveSize * kWaveSize));
    const dim3 grid((r->tokens + per_group - 1) / per_group);
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("rotary device", device.error());
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    if (r->dtype == QWN_HIP_DTYPE_F32) {
        hipLaunchKernelGGL(rotary_kernel<float>, grid, dim3(threads), 0, s, a, per_group);
    } else if (r->dtype == QWN_HIP_DTYPE_F16) {
        hipLaunchKernelGGL(rotary_kernel<f16>, grid, dim3(threads), 0, s, a, per_group);
    } else {
        hipLaunchKernelGGL(rotary_kernel<bf16>, grid, dim3(threads), 0, s, a, per_group);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("rotary launch", e);
}

}  // extern "C"
