// Rotary positions with several axes on queries and keys, each head normed
// first where weights are given (qwn_hip_ext_rotary_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace qwn;

constexpr uint32_t kPairsMost = 128;
constexpr uint32_t kThreadsMost = 512;

struct RotaryArgs {
    const void *in[2];       // queries, keys
    void *out[2];
    const float *norm[2];
    const int32_t *positions;
    uint32_t heads[2], in_stride[2], out_stride[2];
    uint32_t tokens, head_dim, rope, position_stride, lanes;  // lanes: of a head, a power of two
    double eps, inv_dim;
    uint8_t axis[kPairsMost];
    double turns[kPairsMost];  // theta^(-2 i / rope_dims) / (2 pi)
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
template <typename T, int N, typename R>
__device__ __forceinline__ void store_part(T *row, uint32_t c, uint32_t end, const R y[N]) {
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

// v of the lanes next to each other added up, `lanes` (a power of two up to 32) at a
// time, to all of them.
template <int CTRL>
__device__ __forceinline__ float lane_moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double lane_moved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <typename R>
__device__ __forceinline__ R lanes_sum(R v, uint32_t lanes) {
    if (lanes > 1) v += lane_moved<0xb1>(v);   // quad_perm [1, 0, 3, 2]
    if (lanes > 2) v += lane_moved<0x4e>(v);   // quad_perm [2, 3, 0, 1]
    if (lanes > 4) v += lane_moved<0x141>(v);  // row_half_mirror: the other four
    if (lanes > 8) v += lane_moved<0x140>(v);  // row_mirror: the other eight
    if (lanes > 16) v += __shfl_xor(v, 16);
    return v;
}

// Cosine and sine of t turns: what is left of the nearest quarter, at most pi / 4, by
// Taylor's series to the 12th and 11th power (the next terms are below 2^-37).  The
// library's functions take 90 registers more, which is a third of the waves.
__device__ __forceinline__ double2 angle(double t) {
    const double quarters = rint(4.0 * t), x = (4.0 * t - quarters) * 1.57079632679489661923, y = x * x;
    const double c = 1.0 + y * (-1.0 / 2 + y * (1.0 / 24 + y * (-1.0 / 720 + y * (1.0 / 40320 + y * (-1.0 / 3628800 + y * (1.0 / 479001600))))));
    const double s = x * (1.0 + y * (-1.0 / 6 + y * (1.0 / 120 + y * (-1.0 / 5040 + y * (1.0 / 362880 + y * (-1.0 / 39916800))))));
    const int64_t q = static_cast<int64_t>(quarters);
    const double a = q & 1 ? s : c, b = q & 1 ? c : s;
    return make_double2((q + 1) & 2 ? -a : a, q & 2 ? -b : b);
}

// What fp32 rows are computed in, and 16-bit ones, whose own rounding is 2^-11 and
// more (64 bits take twice the registers and half the waves).
template <typename T>
struct Work {
    typedef float real;
    typedef float2 pair;
};
template <>
struct Work<float> {
    typedef double real;
    typedef double2 pair;
};
// A mean square of bf16 may be past fp32, or lie where its squares lose bits: such heads are
// normed in 64 bits.  f16's squares cannot be.
template <typename T>
constexpr bool kWide = std::is_same_v<T, bf16>;
__device__ __forceinline__ float root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double root(double v) { return rsqrt(v); }

// A thread takes 8 pairs of a head (both channels of a pair in one thread: results
// may be in place), or 16 of the channels behind the rotated ones, of TOKENS tokens;
// the `lanes` threads of a head, next to each other, add up its squares.
// grid (tokens, heads): all loads are issued first; while they are on their way the
// tokens' angles are computed, in 64 bits (at position 100000 an fp32 angle would be
// off by hundredths).
// Bound by HBM: 4099 tokens of 40 bf16 heads of 128 with norms, 84 MB, 20 us, 4.2 TB/s of the
// 5.1 that a large copy reaches; few tokens by a launch and two loads, one
// after the other, 2.9 us.
template <typename T, int TOKENS>
__global__ __launch_bounds__(kThreadsMost, sizeof(T) == 4 ? 3 : 4) void rotary_kernel(RotaryArgs a) {
    using R = typename Work<T>::real;
    __shared__ typename Work<T>::pair cs[TOKENS][kPairsMost];  // pair f at f % 8 * 16 + f / 8: lanes read next to each other
    const uint32_t half = a.rope / 2, pair_lanes = (half + 7) / 8, D = a.head_dim;
    const uint32_t token0 = blockIdx.x * TOKENS, x = blockIdx.y * blockDim.x + threadIdx.x;
    const uint32_t lane = x % a.lanes, h = x / a.lanes;  // lanes: a power of two
    const bool real = h < a.heads[0] + a.heads[1];
    const uint32_t kind = real && h >= a.heads[0] ? 1u : 0u, head = real ? h - (kind ? a.heads[0] : 0u) : 0u;
    const bool pair = lane < pair_lanes;
    // first and second channels of the pairs, or 8 channels and the 8 behind them
    const uint32_t c = pair ? lane * 8 : a.rope + (lane - pair_lanes) * 16, next = pair ? half : 8u, end = pair ? half : D;
    const uint32_t end2 = pair ? half : D > 8 ? D - 8 : 0u;  // of the second ones, counted from `next`
    const T *in = static_cast<const T *>(kind ? a.in[1] : a.in[0]) + static_cast<size_t>(head) * D;
    T *out = static_cast<T *>(kind ? a.out[1] : a.out[0]) + static_cast<size_t>(head) * D;
    const size_t in_stride = kind ? a.in_stride[1] : a.in_stride[0], out_stride = kind ? a.out_stride[1] : a.out_stride[0];
    const float *norm = kind ? a.norm[1] : a.norm[0];
    Vec<T, 8> u[TOKENS], v[TOKENS];
    if (real) {
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            const T *row = in + min(token0 + t, a.tokens - 1) * in_stride;
            u[t] = load_part<T, 8>(row, c, end);
            v[t] = load_part<T, 8>(row + next, c, end2);
        }
    }
    Vec<float, 8> wu, wv;
    if (real && norm) {
        wu = load_part<float, 8>(norm, c, end);
        wv = load_part<float, 8>(norm + next, c, end2);
    }
    for (uint32_t i = threadIdx.x; i < TOKENS * half; i += blockDim.x) {
        const uint32_t t = i / half, f = i % half;
        const double p = a.positions[static_cast<size_t>(a.axis[f]) * a.position_stride + min(token0 + t, a.tokens - 1)];
        const double2 r = angle(p * a.turns[f]);
        cs[t][f % 8 * 16 + f / 8] = {static_cast<R>(r.x), static_cast<R>(r.y)};
    }
    lds_barrier();
    if (!real) return;  // all the lanes of a head
    uint32_t wide = 0;  // tokens
    auto finish = [&](auto in_64) {
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            if (token0 + t >= a.tokens) break;
            if (decltype(in_64)::value && !(wide >> t & 1)) continue;
            __builtin_amdgcn_sched_barrier(0);
            R p[8], q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = to_float(u[t].v[e]), q[e] = to_float(v[t].v[e]);
            if constexpr (decltype(in_64)::value) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += static_cast<double>(p[e]) * p[e] + static_cast<double>(q[e]) * q[e];
                const double inv = root(lanes_sum(sum, a.lanes) * a.inv_dim + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = static_cast<R>(p[e] * inv * wu.v[e]), q[e] = static_cast<R>(q[e] * inv * wv.v[e]);
            } else if (norm) {
                R sum = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += p[e] * p[e] + q[e] * q[e];
                const R mean = lanes_sum(sum, a.lanes) * static_cast<R>(a.inv_dim) + static_cast<R>(a.eps), inv = root(mean);
                wide |= mean > 0x1p-80f && mean < INFINITY ? 0u : 1u << t;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] *= inv * wu.v[e], q[e] *= inv * wv.v[e];
            }
            if (pair) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const auto r = cs[t][e * 16 + lane];  // past the last pair: anything, not stored
                    const R first = p[e] * r.x - q[e] * r.y;
                    q[e] = p[e] * r.y + q[e] * r.x;
                    p[e] = first;
                }
            }
            T *row = out + (token0 + t) * out_stride;
            store_part<T, 8, R>(row, c, end, p);
            store_part<T, 8, R>(row + next, c, end2, q);
        }
    };
    finish(std::false_type{});
    if (kWide<T> && wide) finish(std::true_type{});  // again, from what was loaded (decided before: 3 to 10 % more for all)
}

// Tokens of a workgroup: more where the grid fills the GPU all the same.
constexpr uint32_t kManyTokens = 2048, kTokens = 2;
uint32_t block_of(uint64_t threads) {
    return static_cast<uint32_t>(std::min<uint64_t>(kThreadsMost, (threads + kWaveSize - 1) / kWaveSize * kWaveSize));
}
template <typename T>
void launch_rotary(const RotaryArgs &a, uint64_t threads, hipStream_t stream) {
    const uint32_t block = block_of(threads);
    const uint32_t groups = static_cast<uint32_t>((threads + block - 1) / block);
    if (a.tokens >= kManyTokens) {
        hipLaunchKernelGGL((rotary_kernel<T, kTokens>), dim3((a.tokens + kTokens - 1) / kTokens, groups), dim3(block), 0, stream, a);
    } else {
        hipLaunchKernelGGL((rotary_kernel<T, 1>), dim3(a.tokens, groups), dim3(block), 0, stream, a);
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
        a.turns[i] = std::pow(static_cast<double>(r->rope_theta), -2.0 * i / static_cast<double>(r->rope_dims)) / 6.28318530717958647693;
    }
    a.positions = r->positions;
    a.tokens = r->tokens;
    a.head_dim = r->head_dim;
    a.rope = r->rope_dims;
    a.eps = r->eps;
    a.inv_dim = 1.0 / r->head_dim;
    const uint32_t lanes = (half + 7) / 8 + (r->head_dim - r->rope_dims + 15) / 16;  // at most 17
    for (a.lanes = 1; a.lanes < lanes;) a.lanes *= 2;
    const uint64_t threads = static_cast<uint64_t>(heads[0] + heads[1]) * a.lanes;
    if ((tokens + kTokens - 1) / kTokens * block_of(threads) > 0xffffffffu) {  // a launch's threads are counted in 32 bits
        set_error("unsupported rotary request: %u tokens of %u heads in one call", r->tokens, heads[0] + heads[1]);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("rotary device", device.error());
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    if (r->dtype == QWN_HIP_DTYPE_F32) {
        launch_rotary<float>(a, threads, s);
    } else if (r->dtype == QWN_HIP_DTYPE_F16) {
        launch_rotary<f16>(a, threads, s);
    } else {
        launch_rotary<bf16>(a, threads, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("rotary launch", e);
}

}  // extern "C"
