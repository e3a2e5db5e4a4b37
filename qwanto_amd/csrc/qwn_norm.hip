// The residual's addition, RMSNorm and the per-token int8 quantization of a
// batch of tokens in one pass (qwn_hip_ext_norm_quantize_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_types.h"

namespace {

using namespace qwn;

struct NormArgs {
    const void *x, *residual;
    void *residual_out, *y;
    const float *norm;
    int8_t *q8;
    float *scales;
    uint32_t cols, x_stride, residual_stride, residual_out_stride, y_stride, q8_stride;
    float eps;
};

// Sum over the workgroup, in every thread; red holds a value per wave.
__device__ __forceinline__ double block_sum(double v, double *red) {
    v = wave_sum_f64(v);
    const uint32_t waves = blockDim.x / kWaveSize;
    if (waves == 1) return v;
    if (threadIdx.x % kWaveSize == 0) red[threadIdx.x / kWaveSize] = v;
    lds_barrier();
    double s = red[0];
    for (uint32_t w = 1; w < waves; ++w) s += red[w];
    return s;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
    v = wave_max_u32(v);
    const uint32_t waves = blockDim.x / kWaveSize;
    if (waves == 1) return v;
    if (threadIdx.x % kWaveSize == 0) red[threadIdx.x / kWaveSize] = v;
    lds_barrier();
    uint32_t s = red[0];
    for (uint32_t w = 1; w < waves; ++w) s = max(s, red[w]);
    return s;
}

constexpr uint32_t kNotFinite = 0x7f800000u;  // |y| as bits: infinities and NaN from here

// The scale of a token from the bits of its largest |y|, and the factor its
// values are quantized with (IEEE division and reciprocal, as quantize_device).
__device__ __forceinline__ void scale_of(uint32_t amax_bits, float &scale, float &inv) {
    const float amax = __builtin_bit_cast(float, amax_bits);
    scale = amax > 0.0f ? amax / 127.0f : 1.0f;
    inv = 1.0f / scale;
    if (amax_bits >= kNotFinite) scale = __builtin_nanf(""), inv = 0.0f;
}
__device__ __forceinline__ uint32_t q8_of(float y, float inv, bool finite) {
    const uint32_t q = q8_low_byte(fminf(127.0f, fmaxf(-127.0f, y * inv)));
    return finite ? q : 0u;
}

// One workgroup a token; thread t holds the row's vectors t, t + NT, ... (VPT
// of at most 16 bytes a load) and, the first cols % VEC threads, one element
// of its end, in registers: the row is read once.  The mean square and y are
// in 64 bits (fp64 arithmetic runs at the fp32 rate here and the row's bytes
// bound the pass): a code of q8 then depends on the inputs alone, not on the
// order of a sum.
template <typename T, int VPT>
__global__ __launch_bounds__(1024) void norm_quantize_kernel(NormArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ double red_sum[1024 / kWaveSize];
    __shared__ uint32_t red_max[1024 / kWaveSize];
    const size_t t = blockIdx.x;
    const uint32_t tid = threadIdx.x, nt = blockDim.x;
    const uint32_t full = a.cols / VEC, rest = a.cols % VEC;
    const T *x = static_cast<const T *>(a.x) + t * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + t * a.residual_stride : nullptr;
    T *out = a.residual_out ? static_cast<T *>(a.residual_out) + t * a.residual_out_stride : nullptr;
    float h[VPT][VEC], w[VPT][VEC], he = 0.0f, we = 0.0f;
    const uint32_t end = full * VEC + tid;  // the element of the row's end, if any
    const bool tail = tid < rest;
    Vec<T, VEC> xv[VPT], rv[VPT];
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const uint32_t c = tid + nt * e;
        if (c < full) {
            xv[e] = load_vec<T, VEC>(x + c * VEC);
            if (r) rv[e] = load_vec<T, VEC>(r + c * VEC);
            const Vec<float, VEC> wv = load_vec<float, VEC>(a.norm + c * VEC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[e][i] = wv.v[i];
        }
    }
    if (tail) {
        he = to_float(x[end]);
        if (r) he = to_float(from_float<T>(he + to_float(r[end])));
        we = a.norm[end];
    }
    double ss = static_cast<double>(he) * he;
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const uint32_t c = tid + nt * e;
        if (c < full) {
            Vec<T, VEC> hv;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                hv.v[i] = r ? from_float<T>(to_float(xv[e].v[i]) + to_float(rv[e].v[i])) : xv[e].v[i];
                h[e][i] = to_float(hv.v[i]);
                ss = fma(static_cast<double>(h[e][i]), static_cast<double>(h[e][i]), ss);
            }
            if (out) store_vec<T, VEC>(out + c * VEC, hv);
        }
    }
    if (tail && out) out[end] = from_float<T>(he);
    ss = block_sum(ss, red_sum);
    const double inv_rms = 1.0 / sqrt(ss / static_cast<double>(a.cols) + static_cast<double>(a.eps));
    uint32_t amax = 0;
    auto normed = [&](float hh, float ww) {
        const float y = static_cast<float>(static_cast<double>(hh) * inv_rms * static_cast<double>(ww));
        amax = max(amax, __builtin_bit_cast(uint32_t, y) & 0x7fffffffu);
        return y;
    };
    T *yrow = a.y ? static_cast<T *>(a.y) + t * a.y_stride : nullptr;
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const uint32_t c = tid + nt * e;
        if (c < full) {
            Vec<T, VEC> yv;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[e][i] = normed(h[e][i], w[e][i]);
                yv.v[i] = from_float<T>(h[e][i]);
            }
            if (yrow) store_vec<T, VEC>(yrow + c * VEC, yv);
        }
    }
    if (tail) {
        he = normed(he, we);
        if (yrow) yrow[end] = from_float<T>(he);
    }
    if (!a.q8) return;
    amax = block_max(amax, red_max);
    float scale, inv;
    scale_of(amax, scale, inv);
    const bool finite = amax < kNotFinite;
    if (tid == 0) a.scales[t] = scale;
    uint8_t *q = reinterpret_cast<uint8_t *>(a.q8) + t * a.q8_stride;
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const uint32_t c = tid + nt * e;
        if (c < full) {
            Vec<uint8_t, VEC> qv;
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const uint32_t word = pack_low_bytes(q8_of(h[e][i], inv, finite), q8_of(h[e][i + 1], inv, finite),
                                                     q8_of(h[e][i + 2], inv, finite), q8_of(h[e][i + 3], inv, finite));
                __builtin_memcpy(qv.v + i, &word, 4);
            }
            store_vec<uint8_t, VEC>(q + c * VEC, qv);
        }
    }
    if (tail) q[end] = static_cast<uint8_t>(q8_of(he, inv, finite));
    for (uint32_t k = a.cols + tid; k < a.q8_stride; k += nt) q[k] = 0;
}

// Rows too long for a workgroup's registers: the row is read three times
// (from the caches after the first), each thread writing only elements that
// it alone reads, so residual_out may still be x or residual.
template <typename T>
__global__ __launch_bounds__(1024) void norm_quantize_long_kernel(NormArgs a) {
    __shared__ double red_sum[1024 / kWaveSize];
    __shared__ uint32_t red_max[1024 / kWaveSize];
    const size_t t = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + t * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + t * a.residual_stride : nullptr;
    T *out = a.residual_out ? static_cast<T *>(a.residual_out) + t * a.residual_out_stride : nullptr;
    T *yrow = a.y ? static_cast<T *>(a.y) + t * a.y_stride : nullptr;
    auto value = [&](uint32_t k) {
        const T v = x[k];
        return r ? to_float(from_float<T>(to_float(v) + to_float(r[k]))) : to_float(v);
    };
    double ss = 0.0;
    for (uint32_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
        const double h = value(k);
        ss = fma(h, h, ss);
    }
    ss = block_sum(ss, red_sum);
    const double inv_rms = 1.0 / sqrt(ss / static_cast<double>(a.cols) + static_cast<double>(a.eps));
    auto normed = [&](float h, uint32_t k) {
        return static_cast<float>(static_cast<double>(h) * inv_rms * static_cast<double>(a.norm[k]));
    };
    uint32_t amax = 0;
    if (a.q8)
        for (uint32_t k = threadIdx.x; k < a.cols; k += blockDim.x)
            amax = max(amax, __builtin_bit_cast(uint32_t, normed(value(k), k)) & 0x7fffffffu);
    amax = block_max(amax, red_max);
    float scale, inv;
    scale_of(amax, scale, inv);
    const bool finite = amax < kNotFinite;
    if (a.q8 && threadIdx.x == 0) a.scales[t] = scale;
    int8_t *q = a.q8 ? a.q8 + t * a.q8_stride : nullptr;
    for (uint32_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
        const float h = value(k), y = normed(h, k);
        if (out) out[k] = from_float<T>(h);
        if (yrow) yrow[k] = from_float<T>(y);
        if (q) q[k] = static_cast<int8_t>(q8_of(y, inv, finite) & 0xffu);
    }
    if (q)
        for (uint32_t k = a.cols + threadIdx.x; k < a.q8_stride; k += blockDim.x) q[k] = 0;
}

template <typename T>
hipError_t launch_norm(const NormArgs &a, uint32_t tokens, hipStream_t stream) {
    constexpr uint32_t VEC = 16 / sizeof(T);
    const uint32_t vectors = std::max(1u, a.cols / VEC);
    auto threads = [&](uint32_t vpt) { return ((vectors + vpt - 1) / vpt + kWaveSize - 1) / kWaveSize * kWaveSize; };
    if (vectors <= 2 * 1024) {
        // two vectors a thread: 4099 tokens of 2560 fp32 27 us (5.0 TB/s), one a
        // thread 31 (fewer rows at a time), four 28; one token the same
        hipLaunchKernelGGL((norm_quantize_kernel<T, 2>), dim3(tokens), dim3(threads(2)), 0, stream, a);
    } else if (vectors <= 4 * 1024) {
        // some of the 4 vectors spill (16-bit rows), still for less than a row read
        // again: 1000 tokens of 16392 bf16 44 us, 65 below; of 32768 84 and 144
        hipLaunchKernelGGL((norm_quantize_kernel<T, 4>), dim3(tokens), dim3(threads(4)), 0, stream, a);
    } else {
        hipLaunchKernelGGL((norm_quantize_long_kernel<T>), dim3(tokens), dim3(1024), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API int qwn_hip_ext_norm_quantize_device(QwnCudaContextHandle *handle, const QwnHipNormRequest *r,
                                                      void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || !r || !header_ok(*r) || r->tokens == 0 || r->cols == 0 || r->tokens > 0x7fffffffu || !r->x ||
        !r->norm || r->dtype > QWN_HIP_DTYPE_BF16 || (r->q8 && !r->scales) || (!r->residual_out && !r->y && !r->q8)) {
        set_error("invalid norm request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    NormArgs a{};
    a.x = r->x;
    a.residual = r->residual;
    a.residual_out = r->residual_out;
    a.y = r->y;
    a.norm = r->norm;
    a.q8 = r->q8;
    a.scales = r->scales;
    a.cols = r->cols;
    a.x_stride = stride_or(r->x_stride, r->cols);
    a.residual_stride = stride_or(r->residual_stride, r->cols);
    a.residual_out_stride = stride_or(r->residual_out_stride, r->cols);
    a.y_stride = stride_or(r->y_stride, r->cols);
    a.q8_stride = stride_or(r->q8_stride, r->cols);
    a.eps = r->eps;
    if (a.x_stride < a.cols || a.residual_stride < a.cols || a.residual_out_stride < a.cols || a.y_stride < a.cols ||
        a.q8_stride < a.cols || (a.residual_out == a.x && a.residual_out_stride != a.x_stride) ||
        (a.residual_out && a.residual_out == a.residual && a.residual_out_stride != a.residual_stride)) {
        set_error("norm request: a row stride is shorter than its row, or differs in place");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t size = dtype_bytes(r->dtype);
    const Rows x = row_block(a.x, r->tokens, a.cols, a.x_stride, size), res = row_block(a.residual, r->tokens, a.cols, a.residual_stride, size),
               out = row_block(a.residual_out, r->tokens, a.cols, a.residual_out_stride, size),
               y = row_block(a.y, r->tokens, a.cols, a.y_stride, size),
               q8 = row_block(a.q8, r->tokens, a.q8_stride, a.q8_stride, 1),
               scales = list_of_bytes(a.q8 ? a.scales : nullptr, r->tokens * sizeof(float)),
               norm = list_of_bytes(a.norm, a.cols * sizeof(float));
    if ((!in_place(out, x) && overlap(out, x)) || (!in_place(out, res) && overlap(out, res)) ||
        overlaps_any(y, {x, res, out, norm, q8, scales}) || overlaps_any(q8, {x, res, out, norm, scales}) ||
        overlaps_any(scales, {x, res, out, norm}) || overlap(out, norm)) {
        set_error("norm request: an output overlaps an input or another output");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("norm device", device.error());
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_norm<float>(a, r->tokens, s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_norm<f16>(a, r->tokens, s)
                                                         : launch_norm<bf16>(a, r->tokens, s);
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("norm launch", e);
}

}  // extern "C"
