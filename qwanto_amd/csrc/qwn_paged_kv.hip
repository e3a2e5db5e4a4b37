// The paged 4-bit KV cache: creation, the append of a ragged batch with the
// rotary position applied on the way, and reading tokens back (layout:
// qwn_paged.h; attention over it: qwn_paged_attention.hip).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_paged.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

namespace {

using namespace qwn;

constexpr int kAppendThreads = 256;

struct AppendArgs {
    PagedKv c;
    PagedBatch b;
    const void *key, *value, *query;
    void *query_out;
    const int32_t *positions;
    uint32_t key_stride, value_stride, query_stride, query_out_stride, query_heads;
};

// Elements [c0, c0 + 8) of a row of n, zeros past its end.
template <typename T>
__device__ __forceinline__ void load8(const T *row, uint32_t c0, uint32_t n, float v[8]) {
    if (c0 + 8 <= n) {
        constexpr int VEC = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8; h += VEC) {
            const Vec<T, VEC> x = load_vec<T, VEC>(row + c0 + h);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[h + i] = to_float(x.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < n ? to_float(row[c0 + i]) : 0.0f;
    }
}

// The rotated channels [c0, c0 + 8) of a head: of the pairs (i, i + half) of
// the first `rope` channels, cos and sin [half] of the row's position.
template <typename T>
__device__ __forceinline__ void load8_rotated(const T *row, uint32_t c0, uint32_t n, uint32_t rope, const double2 *cs,
                                              float v[8]) {
    load8(row, c0, n, v);
    if (c0 >= rope) return;
    const uint32_t half = rope / 2;
    float o[8];
    if (half % 8 == 0) {
        load8(row, c0 < half ? c0 + half : c0 - half, n, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = c0 + i;
            o[i] = c < rope ? to_float(row[c < half ? c + half : c - half]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = c0 + i;
        if (c < rope) {
            const double2 t = cs[c < half ? c : c - half];
            const double s = c < half ? -t.y : t.y;
            v[i] = static_cast<float>(static_cast<double>(v[i]) * t.x + static_cast<double>(o[i]) * s);
        }
    }
}

// The 4-bit codes (nibble i: channel c0 + i) of a lane's 8 channels of a
// head, and the group's step and minimum in every lane of the 8 that hold it.
// Channels past n count for nothing.  The quotient that a code is rounded
// from is a 64-bit division: next to a border between two codes, and f16 and
// bf16 inputs lie on borders, fewer bits would choose another one.
__device__ __forceinline__ uint32_t quantize8(const float *x, uint32_t c0, uint32_t n, f16 &step, f16 &least) {
    constexpr float kMax = 65504.0f;  // the largest f16
    float v[8], lo = kMax, hi = -kMax;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = isfinite(x[i]) ? fminf(kMax, fmaxf(-kMax, x[i])) : 0.0f;
        if (c0 + i < n) {
            lo = fminf(lo, v[i]);
            hi = fmaxf(hi, v[i]);
        }
    }
    for (int off = 4; off > 0; off >>= 1) {
        lo = fminf(lo, __shfl_xor(lo, off));
        hi = fmaxf(hi, __shfl_xor(hi, off));
    }
    if (lo > hi) lo = hi = 0.0f;  // a group past the head's channels
    least = static_cast<f16>(lo);
    step = static_cast<f16>((hi - lo) / 15.0f);
    const double d = static_cast<double>(step), m = static_cast<double>(least);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double t = d > 0.0 ? rint((static_cast<double>(v[i]) - m) / d) : 0.0;
        const uint32_t code = t > 0.0 ? static_cast<uint32_t>(fmin(t, 15.0)) : 0u;
        codes |= (c0 + i < n ? code : 0u) << (4 * i);
    }
    return codes;
}

__device__ __forceinline__ uint32_t scale_word(f16 step, f16 least) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, least)) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, step)) << 16;
}

// Nibbles 0 .. 7 into the order of a key word (qwn_paged.h): even nibbles to
// 0 .. 3, odd ones to 4 .. 7.
__device__ __forceinline__ uint32_t key_order(uint32_t n) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= ((n >> (4 * i)) & 15u) << paged_key_bit(i);
    return w;
}

// One workgroup (or gridDim.y of them, which share its tasks) per aligned
// group of 4 slots that new tokens reach: the tokens whose values share a
// word.  The angles of its rows are computed once, in 64 bits: at position
// 100000 an fp32 angle would be off by hundredths.  A task is 8 channels of
// one head: of the values and keys of the group's tokens, or of one row's
// queries.  Keys fill whole words.  A word of values is stored where the call
// brings all 4 of its tokens; else its bits are changed by an exclusive or, so
// that tokens of one word that come from two sequences of a call (a shared
// page) do not lose each other.
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a) {
    __shared__ double2 cs[kPagedUnit][128];
    uint32_t s, unit;
    if (!find_unit(a.b, blockIdx.x, s, unit)) return;
    const PagedSequence q = paged_sequence(a.b, s);
    const PagedKv &c = a.c;
    const uint32_t slot0 = (q.past / kPagedUnit + unit) * kPagedUnit;
    const uint32_t from = slot0 < q.past ? q.past - slot0 : 0u;                       // of the 4 slots
    const uint32_t to = min(kPagedUnit, q.past + q.rows - slot0);
    const uint32_t row0 = q.row + slot0 + from - q.past, count = to - from;           // rows of the batch
    const uint32_t half = c.rope_dims / 2;
    for (uint32_t i = threadIdx.x; i < count * half; i += kAppendThreads) {
        const uint32_t k = i / half, f = i % half;
        const double p = a.positions ? static_cast<double>(a.positions[row0 + k]) : static_cast<double>(slot0 + from + k);
        double2 t;
        sincos(p * c.freqs[f], &t.y, &t.x);
        cs[k][f] = t;
    }
    __syncthreads();
    uint32_t page = 0;
    const bool stored = paged_page(c, a.b, s, slot0, page);
    const uint32_t tile = (slot0 & (c.page_tokens - 1)) / kPagedTile, first = slot0 % kPagedTile;
    const uint32_t lanes = c.width / 8, groups = c.width / kPagedGroup, D = c.head_dim;
    const uint32_t kv_tasks = stored ? c.kv_heads * lanes : 0u, q_lanes = (D + 7) / 8;
    const uint32_t tasks = a.query ? a.query_heads * q_lanes * count : 0u;
    const uint32_t threads = kAppendThreads * gridDim.y, me = blockIdx.y * kAppendThreads + threadIdx.x;
    const uint32_t kv_rounds = (2 * kv_tasks + kWaveSize - 1) / kWaveSize * kWaveSize;
    // whole waves: lanes 8 .. 32 apart exchange below
    for (uint32_t i = me; i < kv_rounds; i += threads) {
        const bool real = i < 2 * kv_tasks, is_key = i >= kv_tasks;
        const uint32_t j = real ? i - (is_key ? kv_tasks : 0u) : 0u;
        const uint32_t head = j / lanes, lane = j % lanes, c0 = lane * 8;
        uint8_t *block = c.pool + paged_block_at(c, page, tile, head);
        uint32_t codes[kPagedUnit] = {};
#pragma unroll
        for (uint32_t k = 0; k < kPagedUnit; ++k) {
            if (k >= count) break;
            float x[8];
            f16 step, least;
            const uint32_t row = row0 + k, token = first + from + k;
            if (is_key) {
                load8_rotated(static_cast<const T *>(a.key) + static_cast<size_t>(row) * a.key_stride + head * D, c0, D,
                              c.rope_dims, cs[k], x);
            } else {
                load8(static_cast<const T *>(a.value) + static_cast<size_t>(row) * a.value_stride + head * D, c0, D, x);
            }
            codes[k] = quantize8(x, c0, D, step, least);
            if (!real) continue;
            if (lane % 8 == 0)
                reinterpret_cast<uint32_t *>(block + (is_key ? paged_key_scales_at(c.width) : paged_value_scales_at(c.width)))
                    [token * groups + lane / 8] = scale_word(step, least);
            if (is_key) reinterpret_cast<uint32_t *>(block)[paged_key_word(c.width, token, c0)] = key_order(codes[k]);
        }
        // values: channels c0 .. c0 + 7 are columns n = c0 % 16 .. of the 16
        // wide half c0 / 16; the other half of their words is two lanes on
        uint32_t other[kPagedUnit];
#pragma unroll
        for (uint32_t k = 0; k < kPagedUnit; ++k) other[k] = __shfl_xor(codes[k], 2);
        if (!real || is_key) continue;
        const bool odd = (lane / 2) % 2;   // this lane's channels are the words' upper halves
        uint32_t *words = reinterpret_cast<uint32_t *>(block + paged_values_at(c.width));
        const uint32_t c_even = c0 & ~16u;
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            const uint32_t i4 = odd ? 4 + m : m;  // of the lane pair's 8 columns the even lane writes 4, the odd lane 4
            uint32_t bits = 0, mask = 0;
#pragma unroll
            for (uint32_t k = 0; k < kPagedUnit; ++k) {
                if (k >= count) break;
                const uint32_t mine = (codes[k] >> (4 * i4)) & 15u, theirs = (other[k] >> (4 * i4)) & 15u;
                const uint32_t lo = paged_value_bit(from + k, 0), hi = paged_value_bit(from + k, 16);
                bits |= (odd ? theirs : mine) << lo | (odd ? mine : theirs) << hi;
                mask |= 15u << lo | 15u << hi;
            }
            uint32_t *w = words + paged_value_word(c.width, first, c_even + i4);
            if (count == kPagedUnit) {
                *w = bits;
            } else {
                atomicXor(w, (*w ^ bits) & mask);
            }
        }
    }
    for (uint32_t i = me; i < tasks; i += threads) {
        const uint32_t k = i / (a.query_heads * q_lanes), j = i % (a.query_heads * q_lanes);
        const uint32_t head = j / q_lanes, c0 = j % q_lanes * 8, row = row0 + k;
        const T *src = static_cast<const T *>(a.query) + static_cast<size_t>(row) * a.query_stride + head * D;
        T *dst = static_cast<T *>(a.query_out) + static_cast<size_t>(row) * a.query_out_stride + head * D;
        // both channels of a pair in one thread: the query may be rotated in place
        float x[8];
        if (c0 >= c.rope_dims) {
            load8(src, c0, D, x);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e < D) dst[c0 + e] = from_float<T>(x[e]);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t ch = c0 + e;
            if (ch >= half) {
                if (ch >= c.rope_dims && ch < D) dst[ch] = src[ch];
                continue;
            }
            const double2 t = cs[k][ch];
            const double u = static_cast<double>(to_float(src[ch])), v = static_cast<double>(to_float(src[ch + half]));
            dst[ch] = from_float<T>(static_cast<float>(u * t.x - v * t.y));
            dst[ch + half] = from_float<T>(static_cast<float>(u * t.y + v * t.x));
        }
    }
}

struct ReadArgs {
    PagedKv c;
    PagedBatch b;
    float *keys, *values;
    uint32_t stride;
};

// The fp32 values of the batch's tokens: a workgroup per aligned group of 4
// slots, a thread a word of codes.
__global__ __launch_bounds__(kAppendThreads) void paged_read_kernel(ReadArgs a) {
    uint32_t s, unit;
    if (!find_unit(a.b, blockIdx.x, s, unit)) return;
    const PagedSequence q = paged_sequence(a.b, s);
    const PagedKv &c = a.c;
    const uint32_t slot0 = (q.past / kPagedUnit + unit) * kPagedUnit;
    const uint32_t from = slot0 < q.past ? q.past - slot0 : 0u;
    const uint32_t to = min(kPagedUnit, q.past + q.rows - slot0);
    uint32_t page = 0;
    if (!paged_page(c, a.b, s, slot0, page)) return;
    const uint32_t tile = (slot0 & (c.page_tokens - 1)) / kPagedTile, first = slot0 % kPagedTile;
    const uint32_t D = c.head_dim, groups = c.width / kPagedGroup, words = c.width / 2;  // of the group's values and of its keys
    for (uint32_t i = threadIdx.x; i < 2 * c.kv_heads * words; i += kAppendThreads) {
        const bool is_key = i >= c.kv_heads * words;
        const uint32_t j = i % (c.kv_heads * words), head = j / words, w = j % words;
        const uint8_t *block = c.pool + paged_block_at(c, page, tile, head);
        const uint32_t *codes = reinterpret_cast<const uint32_t *>(block + (is_key ? 0u : paged_values_at(c.width)));
        const uint32_t *scales = reinterpret_cast<const uint32_t *>(
            block + (is_key ? paged_key_scales_at(c.width) : paged_value_scales_at(c.width)));
        float *out = is_key ? a.keys : a.values;
        if (!out) continue;
        auto put = [&](uint32_t k, uint32_t ch, uint32_t code) {
            if (k < from || k >= to || ch >= D) return;
            const uint32_t sc = scales[(first + k) * groups + ch / kPagedGroup];
            out[static_cast<size_t>(q.row + slot0 + k - q.past) * a.stride + head * D + ch] =
                fmaf(half_to_float(sc >> 16), static_cast<float>(code), half_to_float(sc & 0xffffu));
        };
        if (is_key) {
            const uint32_t k = w / (words / 4), c0 = w % (words / 4) * 8;
            const uint32_t x = codes[paged_key_word(c.width, first + k, c0)];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) put(k, c0 + e, (x >> paged_key_bit(e)) & 15u);
        } else {
            const uint32_t ch = w / 16 * 32 + w % 16;
            const uint32_t x = codes[paged_value_word(c.width, first, ch)];
#pragma unroll
            for (uint32_t k = 0; k < kPagedUnit; ++k) {
                put(k, ch, (x >> paged_value_bit(k, 0)) & 15u);
                put(k, ch + 16, (x >> paged_value_bit(k, 16)) & 15u);
            }
        }
    }
}

void free_paged(ResidentPaged *rp) {
    if (rp->allocation) (void)hipFree(rp->allocation);
    delete rp;
}

}  // namespace

namespace qwn {

ResidentPaged *paged_of(Context *ctx, const QwnHipPagedKvHandle &h) {
    if (!header_ok(h) || !h.opaque) return nullptr;
    auto *c = static_cast<ResidentPaged *>(h.opaque);
    return std::find(ctx->paged.begin(), ctx->paged.end(), c) != ctx->paged.end() ? c : nullptr;
}

void destroy_paged(ResidentPaged *rp) { free_paged(rp); }

bool batch_of(const QwnHipPagedBatch *b, PagedBatch &out) {
    if (!b || !header_ok(*b) || b->sequences == 0 || b->tokens == 0 || b->table_stride == 0 || !b->starts || !b->past ||
        !b->page_table || b->tokens > 0x7fffffffu || b->sequences > 0x7fffffu)
        return false;
    out.sequences = b->sequences;
    out.tokens = b->tokens;
    out.table_stride = b->table_stride;
    out.starts = b->starts;
    out.past = b->past;
    out.table = b->page_table;
    return true;
}

}  // namespace qwn

extern "C" {

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_create(QwnCudaContextHandle *handle, const QwnHipPagedKvOptions *opt,
                                                 QwnHipPagedKvHandle *out) {
    Context *ctx = context_of(handle);
    if (!ctx || !opt || !out || !header_ok(*opt) || !header_ok(*out) || opt->pages == 0 || opt->kv_heads == 0 ||
        opt->head_dim == 0) {
        set_error("invalid paged KV-cache options");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (opt->head_dim > 256 || opt->page_tokens < kPagedTile || opt->page_tokens > 1024 ||
        (opt->page_tokens & (opt->page_tokens - 1)) ||
        opt->rope_dims % 2 || opt->rope_dims > opt->head_dim || opt->pages > 0x7fffffffu || opt->kv_heads > 65535 ||
        (opt->rope_dims && !(opt->rope_theta > 0.0f && std::isfinite(opt->rope_theta)))) {
        set_error("unsupported paged KV-cache options: head_dim %u, page_tokens %u, rope_dims %u", opt->head_dim,
                  opt->page_tokens, opt->rope_dims);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    PagedKv c;
    c.pages = opt->pages;
    c.page_tokens = opt->page_tokens;
    while ((1u << c.page_shift) < c.page_tokens) ++c.page_shift;
    c.kv_heads = opt->kv_heads;
    c.head_dim = opt->head_dim;
    c.width = paged_width(c.head_dim);
    c.rope_dims = opt->rope_dims;
    const size_t freq_bytes = 128 * sizeof(double);
    if (c.pages > (SIZE_MAX / 2) / paged_block_at(c, 1, 0, 0)) {
        set_error("paged KV-cache does not fit the configured GPU memory budget");
        return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    }
    const size_t pool = paged_block_at(c, c.pages, 0, 0);
    c.bytes = freq_bytes + pool;
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    hipError_t e = device.error();
    if (e != hipSuccess) return hip_fail("paged KV-cache device", e);
    size_t free_b = 0, total_b = 0;
    if ((e = hipMemGetInfo(&free_b, &total_b)) != hipSuccess) return hip_fail("paged KV-cache memory query", e);
    if (c.bytes > free_b || (ctx->budget && (c.bytes > ctx->budget || ctx->resident > ctx->budget - c.bytes))) {
        set_error("paged KV-cache does not fit the configured GPU memory budget");
        return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    }
    auto *rp = new (std::nothrow) ResidentPaged();
    if (!rp) return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    try {
        ctx->paged.reserve(ctx->paged.size() + 1);
    } catch (...) {
        delete rp;
        return QWN_CUDA_STATUS_OUT_OF_MEMORY;
    }
    if ((e = hipMalloc(&rp->allocation, c.bytes)) != hipSuccess) {
        rp->allocation = nullptr;
        free_paged(rp);
        return hip_fail("paged KV-cache allocation", e, QWN_CUDA_STATUS_OUT_OF_MEMORY);
    }
    c.freqs = static_cast<double *>(rp->allocation);
    c.pool = static_cast<uint8_t *>(rp->allocation) + freq_bytes;
    double freqs[128] = {};
    for (uint32_t i = 0; i < c.rope_dims / 2; ++i)
        freqs[i] = std::pow(static_cast<double>(opt->rope_theta), -2.0 * i / static_cast<double>(c.rope_dims));
    if ((e = hipMemsetAsync(c.pool, 0, pool, ctx->stream)) != hipSuccess ||
        (e = hipMemcpyAsync(c.freqs, freqs, sizeof(freqs), hipMemcpyHostToDevice, ctx->stream)) != hipSuccess ||
        (e = hipStreamSynchronize(ctx->stream)) != hipSuccess) {
        free_paged(rp);
        return hip_fail("paged KV-cache clear", e);
    }
    rp->c = c;
    ctx->paged.push_back(rp);
    ctx->resident += c.bytes;
    ctx->telemetry.kv_cache_resident_bytes += c.bytes;
    std::memset(out, 0, sizeof(*out));
    qwn_cuda_abi_header_init(&out->header, sizeof(*out));
    out->opaque = rp;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_destroy(QwnCudaContextHandle *handle, QwnHipPagedKvHandle *h) {
    Context *ctx = context_of(handle);
    if (!ctx || !h) {
        set_error("invalid paged KV-cache destroy request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    ResidentPaged *rp = paged_of(ctx, *h);
    if (!rp) {
        set_error("paged KV-cache handle is not resident in this context");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    DeviceScope device(ctx->device);
    // work on the caller's own streams may still read it
    (void)hipDeviceSynchronize();
    const uint64_t bytes = rp->c.bytes;
    ctx->paged.erase(std::find(ctx->paged.begin(), ctx->paged.end(), rp));
    free_paged(rp);
    ctx->resident -= std::min(ctx->resident, bytes);
    ctx->telemetry.kv_cache_resident_bytes -= std::min(ctx->telemetry.kv_cache_resident_bytes, bytes);
    h->opaque = nullptr;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_append_device(QwnCudaContextHandle *handle, QwnHipPagedKvHandle *h,
                                                        const QwnHipPagedAppendRequest *r, void *stream) {
    Context *ctx = context_of(handle);
    AppendArgs a{};
    if (!ctx || !h || !r || !header_ok(*r) || !batch_of(r->batch, a.b) || !r->key || !r->value ||
        r->dtype > QWN_HIP_DTYPE_BF16 || (r->query && (!r->query_out || r->query_heads == 0 || r->query_heads > 65535))) {
        set_error("invalid paged KV append request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    ResidentPaged *rp = paged_of(ctx, *h);
    if (!rp) {
        set_error("paged KV-cache handle is not resident in this context");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint32_t channels = rp->c.kv_heads * rp->c.head_dim, q_channels = r->query_heads * rp->c.head_dim;
    a.key_stride = stride_or(r->key_stride, channels);
    a.value_stride = stride_or(r->value_stride, channels);
    a.query_stride = stride_or(r->query_stride, q_channels);
    a.query_out_stride = stride_or(r->query_out_stride, q_channels);
    if (a.key_stride < channels || a.value_stride < channels ||
        (r->query && (a.query_stride < q_channels || a.query_out_stride < q_channels ||
                      (r->query == r->query_out && a.query_stride != a.query_out_stride)))) {
        set_error("paged KV append request: a row stride is shorter than its row, or differs in place");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("paged KV append device", device.error());
    a.c = rp->c;
    a.key = r->key;
    a.value = r->value;
    a.query = r->query;
    a.query_out = r->query_out;
    a.positions = r->positions;
    a.query_heads = r->query ? r->query_heads : 0u;
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const uint32_t units = paged_units_most(a.b.sequences, a.b.tokens);
    const dim3 grid(units, 1);
    if (r->dtype == QWN_HIP_DTYPE_F32) {
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(kAppendThreads), 0, s, a);
    } else if (r->dtype == QWN_HIP_DTYPE_F16) {
        hipLaunchKernelGGL(paged_append_kernel<f16>, grid, dim3(kAppendThreads), 0, s, a);
    } else {
        hipLaunchKernelGGL(paged_append_kernel<bf16>, grid, dim3(kAppendThreads), 0, s, a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail("paged KV append launch", e);
    ctx->telemetry.kv_cache_kernel_count++;
    return QWN_CUDA_STATUS_OK;
}

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_read_device(QwnCudaContextHandle *handle, QwnHipPagedKvHandle *h,
                                                      const QwnHipPagedBatch *batch, float *keys, float *values,
                                                      uint32_t stride, void *stream) {
    Context *ctx = context_of(handle);
    ReadArgs a{};
    if (!ctx || !h || !batch_of(batch, a.b) || (!keys && !values)) {
        set_error("invalid paged KV read request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    ResidentPaged *rp = paged_of(ctx, *h);
    if (rp) a.stride = stride_or(stride, rp->c.kv_heads * rp->c.head_dim);
    if (!rp || a.stride < rp->c.kv_heads * rp->c.head_dim) {
        set_error("invalid paged KV read request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("paged KV read device", device.error());
    a.c = rp->c;
    a.keys = keys;
    a.values = values;
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    hipLaunchKernelGGL(paged_read_kernel, dim3(paged_units_most(a.b.sequences, a.b.tokens)), dim3(kAppendThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("paged KV read launch", e);
}

}  // extern "C"
