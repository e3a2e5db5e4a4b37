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

// 8 elements as they lie in memory.
template <typename T>
struct Eight {
    static constexpr int VEC = 16 / sizeof(T);
    Vec<T, VEC> v[8 / VEC];

    __device__ __forceinline__ T &raw(int i) { return v[i / VEC].v[i % VEC]; }
    __device__ __forceinline__ float at(int i) const { return to_float(v[i / VEC].v[i % VEC]); }
    // Elements [c0, c0 + 8) of a row of n, zeros past its end.
    __device__ __forceinline__ void load(const T *row, uint32_t c0, uint32_t n) {
        if (c0 + 8 <= n) {
#pragma unroll
            for (int h = 0; h < 8 / VEC; ++h) v[h] = load_vec<T, VEC>(row + c0 + h * VEC);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) raw(i) = c0 + i < n ? row[c0 + i] : from_float<T>(0.0f);
        }
    }
    // Of the channels [c0, c0 + 8) of a head, the ones that they are paired
    // with: pairs (i, i + half) of the first `rope` channels.
    __device__ __forceinline__ void load_partners(const T *row, uint32_t c0, uint32_t n, uint32_t rope) {
        const uint32_t half = rope / 2;
        if (half % 8 == 0) {
            load(row, c0 >= rope ? c0 : c0 < half ? c0 + half : c0 - half, n);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t c = c0 + i;
                raw(i) = c < rope ? row[c < half ? c + half : c - half] : from_float<T>(0.0f);
            }
        }
    }
};
template <typename T>
__device__ __forceinline__ void store8(T *row, uint32_t c0, uint32_t n, const float v[8]) {
    if (c0 + 8 <= n) {
        constexpr int VEC = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8; h += VEC) {
            Vec<T, VEC> x;
#pragma unroll
            for (int i = 0; i < VEC; ++i) x.v[i] = from_float<T>(v[h + i]);
            store_vec<T, VEC>(row + c0 + h, x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < n) row[c0 + i] = from_float<T>(v[i]);
    }
}

// Where the angle of pair f stands in LDS: threads that take 8 pairs each read
// next to each other.
__device__ __forceinline__ uint32_t angle_at(uint32_t f) { return f % 8 * 16 + f / 8; }

// v, of channels [c0, c0 + 8), rotated with their partners o; cs: cos and sin
// of the position, at angle_at(pair).
template <typename T>
__device__ __forceinline__ void rotate8(float v[8], const Eight<T> &o, uint32_t c0, uint32_t rope, const double2 *cs) {
    const uint32_t half = rope / 2;
    if (half % 8 == 0) {  // all 8 are first channels of their pairs, or second ones, or not rotated
        if (c0 >= rope) return;
        const double2 *t = cs + (c0 < half ? c0 : c0 - half) / 8;
        const uint32_t flip = c0 < half ? 0x80000000u : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, o.at(i)) ^ flip);
            v[i] = static_cast<float>(static_cast<double>(v[i]) * t[16 * i].x + static_cast<double>(w) * t[16 * i].y);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = c0 + i;
        if (c < rope) {
            const double2 t = cs[angle_at(c < half ? c : c - half)];
            const double s = c < half ? -t.y : t.y;
            v[i] = static_cast<float>(static_cast<double>(v[i]) * t.x + static_cast<double>(o.at(i)) * s);
        }
    }
}

// The lanes' values 1, 2 and 7 - i apart within 8: after all three every lane
// has met all 8.
template <int STEP>
__device__ __forceinline__ float lane_near(float v) {
    constexpr int kCtrl = STEP == 0 ? 0xb1 : STEP == 1 ? 0x4e : 0x141;  // quad_perm [1, 0, 3, 2], [2, 3, 0, 1]; row_half_mirror
    const int x = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, kCtrl, 0xf, 0xf, true));
}

// The 4-bit codes (nibble i: channel c0 + i) of a lane's 8 channels of a
// head, and the group's step and minimum in every lane of the 8 that hold it.
// Channels past n count for nothing.  A code is the 64-bit quotient rounded,
// halves to even: f16 and bf16 inputs lie on borders between two codes.  The
// fp32 quotient is off by less than 2^-18 (three roundings of a number up to
// 16), so only next to a border does a lane compare in 64 bits what the border
// (of at most 16 bits) and the value are.
__device__ __forceinline__ uint32_t quantize8(float v[8], uint32_t c0, uint32_t n, f16 &step, f16 &least) {
    constexpr float kMax = 65504.0f;  // the largest f16
    float lo = v[0], hi = v[0];
    bool odd = c0 + 8 > n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
        if (i % 2) odd |= __builtin_isunordered(v[i - 1], v[i]);
    }
    if (__any(odd || lo < -kMax || hi > kMax)) {  // values that are not finite or past f16, channels past n
        lo = kMax, hi = -kMax;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = isfinite(v[i]) ? fminf(kMax, fmaxf(-kMax, v[i])) : 0.0f;
            if (c0 + i < n) {
                lo = fminf(lo, v[i]);
                hi = fmaxf(hi, v[i]);
            }
        }
    }
    lo = fminf(lo, lane_near<0>(lo)), hi = fmaxf(hi, lane_near<0>(hi));
    lo = fminf(lo, lane_near<1>(lo)), hi = fmaxf(hi, lane_near<1>(hi));
    lo = fminf(lo, lane_near<2>(lo)), hi = fmaxf(hi, lane_near<2>(hi));
    if (lo > hi) lo = hi = 0.0f;  // a group past the head's channels
    least = static_cast<f16>(lo);
    step = static_cast<f16>((hi - lo) / 15.0f);
    const float d = static_cast<float>(step), m = static_cast<float>(least), inv = d > 0.0f ? 1.0f / d : 0.0f;
    constexpr float kOne = 8388608.0f;  // 2^23: the sum's last bits are the number, rounded
    uint32_t codes = 0;
    float far = 0.0f;  // from a code
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = __builtin_amdgcn_fmed3f((v[i] - m) * inv, 0.0f, 15.0f), r = t + kOne;
        codes += __builtin_bit_cast(uint32_t, r) << (4 * i);
        far = fmaxf(far, fabsf(t - (r - kOne)));
    }
    codes -= 0x4b000000u + 0xb0000000u;  // kOne's bits, not shifted and shifted by 4: of the others nothing is left
    if (far > 0.49999f) {
        codes = 0;
        const double wide = static_cast<double>(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float h = floorf((v[i] - m) * inv);
            const double x = static_cast<double>(v[i]) - static_cast<double>(m), border = (static_cast<double>(h) + 0.5) * wide;
            const float code = x > border ? h + 1.0f : x < border ? h : rintf(h + 0.5f);
            codes |= static_cast<uint32_t>(__builtin_amdgcn_fmed3f(code, 0.0f, 15.0f)) << (4 * i);
        }
    }
    if (c0 + 8 > n) codes &= c0 < n ? (1u << 4 * (n - c0)) - 1 : 0u;
    return codes;
}

__device__ __forceinline__ uint32_t scale_word(f16 step, f16 least) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, least)) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, step)) << 16;
}

// Nibbles 0 .. 7 into the order of a key word (qwn_paged.h): even nibbles to
// 0 .. 3, odd ones to 4 .. 7.
__device__ __forceinline__ uint32_t key_order(uint32_t n) {
    auto gather = [](uint32_t x) {  // the low nibbles of the 4 bytes
        x &= 0x0f0f0f0fu;
        x = (x | x >> 4) & 0x00ff00ffu;
        return (x | x >> 8) & 0xffffu;
    };
    return gather(n) | gather(n >> 4) << 16;
}

// The rows of the batch that bring tokens to unit `unit` of sequence s.
struct Unit {
    uint32_t slot, from, count, row;  // its first slot; of its 4 slots the first that is new; how many; the first's row
};
__device__ __forceinline__ Unit unit_of(const PagedSequence &q, uint32_t unit) {
    Unit u;
    u.slot = (q.past / kPagedUnit + unit) * kPagedUnit;
    u.from = u.slot < q.past ? q.past - u.slot : 0u;
    u.count = min(kPagedUnit, q.past + q.rows - u.slot) - u.from;
    u.row = q.row + u.slot + u.from - q.past;
    return u;
}

// A unit's values and keys: a task is 8 channels of one head of either, of all
// its tokens, the next one's loads issued before this one's work.  (A loop, not
// four copies: those were 42 KB of instructions, most of a call of few tokens
// spent on fetching them, and 130 registers.)  Keys fill whole words.  A word
// of values is stored where the call brings all 4 of its tokens; else its bits
// are changed by an exclusive or, so that tokens of one word that come from two
// sequences of a call (a shared page) do not lose each other.
template <typename T>
struct KvTask {
    uint32_t head, lane;
    bool real, is_key;
    Eight<T> x, o;

    __device__ __forceinline__ void take(const AppendArgs &a, uint32_t i) {
        const uint32_t lanes = a.c.width / 8, kv_tasks = a.c.kv_heads * lanes;
        real = i < 2 * kv_tasks;
        is_key = i >= kv_tasks;
        const uint32_t j = real ? i - (is_key ? kv_tasks : 0u) : 0u;
        head = j / lanes;
        lane = j % lanes;
    }
    __device__ __forceinline__ void load(const AppendArgs &a, const Unit &u, uint32_t k) {
        const PagedKv &c = a.c;
        const size_t row = u.row + k;
        const T *src = (is_key ? static_cast<const T *>(a.key) + row * a.key_stride
                               : static_cast<const T *>(a.value) + row * a.value_stride) + head * c.head_dim;
        x.load(src, lane * 8, c.head_dim);
        if (is_key && c.rope_dims) o.load_partners(src, lane * 8, c.head_dim, c.rope_dims);
    }

    // Whole waves: lanes 1 to 4 apart exchange.
    __device__ __forceinline__ void store(const AppendArgs &a, const Unit &u, uint32_t page, const double2 (*cs)[128]) {
        const PagedKv &c = a.c;
        const uint32_t tile = (u.slot & (c.page_tokens - 1)) / kPagedTile, first = u.slot % kPagedTile;
        const uint32_t groups = c.width / kPagedGroup, c0 = lane * 8;
        uint8_t *block = c.pool + paged_block_at(c, page, tile, head);
        // values: channels c0 .. c0 + 7 are columns c0 % 16 .. of the 16 wide half
        // c0 / 16; the other half of their words is two lanes on.  Of the 8 columns
        // the first lane writes 4 words, the second 4; a word holds tokens 0 and 2 of
        // the first half, of the second, then 1 and 3.  even[t % 2], odd: tokens t and
        // t + 2 of columns 0 and 2, and of 1 and 3, a byte a half and column.
        const bool second = (lane / 2) % 2;  // this lane's channels are the words' second halves
        uint32_t even0 = 0, even1 = 0, odd0 = 0, odd1 = 0, mask = 0;
#pragma unroll 1
        for (uint32_t k = 0; k < u.count; ++k) {
            const uint32_t t = u.from + k, token = first + t;
            f16 step, least;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = x.at(i);
            if (is_key) rotate8(v, o, c0, c.rope_dims, cs[k]);
            if (k + 1 < u.count) load(a, u, k + 1);
            const uint32_t codes = quantize8(v, c0, c.head_dim, step, least);
            if (real && lane % 8 == 0)
                reinterpret_cast<uint32_t *>(block + (is_key ? paged_key_scales_at(c.width) : paged_value_scales_at(c.width)))
                    [token * groups + lane / 8] = scale_word(step, least);
            if (real && is_key) reinterpret_cast<uint32_t *>(block)[paged_key_word(c.width, token, c0)] = key_order(codes);
            const uint32_t other = __builtin_amdgcn_update_dpp(0, static_cast<int>(codes), 0x4e, 0xf, 0xf, true);
            // a token's 4 nibbles of the first half, and of the second
            const uint32_t cols = __builtin_amdgcn_perm(other, codes, second ? 0x03020706u : 0x05040100u);
            const uint32_t up = t & 2 ? 4 : 0, even = (cols & 0x0f0f0f0fu) << up, odd = (cols >> 4 & 0x0f0f0f0fu) << up;
            even0 |= t & 1 ? 0u : even, odd0 |= t & 1 ? 0u : odd;
            even1 |= t & 1 ? even : 0u, odd1 |= t & 1 ? odd : 0u;
            mask |= 15u << paged_value_bit(t, 0) | 15u << paged_value_bit(t, 16);
        }
        if (!real || is_key) return;
        const uint32_t bits[4] = {__builtin_amdgcn_perm(even1, even0, 0x06040200u), __builtin_amdgcn_perm(odd1, odd0, 0x06040200u),
                                  __builtin_amdgcn_perm(even1, even0, 0x07050301u), __builtin_amdgcn_perm(odd1, odd0, 0x07050301u)};
        uint32_t *words = reinterpret_cast<uint32_t *>(block + paged_values_at(c.width));
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            uint32_t *w = words + paged_value_word(c.width, first, (c0 & ~16u) + (second ? 4 + m : m));
            if (u.count == kPagedUnit) {
                *w = bits[m];
            } else {
                atomicXor(w, (*w ^ bits[m]) & mask);
            }
        }
    }
};

// A unit's queries: a task is 8 pairs of one head (both channels of a pair in
// one thread: the query may be rotated in place), or 8 of the channels behind
// the rotated ones, of all the unit's rows.
template <typename T>
struct QueryTask {
    uint32_t head, c0, end;
    bool real, pair;
    Eight<T> x, y;

    __device__ __forceinline__ void take(const AppendArgs &a, uint32_t i) {
        const uint32_t D = a.c.head_dim, rope = a.c.rope_dims, half = rope / 2;
        const uint32_t pairs = (half + 7) / 8, lanes = pairs + (D - rope + 7) / 8;
        real = i < a.query_heads * lanes;
        head = i / lanes;
        const uint32_t lane = i % lanes;
        pair = lane < pairs;
        c0 = pair ? lane * 8 : rope + (lane - pairs) * 8;
        end = pair ? half : D;
    }
    __device__ __forceinline__ void load(const AppendArgs &a, const Unit &u, uint32_t k) {
        if (!real) return;
        const T *src = static_cast<const T *>(a.query) + static_cast<size_t>(u.row + k) * a.query_stride + head * a.c.head_dim;
        x.load(src, c0, end);
        if (pair) y.load(src + a.c.rope_dims / 2, c0, a.c.rope_dims / 2);
    }

    __device__ __forceinline__ void store(const AppendArgs &a, const Unit &u, const double2 (*cs)[128]) {
        if (!real) return;
        const uint32_t half = a.c.rope_dims / 2;
#pragma unroll 1
        for (uint32_t k = 0; k < u.count; ++k) {
            T *dst = static_cast<T *>(a.query_out) + static_cast<size_t>(u.row + k) * a.query_out_stride + head * a.c.head_dim;
            float p[8], r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = x.at(e), r[e] = y.at(e);
            if (k + 1 < u.count) load(a, u, k + 1);
            if (pair) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double2 t = cs[k][angle_at(min(c0 + e, half - 1))];
                    const double v = static_cast<double>(p[e]), w = static_cast<double>(r[e]);
                    p[e] = static_cast<float>(v * t.x - w * t.y);
                    r[e] = static_cast<float>(v * t.y + w * t.x);
                }
                store8(dst + half, c0, half, r);
            }
            store8(dst, c0, end, p);
        }
    }
};

// grid (units of 4 slots at most, parts): the first kv_parts workgroups of a
// unit take its values and keys, the others its queries, a task a thread.  The
// angles of the unit's rows are computed once in each, in 64 bits (at position
// 100000 an fp32 angle would be off by hundredths), while the first loads are
// in flight.
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a, uint32_t kv_parts) {
    __shared__ double2 cs[kPagedUnit][128];
    uint32_t s, unit;
    PagedSequence q;
    const uint32_t half = a.c.rope_dims / 2;
    // ahead of the tasks' loads, which come back in order
    const double freq = a.c.freqs[half ? threadIdx.x % half : 0u];
    if (!find_unit(a.b, blockIdx.x, s, unit, q)) return;
    const Unit u = unit_of(q, unit);
    const uint32_t k0 = half ? threadIdx.x / half : kPagedUnit;
    const int32_t own = a.positions && k0 < u.count ? a.positions[u.row + k0] : 0;
    auto angles = [&] {
        for (uint32_t i = threadIdx.x; i < u.count * half; i += kAppendThreads) {
            const uint32_t k = i / half, f = i % half;
            const bool first = i == threadIdx.x;
            const double p = a.positions ? static_cast<double>(first ? own : a.positions[u.row + k])
                                         : static_cast<double>(u.slot + u.from + k);
            double2 t;
            sincos(p * (first ? freq : a.c.freqs[f]), &t.y, &t.x);
            cs[k][angle_at(f)] = t;
        }
        lds_barrier();
    };
    if (blockIdx.y < kv_parts) {
        uint32_t page = 0;
        const bool stored = paged_page(a.c, a.b, s, u.slot, page);  // looked up while the task's loads are on their way
        KvTask<T> task;
        task.take(a, blockIdx.y * kAppendThreads + threadIdx.x);
        task.load(a, u, 0);
        angles();
        if (stored) task.store(a, u, page, cs);
    } else {
        QueryTask<T> task;
        task.take(a, (blockIdx.y - kv_parts) * kAppendThreads + threadIdx.x);
        task.load(a, u, 0);
        angles();
        task.store(a, u, cs);
    }
}

struct ReadArgs {
    PagedKv c;
    PagedBatch b;
    float *keys, *values;
    uint32_t stride;
};

// The fp32 values of the batch's tokens: a workgroup per unit of 4 slots; a
// thread takes a word of keys (8 channels of a token) or four words of values
// (4 channels twice, of 4 tokens).
__global__ __launch_bounds__(kAppendThreads) void paged_read_kernel(ReadArgs a) {
    uint32_t s, unit;
    PagedSequence q;
    if (!find_unit(a.b, blockIdx.x, s, unit, q)) return;
    const PagedKv &c = a.c;
    const Unit u = unit_of(q, unit);
    uint32_t page = 0;
    if (!paged_page(c, a.b, s, u.slot, page)) return;
    const uint32_t tile = (u.slot & (c.page_tokens - 1)) / kPagedTile, first = u.slot % kPagedTile;
    const uint32_t D = c.head_dim, groups = c.width / kPagedGroup;
    const uint32_t key_tasks = c.width / 2, value_tasks = c.width / 8, tasks = key_tasks + value_tasks;  // of a head
    auto value = [](uint32_t scale, uint32_t code) {
        return fmaf(half_to_float(scale >> 16), static_cast<float>(code), half_to_float(scale & 0xffffu));
    };
    for (uint32_t i = threadIdx.x; i < c.kv_heads * tasks; i += kAppendThreads) {
        const uint32_t head = i / tasks, j = i % tasks;
        const uint8_t *block = c.pool + paged_block_at(c, page, tile, head);
        float v[8];
        if (j < key_tasks) {
            const uint32_t k = j / (key_tasks / 4), c0 = j % (key_tasks / 4) * 8;
            if (!a.keys || k < u.from || k >= u.from + u.count) continue;
            const uint32_t x = reinterpret_cast<const uint32_t *>(block)[paged_key_word(c.width, first + k, c0)];
            const uint32_t sc = reinterpret_cast<const uint32_t *>(block + paged_key_scales_at(c.width))[(first + k) * groups + c0 / kPagedGroup];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = value(sc, (x >> paged_key_bit(e)) & 15u);
            store8(a.keys + static_cast<size_t>(u.row + k - u.from) * a.stride + head * D, c0, D, v);
        } else if (a.values) {
            const uint32_t m = j - key_tasks, ch = m / 4 * 32 + m % 4 * 4;  // channels ch .. + 3 and ch + 16 .. + 19
            const uint32_t *codes = reinterpret_cast<const uint32_t *>(block + paged_values_at(c.width));
            uint32_t x[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = codes[paged_value_word(c.width, first, ch + e)];
#pragma unroll
            for (uint32_t k = 0; k < kPagedUnit; ++k) {
                if (k < u.from || k >= u.from + u.count) continue;
                const uint32_t sc = reinterpret_cast<const uint32_t *>(block + paged_value_scales_at(c.width))[(first + k) * groups + ch / kPagedGroup];
                float *row = a.values + static_cast<size_t>(u.row + k - u.from) * a.stride + head * D;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    Vec<float, 4> y;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) y.v[e] = value(sc, (x[e] >> paged_value_bit(k, 16 * h)) & 15u);
                    const uint32_t at = ch + 16 * h;
                    if (at + 4 <= D) {
                        store_vec<float, 4>(row + at, y);
                    } else {
                        for (uint32_t e = 0; e < 4 && at + e < D; ++e) row[at + e] = y.v[e];
                    }
                }
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
    const uint64_t size = dtype_bytes(r->dtype), rows = a.b.tokens;
    const Rows in = row_block(r->query, rows, q_channels, a.query_stride, size),
               out = row_block(r->query ? r->query_out : nullptr, rows, q_channels, a.query_out_stride, size);
    if ((!in_place(out, in) && overlap(out, in)) || overlaps_batch(out, a.b) ||
        overlaps_any(out, {row_block(r->key, rows, channels, a.key_stride, size), row_block(r->value, rows, channels, a.value_stride, size),
                           list_of_bytes(r->positions, 4 * rows)})) {
        set_error("paged KV append request: the rotated queries overlap an input");
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
    // a thread a task of the values and keys; of the queries a task of one token
    const uint32_t kv_parts = (2 * a.c.kv_heads * (a.c.width / 8) + kAppendThreads - 1) / kAppendThreads;
    const uint32_t q_parts = (a.query_heads * ((a.c.rope_dims / 2 + 7) / 8 + (a.c.head_dim - a.c.rope_dims + 7) / 8) +
                              kAppendThreads - 1) / kAppendThreads;
    const dim3 grid(paged_units_most(a.b.sequences, a.b.tokens), kv_parts + q_parts);
    if (r->dtype == QWN_HIP_DTYPE_F32) {
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(kAppendThreads), 0, s, a, kv_parts);
    } else if (r->dtype == QWN_HIP_DTYPE_F16) {
        hipLaunchKernelGGL(paged_append_kernel<f16>, grid, dim3(kAppendThreads), 0, s, a, kv_parts);
    } else {
        hipLaunchKernelGGL(paged_append_kernel<bf16>, grid, dim3(kAppendThreads), 0, s, a, kv_parts);
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
    const uint32_t channels = rp->c.kv_heads * rp->c.head_dim;
    const Rows k = row_block(keys, a.b.tokens, channels, a.stride, 4), v = row_block(values, a.b.tokens, channels, a.stride, 4);
    if (overlap(k, v) || overlaps_batch(k, a.b) || overlaps_batch(v, a.b)) {
        set_error("paged KV read: the keys, the values and the batch overlap");
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
