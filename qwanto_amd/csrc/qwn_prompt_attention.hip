// Causal attention of packed sequences over their own keys and values
// (qwn_hip_ext_prompt_attention_device).
//
//   out[i] = sum_{t <= i} p_t v_t / sum_{t <= i} p_t,  p_t = exp(scale q_i.k_t - max)
//
// The rows of a KV head are its tokens times the query heads that share it, so
// that all of them read a tile of keys and values once.  Scores are computed
// transposed, S^T = K Q^T, on the 32 x 32 matrix instructions: a lane then
// holds, of one row, 16 of 32 tokens, four next to each other, which is
// what the second product O^T = V^T P^T takes of its right operand once the
// tokens are counted in that order: probabilities go from one product to the
// other in their registers.  Rows of V^T come from LDS by the transposing read.
//
// Scores and sums are fp32; probabilities are rounded to the inputs' type for the
// second product (by at most 2^-8 of each in bf16, 2^-11 in f16, as the output itself is; over
// the tokens it averages out; in f16 those below 2^-20 of the row's largest by up to 2^-31 of that),
// and fp32 goes in fp32 throughout.
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace {

using namespace qwn;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr uint32_t kWaves = 4, kThreads = kWaves * kWaveSize, kWaveRows = 32;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFar = 0x1p20f;               // of references: past it their rounding would be more than 2^-4 of an exponent

// Workgroups from which on blocks of 128 rows are best (bf16, 32 heads of 128: one
// prompt of 512 tokens, 128 groups, 18 us and in blocks of 64 14; of 1777 and eight
// shorter, 728 groups, 52 and 59).
constexpr uint64_t kManyGroups = 320;
// Heads of 64 channels have half the products between two barriers: in sequences of that
// many tokens on average tiles of 128, until so many workgroups hide the barriers by
// themselves.  16 heads, tiles of 128 and of 64: one prompt of 300 tokens 8.6 and 8.6 us, of 500 9.6 and
// 10.4, of 2000 21.7 and 25.0, of 3000, 1200 and 300 41 and 45; six of 400 13.7 and 13.2, four of 500 12.1
// and 12.4, but of 600 15.6 and 13.8, three of 800 16.5 and 15.2, two of 1000 16.8 and 17.2: where a sequence
// ends in its tiles counts as much as the average, which is what the host knows.  30 of 200 tokens 19 and
// 16; one of 8192, 1024 groups, 165 and 160.
constexpr uint32_t kLongTokens = 512;
constexpr uint64_t kFullGroups = 1024;

struct PromptArgs {
    const void *query, *key, *value;
    void *output;
    const int32_t *starts;
    uint32_t sequences, tokens, kv_heads, group, head_dim;
    uint32_t query_stride, key_stride, value_stride, output_stride;
    float scale;
};

// The two 16-bit types' operands and products.
template <typename T>
struct Matrix;
template <>
struct Matrix<f16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ v16f mul(frag a, frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Matrix<bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ v16f mul(frag a, frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
// Queries are scaled to below 2^kQueryBits: of f16 products are then below 2^40, and no query is
// scaled down, which its smallest channels have no bits for; of the others, with any finite key, below 2^127.
template <typename T>
constexpr int kQueryBits = std::is_same_v<T, f16> ? 16 : -9;
// The exponent of the reference's own probability.  Of f16 numbers below 2^-14 lose bits: with 2^6, a
// probability is off by 2^-11 of itself, or by 2^-31 of the row's largest, so that 2^20 tokens with next
// to none of the weight still add up to it within f16's own rounding.  (A larger one leaves less room until the
// reference moves: scores spread by 4, 1500 tokens of 128 channels 30 us, with 2^8 32, with 1 27.)
template <typename T>
constexpr float kLift = std::is_same_v<T, f16> ? 6.0f : 0.0f;
// What a lane's probabilities of a tile may add up to: of f16 none passes it.
template <typename T>
constexpr float kMost = std::is_same_v<T, f16> ? 65504.0f : 0x1p40f;
// Probabilities of up to 2^40 times values past 2^88, or a sum of values next to the
// type's largest, are past fp32 although their average is not.  A block with sums near that is
// gone through again, with probabilities 2^-34 as large and references at each
// row's largest so far: those of 2^31 tokens add up to less than 1.  Only what was not finite and
// now is takes the second result, so what one channel holds shows in no other.  f16's products
// are below 2^32: its averages may only be rounded past the largest.
constexpr float kSecondLift = -34.0f;
template <typename T>
constexpr bool kTwice = !std::is_same_v<T, f16>;
// The type's largest number: an average of finite values is not past it, but may be rounded past it.
template <typename T>
constexpr float kLargest = std::is_same_v<T, f16> ? 65504.0f : std::is_same_v<T, bf16> ? 0x1.fep127f : 0x1.fffffep127f;

struct Span {
    uint32_t row = 0, rows = 0;  // of a sequence; none where its starts do not lie in the batch
};
__device__ __forceinline__ Span span_of(const PromptArgs &a, uint32_t s) {
    Span q;
    if (s >= a.sequences) return q;
    const int32_t r0 = a.starts[s], r1 = a.starts[s + 1];
    if (r0 < 0 || r1 <= r0 || static_cast<uint32_t>(r1) > a.tokens) return q;
    q.row = static_cast<uint32_t>(r0);
    q.rows = static_cast<uint32_t>(r1 - r0);
    return q;
}
// The sequence that holds block `index` of the batch, and its number there;
// false past the last.  Every wave searches for itself, 64 sequences a step.
__device__ __forceinline__ bool find_block(const PromptArgs &a, uint32_t lane, uint32_t block_rows, uint32_t index, Span &q, uint32_t &at) {
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += kWaveSize) {
        const Span mine = span_of(a, s0 + lane);
        const uint32_t n = (mine.rows * a.group + block_rows - 1) / block_rows, end = wave_scan(n);
        const uint64_t past = __ballot(end > index);
        if (past) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            at = index - (lane_of(end, first) - lane_of(n, first));
            if (at >= lane_of(n, first)) return false;  // starts that do not ascend: the sums have wrapped
            q = Span{lane_of(mine.row, first), lane_of(mine.rows, first)};
            return true;
        }
        index -= lane_of(end, kWaveSize - 1);
    }
    return false;
}

// What a row's products, of queries times the power of two `up`, are multiplied
// by to be exponents of 2: positive, the scale's sign is the queries'.  Products are below 2^127:
// where it is below fp32's numbers all scores are alike (its rounding to the smallest of them is off by
// 2^-22 of an exponent); past fp32 the largest fp32 stands in its place.
__device__ __forceinline__ float exponents_of(float scale, int bits, float &up) {
    const float mul = fminf(ldexpf(fabsf(scale), bits) * 1.44269504088896340736f, 3.402823466e38f);
    const bool alike = mul == 0.0f;
    up = alike ? 0.0f : copysignf(up, scale);
    if (!isfinite(scale)) up = __builtin_nanf("");  // the row is NaN, whatever the keys are
    return alike ? 1.0f : mul;
}

// The two halves of the wave hold a row's tokens together: what both have of v.
struct Both {
    float low, high;
};
__device__ __forceinline__ Both both_halves(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t low = r[0], high = r[1];
    return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}
__device__ __forceinline__ float halves_max(float v) {
    const Both b = both_halves(v);
    return fmaxf(b.low, b.high);
}
__device__ __forceinline__ float halves_sum(float v) {
    const Both b = both_halves(v);
    return b.low + b.high;
}

// A row's softmax so far: the reference as a product, and what exponents are taken from,
// mul times it less lift; far: some row of the wave has one too far to be rounded.  m is 0 of a
// row that has seen nothing.  lift: the exponent of the reference's own probability.
struct Softmax {
    float m = 0.0f, ref = 0.0f, sum = 0.0f, mul = 0.0f, lift = 0.0f;
    bool far = false;
    __device__ __forceinline__ float reference(float mx) const { return mul_rounded(mx, mul) - lift; }
    // What sums are multiplied by as the reference goes from (from, was) to (to, is): exponents
    // were taken from `was` itself where it is near, else from `from` times mul as it is.
    __device__ __forceinline__ float moved(float from, float was, float to, float is) const {
        const bool near = fabsf(was) < kFar, stays = fabsf(is) < kFar;
        return __builtin_amdgcn_exp2f(near ? (stays ? was - is : fmaf(-to, mul, was) + lift)
                                           : stays ? fmaf(from, mul, -is) - lift : (from - to) * mul);
    }
};
template <int S>
__device__ __forceinline__ float largest_of(const v16f (&sc)[S]) {
    float mx = sc[0][0];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[s][e]);
    return halves_max(mx);
}
// The probabilities of products sc, and their sum.
template <int S>
__device__ __forceinline__ float weigh(const v16f (&sc)[S], const Softmax &x, float (&p)[S][16]) {
    float add = 0.0f;
    if (x.far) {  // of rows with a far reference the product is taken off first
        const bool mine = !(fabsf(x.ref) < kFar);
        const float off = mine ? x.m : 0.0f, less = mine ? -x.lift : x.ref;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                p[s][e] = __builtin_amdgcn_exp2f(fmaf(sc[s][e] - off, x.mul, -less));
                add += p[s][e];
            }
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                p[s][e] = __builtin_amdgcn_exp2f(fmaf(sc[s][e], x.mul, -x.ref));
                add += p[s][e];
            }
    }
    return add;
}
// A tile's probabilities, the sums moved to another reference where they would pass
// `top`.  first: the wave's first tile; sees: the row sees some of it.
template <int S, int C>
__device__ __forceinline__ void softmax_tile(const v16f (&sc)[S], Softmax &x, float (&p)[S][16], v16f (&acc)[C], bool first, bool sees,
                                             float top) {
    if (first) {
        x.m = sees ? fmaxf(largest_of(sc), kLowest) : 0.0f;
        x.ref = x.reference(x.m);
        x.far = __any(!(fabsf(x.ref) < kFar));
    }
    float add = weigh(sc, x, p);
    if (__any(!(add < top))) {
        // of the rows that pass it, which does not depend on other rows
        const bool over = halves_max(add < top ? 0.0f : 1.0f) > 0.0f;
        const float mx = over ? fmaxf(x.m, largest_of(sc)) : x.m, to = x.reference(mx);
        const float alpha = x.moved(x.m, x.ref, mx, to);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= alpha;
        x.sum *= alpha;
        x.m = mx;
        x.ref = to;
        x.far = __any(!(fabsf(to) < kFar));
        add = weigh(sc, x, p);
    }
    x.sum += add;
}

// The sums of the waves that took parts of the same rows' tokens, RW waves a part,
// in those of part 0; false in the others.  A row that has seen none of a part's
// tokens has the sum 0 there, and no reference.
template <int C, int RW, int NW>
constexpr size_t join_bytes = RW == NW ? 0 : NW * kWaveSize * 16 + (NW - RW) * C * 16 * kWaveSize * 4;
template <int C, int RW, int NW>
__device__ __forceinline__ bool join_parts(v4u *lds, uint32_t wave, uint32_t lane, bool sees, Softmax &x, v16f (&acc)[C]) {
    constexpr int KW = NW / RW;
    x.sum = halves_sum(x.sum);
    if constexpr (KW > 1) {
        lds_barrier();
        float4 *state = reinterpret_cast<float4 *>(lds);                     // [wave][lane]
        float *sums = reinterpret_cast<float *>(state + NW * kWaveSize);     // [wave past part 0][element][lane]
        state[wave * kWaveSize + lane] = make_float4(x.m, x.ref, x.sum, sees ? 1.0f : 0.0f);
        if (wave >= RW) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) sums[((wave - RW) * C * 16 + c * 16 + e) * kWaveSize + lane] = acc[c][e];
        }
        lds_barrier();
        if (wave >= RW) return false;
        float mx = x.m;
#pragma unroll
        for (int k = 1; k < KW; ++k) {
            const float4 o = state[(wave + k * RW) * kWaveSize + lane];
            if (o.w > 0.0f) mx = fmaxf(mx, o.x);
        }
        const float to = x.reference(mx), mine = x.moved(x.m, x.ref, mx, to);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= mine;
        x.sum *= mine;
#pragma unroll
        for (int k = 1; k < KW; ++k) {
            const float4 o = state[(wave + k * RW) * kWaveSize + lane];
            const bool any = o.w > 0.0f;
            const float f = any ? x.moved(o.x, o.y, mx, to) : 0.0f;
            x.sum += any ? o.z * f : 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float o2 = sums[((wave + (k - 1) * RW) * C * 16 + c * 16 + e) * kWaveSize + lane];
                    acc[c][e] += any ? o2 * f : 0.0f;
                }
        }
    }
    return true;
}

// A block of rows of a KV head, and a lane's row of it.
struct Block {
    Span q;
    uint32_t head, row0, last;   // of the sequence's rows: the first, and the last real one
    uint32_t most, least;        // tokens that any row sees, and every one
};
template <uint32_t ROWS>
__device__ __forceinline__ bool block_of(const PromptArgs &a, uint32_t lane, Block &b) {
    uint32_t at;
    b.head = blockIdx.x % a.kv_heads;
    if (!find_block(a, lane, ROWS, blockIdx.x / a.kv_heads, b.q, at)) return false;
    const uint32_t all = b.q.rows * a.group, blocks = (all + ROWS - 1) / ROWS;
    b.row0 = (blocks - 1 - at) * ROWS;  // a sequence's longest contexts first
    b.last = min(b.row0 + ROWS, all) - 1;
    b.most = b.last / a.group + 1;
    b.least = b.row0 / a.group + 1;
    return true;
}
struct Row {
    uint32_t token, at;          // of the sequence; elements from the token's first query channel
    uint32_t visible;            // tokens it sees; none where it is no row
    uint32_t w_most, w_least;    // tokens that any row of the wave sees, and every one
};
__device__ __forceinline__ Row row_of(const PromptArgs &a, const Block &b, uint32_t w_row0, uint32_t n) {
    Row r;
    const uint32_t rr = min(w_row0 + n, b.last);
    r.token = rr / a.group;
    r.at = (b.head * a.group + rr % a.group) * a.head_dim;
    r.visible = w_row0 + n <= b.last ? r.token + 1 : 0u;
    const bool idle = w_row0 > b.last;
    r.w_most = idle ? 0u : min(w_row0 + kWaveRows - 1, b.last) / a.group + 1;
    r.w_least = idle ? 0u : w_row0 / a.group + 1;
    return r;
}

// A tile of `KT` tokens of W channels in LDS, 16 bytes (CE channels) a chunk.
// Chunk c of token t lies in place c ^ spread(t) of its row: reads of one chunk
// of 16 tokens, and of 4 chunks of 4 tokens, both reach each bank once.
template <typename T, int W>
struct Tile {
    static constexpr uint32_t CE = 16 / sizeof(T), NC = W / CE;
    static __device__ __forceinline__ uint32_t spread(uint32_t t) {
        return NC >= 16 ? (t % 4) * 4 + t / 4 % 4 : t / 2 % 2 * 4 + t / 4 % 4;
    }
    // in chunks
    static __device__ __forceinline__ uint32_t at(uint32_t t, uint32_t c) { return t * NC + (c ^ spread(t)); }
};

// 16 bytes of a row of n elements from element c on, zeros past its end.
template <typename T>
__device__ __forceinline__ v4u load_chunk(const T *row, uint32_t c, uint32_t n) {
    constexpr uint32_t CE = 16 / sizeof(T);
    if (c + CE <= n) return __builtin_bit_cast(v4u, load_vec<T, CE>(row + c));
    Vec<T, CE> x;
#pragma unroll
    for (uint32_t e = 0; e < CE; ++e) x.v[e] = c + e < n ? row[c + e] : from_float<T>(0.0f);
    return __builtin_bit_cast(v4u, x);
}
// 16 bytes a lane into LDS, the wave's next to each other from `to` on.  In
// assembly, as the compiler would wait for all such loads before the transposing reads
// of the other buffer; it does not count them: wait_vmcnt does.  m0 is one of the compiler's own
// registers, of which it warns; named, it knows that what m0 held is gone.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void *from, v4u *to) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
template <typename T>
__device__ __forceinline__ bool finite(T v) {
    if constexpr (sizeof(T) == 4) {
        return (__builtin_bit_cast(uint32_t, v) & 0x7f800000u) != 0x7f800000u;
    } else {
        constexpr uint16_t kExponent = std::is_same_v<T, f16> ? 0x7c00u : 0x7f80u;
        return (__builtin_bit_cast(uint16_t, v) & kExponent) != kExponent;
    }
}

// The lane's number, from the hardware: what is made of it before a loop need not be kept over it.
__device__ __forceinline__ uint32_t lane_anew() {
    uint32_t lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// Whether some of a part's sums are past 2^-4 of fp32's largest, or NaN: else the joined ones, of four parts at
// most, are finite, and so are their averages.  (More is taken for it where several come near; that costs a pass.)
template <int C>
__device__ __forceinline__ bool past_range(const v16f (&acc)[C]) {
    float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd[e % 4] = fmaf(acc[c][e], 16.0f, odd[e % 4]);
    return !(fabsf((odd[0] + odd[1]) + (odd[2] + odd[3])) < INFINITY);
}
// N of a row's sums from channel ch on as averages.
template <typename T, int N>
__device__ __forceinline__ void store_averages(T *dst, uint32_t ch, uint32_t channels, const float (&sums)[N], float inv) {
    Vec<T, N> y;
#pragma unroll
    for (int k = 0; k < N; ++k) y.v[k] = from_float<T>(sums[k] * inv);
    if (ch + N <= channels) {
        store_vec<T, N>(dst + ch, y);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (ch + k < channels) dst[ch + k] = y.v[k];
    }
}
// The same where what is there is not finite, and can be.
template <typename T, int N>
__device__ __forceinline__ void mend_averages(T *dst, uint32_t ch, uint32_t channels, const float (&sums)[N], float inv) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float v = sums[k] * inv;
        if (ch + k < channels && fabsf(sums[k]) < INFINITY && !finite(dst[ch + k]))
            dst[ch + k] = from_float<T>(fabsf(v) > kLargest<T> ? copysignf(kLargest<T>, v) : v);
    }
}

// Keys and values of a tile, and how many tiles LDS is given room for.
template <typename T, int W, int KT>
constexpr size_t tile_bytes = 2 * KT * W * sizeof(T);

constexpr int kSchedMatrix = 0x8, kSchedLds = 0x100;  // kinds of instructions to the scheduler
typedef __attribute__((address_space(3))) char lds_char;
template <typename V>
using lds_ptr = __attribute__((address_space(3))) V *;

// A lane's 16-byte pieces of its query, CE channels each, scaled; pieces 2 j + h.
template <typename T, int J>
__device__ __forceinline__ void load_query(const PromptArgs &a, const Block &b, const Row &r, uint32_t h, v4u (&qf)[J], float &mul) {
    constexpr uint32_t CE = 16 / sizeof(T);
    const T *qp = static_cast<const T *>(a.query) + static_cast<size_t>(b.q.row + r.token) * a.query_stride + r.at;
    Vec<T, CE> raw[J];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) raw[j] = __builtin_bit_cast(Vec<T, CE>, load_chunk(qp, (2 * j + h) * CE, a.head_dim));
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (uint32_t e = 0; e < CE; ++e) top = fmaxf(top, fabsf(to_float(raw[j].v[e])));
    top = halves_max(top);
    int e2 = kQueryBits<T>;  // top < 2^e2, and as it is where that is not finite (its row is NaN)
    if (top < INFINITY) (void)frexpf(top, &e2);
    e2 = max(e2, -100);
    float up = ldexpf(1.0f, kQueryBits<T> - e2);
    mul = exponents_of(a.scale, e2 - kQueryBits<T>, up);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        Vec<T, CE> x;
#pragma unroll
        for (uint32_t e = 0; e < CE; ++e) x.v[e] = from_float<T>(to_float(raw[j].v[e]) * up);
        qf[j] = __builtin_bit_cast(v4u, x);
    }
}

// f16 and bf16.  A workgroup takes RW blocks of 32 rows of a KV head, a wave's
// each, and goes through the tiles of its context; of a tile's tokens, 4 / RW waves
// with the same rows take a part each, and their sums meet at the end.  Two
// buffers of LDS, one worked on while the other is filled (DIRECT, of whole aligned
// chunks: by loads that go to LDS; else through registers).
// Exponents are taken from a reference, the row's largest product in its first
// tile: where a later tile's probabilities add up to more than kMost, the
// reference is moved to what is largest then, so other tiles need no maximum.  Masked
// tokens have probability 0; so that 0 times a value that is not finite does
// not reach rows that do not see it, such values are taken as 0 in the tiles that
// are masked and added to the rows that see them.
// Bound by the vector unit's exponents and the matrix unit, taken in turn by the two
// waves of a SIMD, long prompts also by the power that clocks are given for (1.9 to 2.1 of 2.4 GHz): bf16,
// 32 heads of 128, one prompt of 8192 tokens 521 to 552 us (1 PFLOP/s, of 1.17 that a
// large product reaches); short ones by the longest block's chain of tiles: nine of up to
// 1777 tokens 45 us, of which a large product would take 25.
template <typename T, int W, int KT, int RW, bool DIRECT, bool AGAIN>
__device__ __forceinline__ bool attend_block(const PromptArgs &a, uint32_t &again_wanted, uint32_t wave, uint32_t lane) {
    using M = Matrix<T>;
    using L = Tile<T, W>;
    constexpr uint32_t CE = L::CE, NC = L::NC;
    constexpr uint32_t kChunks = KT * NC, kOfThread = kChunks / kThreads, kBlockRows = RW * kWaveRows;
    constexpr int KW = kWaves / RW, C = W / 32, S = KT / 32 / KW, J = NC / 2;
    constexpr bool kAhead = W <= 128;
    static_assert(kChunks % kThreads == 0 && S > 0, "whole rounds of loads, a part for each wave");
    extern __shared__ v4u tiles[];          // two times keys, then values
    constexpr uint32_t kMasked = kBlockRows / KT + 2;
    __shared__ uint32_t odd[kMasked][KT / 32];  // of the masked tiles: tokens with values that are not finite
    const uint32_t tid = wave * kWaveSize + lane, n = lane % 32, h = lane / 32, part = wave / RW;  // of a tile's tokens
    Block b;
    if (!block_of<kBlockRows>(a, lane, b)) return false;
    const uint32_t count = (b.most + KT - 1) / KT, masked = b.least / KT;  // tiles, and the first that not every row sees all of
    const T *keys = static_cast<const T *>(a.key) + static_cast<size_t>(b.q.row) * a.key_stride + b.head * a.head_dim;
    const T *values = static_cast<const T *>(a.value) + static_cast<size_t>(b.q.row) * a.value_stride + b.head * a.head_dim;

    // Chunk x of a tile in LDS: its token and place.  A thread's chunks are kRows
    // tokens apart, of which every kSame-th has the same channels.
    constexpr uint32_t kRows = kThreads / NC, kSame = kRows % 16 ? 16 / kRows : 1;
    v4u kr[DIRECT ? 1 : kOfThread], vr[DIRECT ? 1 : kOfThread];
    auto channel = [&](uint32_t e) { return (tid % NC ^ L::spread(tid / NC + kRows * e)) * CE; };
    const T *first_key[kSame], *first_value[kSame];
#pragma unroll
    for (uint32_t e = 0; e < kSame; ++e) {
        first_key[e] = keys + static_cast<size_t>(tid / NC) * a.key_stride + channel(e);
        first_value[e] = values + static_cast<size_t>(tid / NC) * a.value_stride + channel(e);
    }
    auto bring = [&](uint32_t i) {
        v4u *buf = tiles + i % 2 * 2 * kChunks;
        if (DIRECT && (i + 1) * KT <= b.most && a.head_dim == W) {
#pragma unroll
            for (uint32_t e = 0; e < kOfThread; ++e) {
                v4u *to = buf + kThreads * e + wave * kWaveSize;
                const size_t t = i * KT + kRows * e;  // the same for all lanes
                load_to_lds(first_key[e % kSame] + t * a.key_stride, to);
                load_to_lds(first_value[e % kSame] + t * a.value_stride, to + kChunks);
            }
            return;
        }
#pragma unroll
        for (uint32_t e = 0; e < kOfThread; ++e) {
            const uint32_t c = channel(e % kSame);
            const size_t t = min(i * KT + tid / NC + kRows * e, b.most - 1);  // tokens past the last are the last
            if constexpr (DIRECT) {
                if (c >= a.head_dim) continue;  // zeros from the beginning
                v4u *to = buf + kThreads * e + wave * kWaveSize;
                load_to_lds(keys + t * a.key_stride + c, to);
                load_to_lds(values + t * a.value_stride + c, to + kChunks);
            } else {
                kr[e] = load_chunk(keys + t * a.key_stride, c, a.head_dim);
                vr[e] = load_chunk(values + t * a.value_stride, c, a.head_dim);
            }
        }
    };
    // what was brought is in LDS
    auto settle = [&](uint32_t i) {
        if constexpr (DIRECT) {
            wait_vmcnt<0>();
        } else {
            v4u *buf = tiles + i % 2 * 2 * kChunks;
#pragma unroll
            for (uint32_t e = 0; e < kOfThread; ++e) {
                buf[tid + kThreads * e] = kr[e];
                buf[kChunks + tid + kThreads * e] = vr[e];
            }
        }
        lds_barrier();
    };
    auto clean = [&](uint32_t i) {
        v4u *vt = tiles + (i % 2 * 2 + 1) * kChunks;
#pragma unroll 1
        for (uint32_t x = tid; x < kChunks; x += kThreads) {
            Vec<T, CE> v = __builtin_bit_cast(Vec<T, CE>, vt[x]);
            bool bad = false;
#pragma unroll
            for (uint32_t k = 0; k < CE; ++k)
                if (!finite(v.v[k])) bad = true, v.v[k] = from_float<T>(0.0f);
            if (bad) {
                vt[x] = __builtin_bit_cast(v4u, v);
                atomicOr(&odd[i - masked][x / NC / 32], 1u << x / NC % 32);
            }
        }
        lds_barrier();
    };
    if (DIRECT && a.head_dim != W) {
#pragma unroll
        for (uint32_t e = 0; e < 4 * kOfThread; ++e)
            if (channel(e % kSame) >= a.head_dim) tiles[tid + kThreads * e] = (v4u){0, 0, 0, 0};
    }
    bring(0);

    // this lane's row, as a column of the products
    const Row r = row_of(a, b, b.row0 + wave % RW * kWaveRows, n);
    v4u qf[J];
    Softmax soft;
    soft.lift = AGAIN ? kSecondLift : kLift<T>;
    load_query<T>(a, b, r, h, qf, soft.mul);
    if (!AGAIN && tid == 0) again_wanted = 0;
    if (tid < kMasked * (KT / 32)) odd[tid / (KT / 32)][tid % (KT / 32)] = 0;

    // where a lane's operands lie in a buffer: of keys piece 2 j + h of token n, of V^T
    // (16 lanes each read 4 tokens of 16 channels) block c, tokens 0 .. 7 and 8 .. 15 of 16
    lds_char *const lds = (lds_char *)tiles;
    uint32_t keys_at[J], values_at[C][2];
#pragma unroll
    for (int j = 0; j < J; ++j) keys_at[j] = (part * S * 32 * NC + L::at(n, 2 * j + h)) * 16;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            values_at[c][k] = (kChunks + part * S * 32 * NC + L::at(4 * h + lane % 16 / 4 + 8 * k, 4 * c + 2 * (lane / 16 % 2) + lane % 4 / 2)) * 16 +
                              lane % 2 * 8;

    v16f acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;

    for (uint32_t i = 0; i < count; ++i) {
        settle(i);  // tile i is there, and the other buffer is free
        if (i >= masked) clean(i);
        if (i + 1 < count) bring(i + 1);
        const uint32_t t0 = i * KT + part * S * 32;  // the wave's part, and where it lies in the tile
        if (t0 >= r.w_most) continue;
        lds_char *const buf = lds + i % 2 * 2 * kChunks * 16;
        v16f sc[S];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const auto kf = __builtin_bit_cast(typename M::frag, *(lds_ptr<v4u>)(buf + keys_at[j] + s * 32 * NC * 16));
                if (j == 0)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[s][e] = 0.0f;
                sc[s] = M::mul(kf, __builtin_bit_cast(typename M::frag, qf[j]), sc[s]);
            }
        // operands are read four products ahead (of 256 channels that took 267 us where it is 225: registers)
        if constexpr (kAhead) {
            __builtin_amdgcn_sched_group_barrier(kSchedLds, 4, 0);
#pragma unroll
            for (int x = 0; x < J * S; ++x) {
                __builtin_amdgcn_sched_group_barrier(kSchedLds, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMatrix, 1, 0);
            }
        }
        // element e of sc[s]: token t0 + 32 s + 8 (e / 4) + 4 h + e % 4
        if (t0 + S * 32 > r.w_least) {
            const int32_t seen = static_cast<int32_t>(r.visible) - static_cast<int32_t>(t0 + 4 * h);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * s + 8 * (e / 4) + e % 4 >= seen) sc[s][e] = -INFINITY;
        }
        float p[S][16];
        softmax_tile(sc, soft, p, acc, i == 0, r.visible > t0, AGAIN ? 0.0f : kMost<T>);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                typename M::frag pf;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const auto p2 = __builtin_convertvector((v2f){p[s][8 * u + e], p[s][8 * u + e + 1]}, typename M::pair);
                    pf[e] = p2[0], pf[e + 1] = p2[1];
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    union {
                        v4s part[2];
                        typename M::frag whole;
                    } x;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        x.part[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<v4s>)(buf + values_at[c][k] + (32 * s + 16 * u) * NC * 16));
                    acc[c] = M::mul(x.whole, pf, acc[c]);
                }
            }
        if constexpr (kAhead) {
            __builtin_amdgcn_sched_group_barrier(kSchedLds, 8, 1);
#pragma unroll
            for (int x = 0; x < 2 * S * C; ++x) {
                __builtin_amdgcn_sched_group_barrier(kSchedMatrix, 1, 1);
                __builtin_amdgcn_sched_group_barrier(kSchedLds, 2, 1);
            }
        }
        if (i >= masked) {
#pragma unroll 1
            for (int s = 0; s < S; ++s)
                for (uint32_t left = odd[i - masked][part * S + s]; left; left &= left - 1) {
                    const uint32_t t = t0 + 32 * s + __ffs(static_cast<int>(left)) - 1;
                    if (t >= r.visible) continue;
                    const T *row = values + static_cast<size_t>(t) * a.value_stride;
                    uint32_t d = a.head_dim;
                    asm("" : "+s"(d));  // compared here: 16 C masks kept over the loop would not have the registers
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint32_t ch = 32 * c + 8 * (e / 4) + 4 * h + e % 4;
                            if (ch < d && !finite(row[ch])) acc[c][e] += to_float(row[ch]);
                        }
                }
        }
    }

    if (!AGAIN && kTwice<T> && past_range(acc)) again_wanted = 1;
    if (join_parts<C, RW, kWaves>(tiles, wave, lane, r.visible > part * S * 32, soft, acc) && r.visible > 0) {
        const float inv = 1.0f / soft.sum;
        T *dst = static_cast<T *>(a.output) + static_cast<size_t>(b.q.row + r.token) * a.output_stride + r.at;
        auto each = [&](auto take) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float sums[4] = {acc[c][e], acc[c][e + 1], acc[c][e + 2], acc[c][e + 3]};
                    take(32 * c + 8 * (e / 4) + 4 * h, sums);
                }
        };
        if (!AGAIN) each([&](uint32_t ch, const float (&sums)[4]) { store_averages<T, 4>(dst, ch, a.head_dim, sums, inv); });
        if constexpr (!kTwice<T>) {
            float odd = 0.0f;  // infinite or NaN where an average past the type's largest is added
            each([&](uint32_t, const float (&sums)[4]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) odd = fmaf(sums[k], inv * (0x1.fffffep127f / kLargest<T> * 1.0001f), odd);
            });
            if (fabsf(odd) < INFINITY) return false;
        }
        if (AGAIN || !kTwice<T>) each([&](uint32_t ch, const float (&sums)[4]) { mend_averages<T, 4>(dst, ch, a.head_dim, sums, inv); });
    }
    if (AGAIN || !kTwice<T>) return false;
    if (KW == 1) lds_barrier();  // else the join has come past some since
    return __builtin_amdgcn_readfirstlane(again_wanted);
}

// What a workgroup does, and again where the first pass asks for it (every wave returns whether).  The second is
// code of its own, with arguments and lanes taken anew, so that the first keeps nothing in registers for it: as a
// loop over one code both spilled.  The first one's times are what they are without a second, to 0.3 us.
__device__ __forceinline__ PromptArgs arguments_at(uint64_t args) {
    auto word = [&](size_t at) { return *reinterpret_cast<const __attribute__((address_space(4))) uint32_t *>(args + at); };
    auto pointer = [&](size_t at) {
        const uint64_t p = *reinterpret_cast<const __attribute__((address_space(4))) uint64_t *>(args + at);
        return (void *)reinterpret_cast<__attribute__((address_space(1))) void *>(p);
    };
    PromptArgs a;
    a.query = pointer(offsetof(PromptArgs, query));
    a.key = pointer(offsetof(PromptArgs, key));
    a.value = pointer(offsetof(PromptArgs, value));
    a.output = pointer(offsetof(PromptArgs, output));
    a.starts = static_cast<const int32_t *>(pointer(offsetof(PromptArgs, starts)));
    a.sequences = word(offsetof(PromptArgs, sequences));
    a.tokens = word(offsetof(PromptArgs, tokens));
    a.kv_heads = word(offsetof(PromptArgs, kv_heads));
    a.group = word(offsetof(PromptArgs, group));
    a.head_dim = word(offsetof(PromptArgs, head_dim));
    a.query_stride = word(offsetof(PromptArgs, query_stride));
    a.key_stride = word(offsetof(PromptArgs, key_stride));
    a.value_stride = word(offsetof(PromptArgs, value_stride));
    a.output_stride = word(offsetof(PromptArgs, output_stride));
    a.scale = __builtin_bit_cast(float, word(offsetof(PromptArgs, scale)));
    return a;
}
template <auto FIRST, auto SECOND, typename K>
__device__ __forceinline__ void once_or_twice(const PromptArgs &a, K &kept) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    if (!FIRST(a, kept, wave, threadIdx.x % kWaveSize)) return;
    lds_barrier();  // the first pass's LDS is read
    uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    SECOND(arguments_at(args), kept, wave, lane_anew());
}
template <typename T, int W, int KT, int RW, bool DIRECT>
__global__ __launch_bounds__(kThreads, W == 256 ? 1 : W == 64 && KT == 64 ? 3 : 2) void prompt_attention_kernel(PromptArgs a) {
    __shared__ uint32_t again_wanted;
    if constexpr (kTwice<T>) {
        once_or_twice<&attend_block<T, W, KT, RW, DIRECT, false>, &attend_block<T, W, KT, RW, DIRECT, true>>(a, again_wanted);
    } else {
        attend_block<T, W, KT, RW, DIRECT, false>(a, again_wanted, __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize), threadIdx.x % kWaveSize);
    }
}

// What fp32's two passes share: 128 channels take 53.2 KB for the join, of which three workgroups have room in a CU's LDS
// as long as there are 512 bytes more at most; the third starts while the first waves of two write their output
// (four prompts of 1024, 687, 598 and 171 tokens 97 us without it, 93 with it).
struct Kept {
    uint32_t again_wanted;
    uint2 rows[kWaveRows];  // token and place of each, until its output
};

// fp32.  A product of two fp32 operands (v_mfma_f32_32x32x2_f32) takes 64 cycles for
// an operand of 4 bytes a lane, 16 times as long as the 16-bit ones for theirs: L2
// brings a wave's operands in the time, so keys and values need no LDS and no barrier
// (through LDS one call of four prompts of 1024, 300, 100 and 500 tokens, 12 heads, took 225 us, and
// takes 73).  The four waves of a workgroup take the same 32 rows and every fourth
// tile of 32 tokens.  A tile's values are loaded when its scores are there, into the
// registers that held its keys, the next keys after its sums: with the rows' query
// in LDS two waves a SIMD fit (three of 64 channels were not faster, 332 us for 310), one's products run
// while the other waits (one wave with loads ahead: 32 heads of 128 channels, 4096 tokens, 1440 us
// for 1170; of 256 channels, where they did not fit, 430 for 175).  Heads between 128 and 256
// channels have more addresses and compared channels than registers (468 bytes a lane go to
// scratch in both passes): 200 channels, 1024 tokens of 8 heads 163 us.
// A lane's values are W / 32 channels next to each other: block c of the output's
// rows are channels c, c + W / 32, ...  WHOLE: heads of W channels.
// Bound by the matrix unit: those 1160 to 1184 us are 117 TFLOP/s, of 154 that a large product
// reaches; few rows by the longest one's chain of tiles.
template <int W, bool WHOLE, bool AGAIN>
__device__ __forceinline__ bool attend_block_f32(const PromptArgs &a, Kept &kept, uint32_t wave, uint32_t lane) {
    constexpr uint32_t KT = 32, KW = kWaves;
    constexpr int C = W / 32, J = W / 8;
    extern __shared__ v4u lds[];
    uint2 *const rows = kept.rows;
    uint32_t &again_wanted = kept.again_wanted;
    const uint32_t tid = wave * kWaveSize + lane, n = lane % 32, h = lane / 32, part = wave;
    Block b;
    if (!block_of<kWaveRows>(a, lane, b)) return false;
    const Row r = row_of(a, b, b.row0, n);
    const uint32_t count = (r.w_most + KT - 1) / KT;
    const float *keys = static_cast<const float *>(a.key) + static_cast<size_t>(b.q.row) * a.key_stride + b.head * a.head_dim;
    const float *values = static_cast<const float *>(a.value) + static_cast<size_t>(b.q.row) * a.value_stride + b.head * a.head_dim;
    auto piece = [&](const float *row, uint32_t c, uint32_t d) {
        if constexpr (WHOLE) {
            return load_vec<float, 4>(row + c);
        } else {
            return __builtin_bit_cast(Vec<float, 4>, load_chunk(row, c, d));
        }
    };
    // compared for each tile: masks kept over the loop would not have the registers (96 channels, four
    // prompts of 1024, 500, 300 and 100 tokens 94 us for 99; of 256, where they are twice as many, 190 for 165)
    auto channels = [&]() {
        uint32_t d = a.head_dim;
        if constexpr (!WHOLE && W <= 128) asm volatile("" : "+s"(d));
        return d;
    };
    Vec<float, 4> kf[J];
    Vec<float, C> vf[16];
    auto load_keys = [&](uint32_t i) {
        const uint32_t d = channels();
        const float *row = keys + static_cast<size_t>(min(i * KT + n, b.most - 1)) * a.key_stride;
#pragma unroll
        for (int j = 0; j < J; ++j) kf[j] = piece(row, (2 * j + h) * 4, d);
    };
    auto load_values = [&](uint32_t i) {
        const uint32_t d = channels();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float *row = values + static_cast<size_t>(min(i * KT + 8 * (e / 4) + 4 * h + e % 4, b.most - 1)) * a.value_stride;
            if constexpr (C >= 4) {
#pragma unroll
                for (int x = 0; x < C / 4; ++x) {
                    const Vec<float, 4> v = piece(row, C * n + 4 * x, d);
#pragma unroll
                    for (int k = 0; k < 4; ++k) vf[e].v[4 * x + k] = v.v[k];
                }
            } else if constexpr (WHOLE) {
                vf[e] = load_vec<float, C>(row + C * n);
            } else {
#pragma unroll
                for (int k = 0; k < C; ++k) vf[e].v[k] = C * n + k < d ? row[C * n + k] : 0.0f;
            }
        }
    };
    v4u qf[J];
    Softmax soft;
    soft.lift = AGAIN ? kSecondLift : kLift<float>;
    load_query<float>(a, b, r, h, qf, soft.mul);
    v4u *const query = lds + lane;
    if (!AGAIN && tid == 0) again_wanted = 0;
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < J; ++j) query[j * kWaveSize] = qf[j];
        rows[n] = make_uint2(r.token, r.at);
    }
    lds_barrier();
    if (part < count) load_keys(part);
    v16f acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;

    for (uint32_t i = part; i < count; i += KW) {
        const uint32_t t0 = i * KT;
        v16f sc[1], odd;  // two chains of products
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[0][e] = odd[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const v4f q4 = __builtin_bit_cast(v4f, query[j * kWaveSize]);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j].v[e], q4[e], sc[0], 0, 0, 0);
                odd = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j].v[e + 1], q4[e + 1], odd, 0, 0, 0);
            }
        }
        load_values(i);
        __builtin_amdgcn_sched_barrier(0);  // or they are put off until they are needed
        sc[0] += odd;
        uint32_t bad = 0;  // tokens of a masked tile with values that are not finite
        if (t0 + KT > r.w_least) {
            const int32_t seen = static_cast<int32_t>(r.visible) - static_cast<int32_t>(t0 + 4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t t = 8 * (e / 4) + e % 4;
                if (static_cast<int32_t>(t) >= seen) sc[0][e] = -INFINITY;
                bool f = true;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    f = f && finite(vf[e].v[c]);
                    vf[e].v[c] = finite(vf[e].v[c]) ? vf[e].v[c] : 0.0f;
                }
                const uint64_t not_f = __ballot(!f);
                bad |= (static_cast<uint32_t>(not_f) ? 1u << t : 0u) | (not_f >> 32 ? 1u << (t + 4) : 0u);
            }
        }
        float p[1][16];
        softmax_tile(sc, soft, p, acc, i == part, r.visible > t0, AGAIN ? 0.0f : kMost<float>);
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[e].v[c], p[0][e], acc[c], 0, 0, 0);
        load_keys(min(i + KW, count - 1));  // past the last tile too: how many loads are in flight does not depend on a branch
        for (; bad; bad &= bad - 1) {
            const uint32_t t = t0 + __ffs(static_cast<int>(bad)) - 1;
            if (t >= r.visible) continue;
            const float *row = values + static_cast<size_t>(t) * a.value_stride;
            uint32_t d = a.head_dim;
            asm("" : "+s"(d));
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t ch = C * (8 * (e / 4) + 4 * h + e % 4) + c;
                    if (ch < d && !finite(row[ch])) acc[c][e] += row[ch];
                }
        }
    }

    if (!AGAIN && past_range(acc)) again_wanted = 1;
    const uint32_t late = lane_anew(), token = rows[late % 32].x, at = rows[late % 32].y;
    const uint32_t visible = b.row0 + late % 32 <= b.last ? token + 1 : 0u;
    if (join_parts<C, 1, kWaves>(lds, wave, late, visible > part * KT, soft, acc) && visible > 0) {
        const float inv = 1.0f / soft.sum;
        float *dst = static_cast<float *>(a.output) + static_cast<size_t>(b.q.row + token) * a.output_stride + at;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t ch = C * (8 * (e / 4) + 4 * (late / 32) + e % 4);
            float sums[C];
#pragma unroll
            for (int c = 0; c < C; ++c) sums[c] = acc[c][e];
            if (AGAIN) {
                mend_averages<float, C>(dst, ch, a.head_dim, sums, inv);
            } else {
                store_averages<float, C>(dst, ch, a.head_dim, sums, inv);
            }
        }
    }
    return !AGAIN && __builtin_amdgcn_readfirstlane(again_wanted);
}

template <int W, bool WHOLE>
__global__ __launch_bounds__(kThreads, W <= 128 ? 2 : 1) void prompt_attention_f32_kernel(PromptArgs a) {
    __shared__ Kept kept;
    once_or_twice<&attend_block_f32<W, WHOLE, false>, &attend_block_f32<W, WHOLE, true>>(a, kept);
}

// Blocks of a batch at most: one of each sequence is not full.
uint64_t blocks_most(const PromptArgs &a, uint32_t block_rows) {
    return (static_cast<uint64_t>(a.tokens) * a.group + static_cast<uint64_t>(std::min(a.sequences, a.tokens)) * (block_rows - 1)) / block_rows;
}
template <auto KERNEL>
hipError_t launch(const PromptArgs &a, uint32_t block_rows, size_t lds, hipStream_t stream) {
    // once for each device: the call takes longer than the launch
    static std::atomic<uint64_t> ready{0};
    int id = 0;
    hipError_t e = hipGetDevice(&id);
    if (e != hipSuccess) return e;
    const uint64_t device = id < 64 ? 1ull << id : 0;
    if (!(ready.load(std::memory_order_acquire) & device)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (e != hipSuccess) return e;
        ready.fetch_or(device, std::memory_order_release);
    }
    hipLaunchKernelGGL(KERNEL, dim3(static_cast<uint32_t>(blocks_most(a, block_rows)) * a.kv_heads), dim3(kThreads), lds, stream, a);
    return hipGetLastError();
}
template <typename T, int W, int KT, int RW>
hipError_t launch_rows(const PromptArgs &a, hipStream_t stream) {
    constexpr size_t lds = std::max(2 * tile_bytes<T, W, KT>, join_bytes<W / 32, RW, kWaves>);
    static_assert(lds <= 128 * 1024, "a workgroup's LDS");
    // loads to LDS take whole chunks of 16 bytes, aligned
    const uint64_t sizes = (static_cast<uint64_t>(a.head_dim) | a.key_stride | a.value_stride) * sizeof(T) |
                           reinterpret_cast<uintptr_t>(a.key) | reinterpret_cast<uintptr_t>(a.value);
    return sizes % 16 == 0 ? launch<&prompt_attention_kernel<T, W, KT, RW, true>>(a, RW * kWaveRows, lds, stream)
                           : launch<&prompt_attention_kernel<T, W, KT, RW, false>>(a, RW * kWaveRows, lds, stream);
}
template <int W>
hipError_t launch_f32(const PromptArgs &a, hipStream_t stream) {
    constexpr size_t lds = std::max<size_t>(join_bytes<W / 32, 1, kWaves>, kWaveSize * W * 2);
    static_assert(lds <= 128 * 1024, "a workgroup's LDS");
    return a.head_dim == W ? launch<&prompt_attention_f32_kernel<W, true>>(a, kWaveRows, lds, stream)
                           : launch<&prompt_attention_f32_kernel<W, false>>(a, kWaveRows, lds, stream);
}
// Where blocks of 128 rows are too few to fill the GPU, blocks of 64 with two waves
// for the same rows.
template <typename T, int W>
hipError_t launch_width(const PromptArgs &a, hipStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        return launch_f32<W>(a, stream);
    } else {
        const uint64_t groups = blocks_most(a, 4 * kWaveRows) * a.kv_heads;
        if constexpr (W == 64) {
            if (a.tokens / a.sequences >= kLongTokens && groups < kFullGroups)
                return groups >= kManyGroups ? launch_rows<T, W, 128, 4>(a, stream) : launch_rows<T, W, 128, 2>(a, stream);
        }
        return groups >= kManyGroups ? launch_rows<T, W, W == 256 ? 32 : 64, 4>(a, stream) : launch_rows<T, W, 64, 2>(a, stream);
    }
}
template <typename T>
hipError_t launch_prompt(const PromptArgs &a, hipStream_t stream) {
    return a.head_dim <= 64 ? launch_width<T, 64>(a, stream) : a.head_dim <= 128 ? launch_width<T, 128>(a, stream) : launch_width<T, 256>(a, stream);
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API int qwn_hip_ext_prompt_attention_device(QwnCudaContextHandle *handle, const QwnHipPromptAttentionRequest *r,
                                                         void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || !r || !header_ok(*r) || r->sequences == 0 || r->tokens == 0 || !r->starts || !r->query || !r->key || !r->value ||
        !r->output || r->dtype > QWN_HIP_DTYPE_BF16 || r->query_heads == 0 || r->kv_heads == 0 || r->head_dim == 0 ||
        r->query_heads > 65535 || r->sequences > 0x7fffffu || r->tokens > 0x7fffffffu) {
        set_error("invalid prompt attention request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (r->head_dim > 256 || r->query_heads % r->kv_heads) {
        set_error("unsupported prompt attention: head_dim %u, %u query heads of %u KV heads", r->head_dim, r->query_heads, r->kv_heads);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    PromptArgs a{};
    const uint32_t q_channels = r->query_heads * r->head_dim, channels = r->kv_heads * r->head_dim;
    a.query_stride = stride_or(r->query_stride, q_channels);
    a.key_stride = stride_or(r->key_stride, channels);
    a.value_stride = stride_or(r->value_stride, channels);
    a.output_stride = stride_or(r->output_stride, q_channels);
    if (a.query_stride < q_channels || a.key_stride < channels || a.value_stride < channels || a.output_stride < q_channels) {
        set_error("prompt attention request: a row stride is shorter than its row");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t size = dtype_bytes(r->dtype), rows = r->tokens;
    const Rows out = row_block(r->output, rows, q_channels, a.output_stride, size);
    if (overlaps_any(out, {row_block(r->query, rows, q_channels, a.query_stride, size), row_block(r->key, rows, channels, a.key_stride, size),
                           row_block(r->value, rows, channels, a.value_stride, size),
                           list_of_bytes(r->starts, 4 * (static_cast<uint64_t>(r->sequences) + 1))})) {
        set_error("prompt attention: the output overlaps an input");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    a.group = r->query_heads / r->kv_heads;
    // rows are counted in 32 bits, the threads of a launch, too
    const uint64_t all = rows * a.group;
    if (all > 0x7fffffffu || (all / kWaveRows + std::min(r->sequences, r->tokens)) * r->kv_heads > 0xffffffffu / kThreads) {
        set_error("prompt attention: %u tokens of %u heads are too many for one call", r->tokens, r->query_heads);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("prompt attention device", device.error());
    a.query = r->query;
    a.key = r->key;
    a.value = r->value;
    a.output = r->output;
    a.starts = r->starts;
    a.sequences = r->sequences;
    a.tokens = r->tokens;
    a.kv_heads = r->kv_heads;
    a.head_dim = r->head_dim;
    a.scale = r->scale;
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_prompt<float>(a, s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_prompt<f16>(a, s)
                                                         : launch_prompt<bf16>(a, s);
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("prompt attention launch", e);
}

}  // extern "C"
