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
// second product (bf16 2^-9, f16 2^-12 of each, which averages out over the
// tokens: below the rounding of the output), and fp32 goes in fp32 throughout.
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace qwn;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr uint32_t kWaves = 4, kThreads = kWaves * kWaveSize;
constexpr uint32_t kWaveRows = 32, kBlockRows = kWaves * kWaveRows;
constexpr float kFar = 0x1p20f;               // of references: past it their rounding would be more than 2^-4 of an exponent

struct PromptArgs {
    const void *query, *key, *value;
    void *output;
    const int32_t *starts;
    uint32_t sequences, tokens, kv_heads, group, head_dim;
    uint32_t query_stride, key_stride, value_stride, output_stride;
    float scale;
};

// The two 16-bit types' operands and products; of fp32 a lane's operand is one number.
template <typename T>
struct Matrix;
template <>
struct Matrix<f16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ v16f mul(frag a, frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static constexpr int kQueryBits = 15;  // |query| < 2^15: products below 2^40
    static constexpr float kMost = 0x1p15f;  // what a lane's probabilities of a tile may add up to: none passes f16
};
template <>
struct Matrix<bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ v16f mul(frag a, frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static constexpr int kQueryBits = -9;  // |query| < 2^-9: products with any finite key below 2^127
    static constexpr float kMost = 0x1p40f;
};
template <>
struct Matrix<float> {
    typedef float frag __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ v16f mul(float a, float b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
    static constexpr int kQueryBits = -9;
    static constexpr float kMost = 0x1p40f;
};

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
__device__ __forceinline__ bool find_block(const PromptArgs &a, uint32_t index, Span &q, uint32_t &at) {
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += kWaveSize) {
        const Span mine = span_of(a, s0 + threadIdx.x % kWaveSize);
        const uint32_t n = (mine.rows * a.group + kBlockRows - 1) / kBlockRows, end = wave_scan(n);
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
// by to be exponents of 2: positive, the scale's sign is the queries'.  Below
// 2^-100 all scores are alike; past fp32 the largest fp32 stands in its place.
__device__ __forceinline__ float exponents_of(float scale, int bits, float &up) {
    const float mul = fminf(ldexpf(fabsf(scale), bits) * 1.44269504088896340736f, 3.402823466e38f);
    const bool alike = mul < 0x1p-100f;
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
// of the other buffer; it does not count them: wait_vmcnt does.
__device__ __forceinline__ void load_to_lds(const void *from, v4u *to) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(from) : "memory");
}
template <typename T>
__device__ __forceinline__ bool finite(T v) {
    if constexpr (sizeof(T) == 4) {
        return (__builtin_bit_cast(uint32_t, v) & 0x7f800000u) != 0x7f800000u;
    } else {
        constexpr uint16_t kExponent = std::is_same_v<T, f16> ? 0x7c00u : 0x7f80u;
        return (__builtin_bit_cast(uint16_t, v) & kExponent) != kExponent;
    }
}

__device__ const uint4 kZeros = {0, 0, 0, 0};  // what channels past the head's are loaded from

// A workgroup takes 128 rows of a KV head, 32 a wave, and goes through the tiles
// of its context; two buffers of LDS, one worked on while the other is filled
// (DIRECT, of whole aligned chunks: by loads that go to LDS; else through registers).
// Exponents are taken from a reference, the row's largest product in its first
// tile: where a later tile's probabilities add up to more than kMost, the
// reference is moved to what is largest then, so other tiles need no maximum.  Masked
// tokens have probability 0; so that 0 times a value that is not finite does
// not reach rows that do not see it, such values are taken as 0 in the tiles that
// are masked and added to the rows that see them.
template <typename T, int W, int KT, bool DIRECT>
__global__ __launch_bounds__(kThreads, W == 256 ? 1 : 2) void prompt_attention_kernel(PromptArgs a) {
    using M = Matrix<T>;
    using L = Tile<T, W>;
    constexpr uint32_t CE = L::CE, NC = L::NC;
    constexpr uint32_t kChunks = KT * NC, kOfThread = kChunks / kThreads;
    constexpr int C = W / 32, S = KT / 32, J = NC / 2;
    static_assert(kChunks % kThreads == 0, "whole rounds of loads");
    extern __shared__ v4u tiles[];          // two buffers of keys, then values
    constexpr uint32_t kMasked = kBlockRows / KT + 2;
    __shared__ uint32_t odd[kMasked][KT / 32];  // of the masked tiles: tokens with values that are not finite
    const uint32_t tid = threadIdx.x, lane = tid % kWaveSize, wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
    const uint32_t n = lane % 32, h = lane / 32;
    const uint32_t head = blockIdx.x % a.kv_heads;
    Span q;
    uint32_t at;
    if (!find_block(a, blockIdx.x / a.kv_heads, q, at)) return;
    const uint32_t all = q.rows * a.group, blocks = (all + kBlockRows - 1) / kBlockRows;
    const uint32_t row0 = (blocks - 1 - at) * kBlockRows;  // a sequence's longest contexts first
    const uint32_t last = min(row0 + kBlockRows, all) - 1;
    const uint32_t most = last / a.group + 1;              // tokens that any row sees
    const uint32_t least = row0 / a.group + 1;             // and every one
    const uint32_t count = (most + KT - 1) / KT, masked = least / KT;  // tiles, and the first that not every row sees all of
    const T *keys = static_cast<const T *>(a.key) + static_cast<size_t>(q.row) * a.key_stride + head * a.head_dim;
    const T *values = static_cast<const T *>(a.value) + static_cast<size_t>(q.row) * a.value_stride + head * a.head_dim;

    // chunk x of a tile in LDS: its token and place; tokens past the last are the last
    v4u kr[kOfThread], vr[kOfThread];
    auto bring = [&](uint32_t i) {
        v4u *buf = tiles + i % 2 * 2 * kChunks;
#pragma unroll
        for (uint32_t e = 0; e < kOfThread; ++e) {
            const uint32_t x = tid + kThreads * e, t = min(i * KT + x / NC, most - 1), c = (x % NC ^ L::spread(x / NC)) * CE;
            const T *k = keys + static_cast<size_t>(t) * a.key_stride, *v = values + static_cast<size_t>(t) * a.value_stride;
            if constexpr (DIRECT) {
                const bool in = c < a.head_dim;
                v4u *to = buf + kThreads * e + wave * kWaveSize;
                const void *kp = in ? static_cast<const void *>(k + c) : &kZeros, *vp = in ? static_cast<const void *>(v + c) : &kZeros;
                load_to_lds(kp, to);
                load_to_lds(vp, to + kChunks);
            } else {
                kr[e] = load_chunk(k, c, a.head_dim);
                vr[e] = load_chunk(v, c, a.head_dim);
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
    bring(0);

    // this lane's row, as a column of the products
    const uint32_t w_row0 = row0 + wave * kWaveRows, r = w_row0 + n;
    const bool real = r <= last;
    const uint32_t rr = min(r, last), tok = rr / a.group;
    const uint32_t visible = real ? tok + 1 : 0u;
    const bool idle = w_row0 > last;
    const uint32_t w_most = idle ? 0u : min(w_row0 + kWaveRows - 1, last) / a.group + 1, w_least = idle ? 0u : w_row0 / a.group + 1;
    typename M::frag qf[J];
    float mul;
    {
        const T *qp = static_cast<const T *>(a.query) + static_cast<size_t>(q.row + tok) * a.query_stride +
                      static_cast<size_t>(head * a.group + rr % a.group) * a.head_dim;
        Vec<T, CE> raw[J];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) raw[j] = __builtin_bit_cast(Vec<T, CE>, load_chunk(qp, (2 * j + h) * CE, a.head_dim));
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (uint32_t e = 0; e < CE; ++e) top = fmaxf(top, fabsf(to_float(raw[j].v[e])));
        top = halves_max(top);
        int e2 = 0;  // top < 2^e2
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e2);
        e2 = max(e2, -100);
        float up = ldexpf(1.0f, M::kQueryBits - e2);
        mul = exponents_of(a.scale, e2 - M::kQueryBits, up);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            Vec<T, CE> x;
#pragma unroll
            for (uint32_t e = 0; e < CE; ++e) x.v[e] = from_float<T>(to_float(raw[j].v[e]) * up);
            qf[j] = __builtin_bit_cast(typename M::frag, x);
        }
    }
    if (tid < kMasked * (KT / 32)) odd[tid / (KT / 32)][tid % (KT / 32)] = 0;

    v16f acc[C];
    // the reference as a product, and times mul; far: some row's is too far to be rounded
    float m = 0.0f, ref = 0.0f, sum = 0.0f;
    bool far = false;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;

    for (uint32_t i = 0; i < count; ++i) {
        settle(i);  // tile i is there, and the other buffer is free
        if (i >= masked) clean(i);
        if (i + 1 < count) bring(i + 1);
        const uint32_t t0 = i * KT;
        if (t0 >= w_most) continue;
        const v4u *kt = tiles + i % 2 * 2 * kChunks, *vt = kt + kChunks;
        v16f sc[S];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const typename M::frag kf = __builtin_bit_cast(typename M::frag, kt[L::at(32 * s + n, 2 * j + h)]);
                if (j == 0)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[s][e] = 0.0f;
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[s] = M::mul(kf[e], qf[j][e], sc[s]);
                } else {
                    sc[s] = M::mul(kf, qf[j], sc[s]);
                }
            }
        // element e of sc[s]: token 32 s + 8 (e / 4) + 4 h + e % 4 of the tile
        if (t0 + KT > w_least) {
            const int32_t seen = static_cast<int32_t>(visible) - static_cast<int32_t>(t0 + 4 * h);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * s + 8 * (e / 4) + e % 4 >= seen) sc[s][e] = -INFINITY;
        }
        auto largest = [&] {
            float mx = sc[0][0];
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[s][e]);
            return halves_max(mx);
        };
        if (i == 0) {
            m = real ? largest() : 0.0f;
            ref = mul_rounded(m, mul);
            far = __any(!(fabsf(ref) < kFar));
        }
        float p[S][16], add;
        auto weigh = [&] {
            add = 0.0f;
            if (far) {  // of rows with a far reference the product is taken off first
                const bool mine = !(fabsf(ref) < kFar);
                const float off = mine ? m : 0.0f, less = mine ? 0.0f : ref;
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        p[s][e] = __builtin_amdgcn_exp2f(fmaf(sc[s][e] - off, mul, -less));
                        add += p[s][e];
                    }
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        p[s][e] = __builtin_amdgcn_exp2f(fmaf(sc[s][e], mul, -ref));
                        add += p[s][e];
                    }
            }
        };
        weigh();
        if (__any(!(add < M::kMost))) {
            // of the rows that pass it, which does not depend on other rows
            const bool over = halves_max(add < M::kMost ? 0.0f : 1.0f) > 0.0f;
            const float mx = over ? fmaxf(m, largest()) : m, to = mul_rounded(mx, mul);
            // what exponents were taken from, and are now: of near references
            // themselves, else the product times mul, as it is
            const bool was = fabsf(ref) < kFar, is = fabsf(to) < kFar;
            const float alpha = __builtin_amdgcn_exp2f(was ? (is ? ref - to : fmaf(-mx, mul, ref)) : is ? fmaf(m, mul, -to) : (m - mx) * mul);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] *= alpha;
            sum *= alpha;
            m = mx;
            ref = to;
            far = __any(!is);
            weigh();
        }
        sum += add;
        if constexpr (sizeof(T) == 4) {
            const float *v = reinterpret_cast<const float *>(vt);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t t = 32 * s + 8 * (e / 4) + e % 4 + 4 * h;
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        acc[c] = M::mul(v[4 * L::at(t, (32 * c + n) / 4) + n % 4], p[s][e], acc[c]);
                }
        } else {
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
                    // rows of V^T: of 16 lanes each, 4 tokens of 16 channels
                    const uint32_t t = 32 * s + 16 * u + 4 * h + lane % 16 / 4;
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const uint32_t ch = 4 * c + 2 * (lane / 16 % 2) + lane % 4 / 2;
                        typedef __attribute__((address_space(3))) v4s lds_v4s;
                        union {
                            v4s part[2];
                            typename M::frag whole;
                        } x;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint16_t *from = reinterpret_cast<const uint16_t *>(vt + L::at(t + 8 * k, ch)) + 4 * (lane % 2);
                            x.part[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(from));
                        }
                        acc[c] = M::mul(x.whole, pf, acc[c]);
                    }
                }
        }
        if (i >= masked) {
#pragma unroll 1
            for (int s = 0; s < S; ++s)
                for (uint32_t left = odd[i - masked][s]; left; left &= left - 1) {
                    const uint32_t t = t0 + 32 * s + __ffs(static_cast<int>(left)) - 1;
                    if (t >= visible) continue;
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

    if (!real) return;
    const float inv = 1.0f / halves_sum(sum);
    T *dst = static_cast<T *>(a.output) + static_cast<size_t>(q.row + tok) * a.output_stride +
             static_cast<size_t>(head * a.group + rr % a.group) * a.head_dim;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const uint32_t ch = 32 * c + 8 * (e / 4) + 4 * h;
            Vec<T, 4> y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y.v[k] = from_float<T>(acc[c][e + k] * inv);
            if (ch + 4 <= a.head_dim) {
                store_vec<T, 4>(dst + ch, y);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (ch + k < a.head_dim) dst[ch + k] = y.v[k];
            }
        }
}

template <typename T, int W, int KT, bool DIRECT>
hipError_t launch_loads(const PromptArgs &a, hipStream_t stream) {
    constexpr size_t lds = 2 * 2 * KT * W * sizeof(T);
    static_assert(lds <= 128 * 1024, "a workgroup's LDS");
    const void *kernel = reinterpret_cast<const void *>(&prompt_attention_kernel<T, W, KT, DIRECT>);
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return e;
    // at most one block of each sequence is not full
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.group, used = std::min(a.sequences, a.tokens);
    const uint32_t blocks = static_cast<uint32_t>((rows + used * (kBlockRows - 1)) / kBlockRows);
    hipLaunchKernelGGL((prompt_attention_kernel<T, W, KT, DIRECT>), dim3(blocks * a.kv_heads), dim3(kThreads), lds, stream, a);
    return hipGetLastError();
}
template <typename T, int W, int KT>
hipError_t launch_tile(const PromptArgs &a, hipStream_t stream) {
    // loads to LDS take whole chunks of 16 bytes, aligned
    const uint64_t sizes = (static_cast<uint64_t>(a.head_dim) | a.key_stride | a.value_stride) * sizeof(T) |
                           reinterpret_cast<uintptr_t>(a.key) | reinterpret_cast<uintptr_t>(a.value);
    return sizes % 16 == 0 ? launch_loads<T, W, KT, true>(a, stream) : launch_loads<T, W, KT, false>(a, stream);
}
template <typename T>
hipError_t launch_prompt(const PromptArgs &a, hipStream_t stream) {
    if (a.head_dim <= 64) return launch_tile<T, 64, sizeof(T) == 4 ? 32 : 64>(a, stream);
    if (a.head_dim <= 128) return launch_tile<T, 128, sizeof(T) == 4 ? 32 : 64>(a, stream);
    return launch_tile<T, 256, 32>(a, stream);
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
    // rows and blocks are counted in 32 bits
    const uint64_t all = rows * a.group;
    if (all > 0x7fffffffu || (all / kBlockRows + std::min(r->sequences, r->tokens)) * r->kv_heads > 0x7fffffffu) {
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
