// Attention of a ragged batch over the paged 4-bit KV cache (layout:
// qwn_paged.h).
//
//   out[row] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - max)
//
// with k_t = step_t code_t + minimum_t per group of 64 channels.  The codes
// are small integers, so they go to the matrix cores as they are, exact in
// f16, and steps and minima are applied to sums:
//
//   q.k_t  = sum_g step_gt (q_g . code_gt) + minimum_gt (sum of q_g)
//   sum_t p_t v_t = sum_t (p_t step_gt) code_t + sum_t p_t minimum_gt
//
// Scores are computed transposed, S^T = codes Q^T (v_mfma_f32_16x16x32_f16):
// a lane then holds, of one query row, the tokens 4 g .. 4 g + 3 of a tile,
// which is what the second product O^T = codes^T P^T takes of its right
// operand: the probabilities go from one product to the other in their
// registers.
//
// fp32 queries and probabilities are split into two f16 halves (22 bits, two
// products); f16 and bf16 ones take one.  Queries are first divided by a power
// of two per row, probabilities by one per wave that covers the values' steps,
// so that neither halves nor rounded values leave the range of f16.
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_paged.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace qwn;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWaveSize;
constexpr uint32_t kRows = 16;                    // query rows of a block: the matrix cores' columns
constexpr uint32_t kStep = 32;                    // tokens of a wave's step
constexpr uint32_t kPiece = kStep * kWaves;       // tokens of a workgroup's step: the unit work is split in
constexpr uint32_t kMostSlots = 0x7fffff80u;     // of a sequence: slot numbers stay in 32 bits
constexpr uint32_t kWorkers = 512;                // workgroups: two of four waves on each CU

struct AttnArgs {
    PagedKv c;
    PagedBatch b;
    const void *query;
    void *output;
    float *part_o;       // [worker][2][kRows][width]
    float2 *part_ml;     // [worker][2][kRows]: reference exponent, sum
    uint32_t query_stride, output_stride, query_heads, group;
    float scale;
};

// Work is a list of pieces of kPiece tokens: for each sequence, each block of
// kRows query rows (a row is a token and one of the query heads of a KV head),
// each KV head, the pieces of its context in order.  Worker w of W takes the
// w-th share of the list, whatever the lengths of the sequences.
struct Shape {
    uint32_t blocks, pieces;  // of a sequence: row blocks, pieces of one block and head
};
__device__ __forceinline__ Shape shape_of(const AttnArgs &a, uint32_t s) {
    const PagedSequence q = paged_sequence(a.b, s);
    Shape r;
    r.blocks = static_cast<uint32_t>((static_cast<uint64_t>(q.rows) * a.group + kRows - 1) / kRows);
    // slots past the table are attended to by none
    const uint64_t slots = min(min(static_cast<uint64_t>(q.past) + q.rows,
                                   static_cast<uint64_t>(a.b.table_stride) << a.c.page_shift),
                               static_cast<uint64_t>(kMostSlots));
    r.pieces = q.rows ? static_cast<uint32_t>((slots + kPiece - 1) / kPiece) : 0u;
    return r;
}

// 64-bit prefix over the batch, 64 sequences a step: the sequence that holds
// piece `index`, the pieces before it, and the whole list's length.
struct Place {
    uint32_t seq;
    uint64_t before;
};
__device__ __forceinline__ uint64_t scan64(uint64_t v) {
    const uint32_t lane = threadIdx.x % kWaveSize;
#pragma unroll
    for (int off = 1; off < kWaveSize; off <<= 1) {
        const uint64_t o = __shfl_up(v, off);
        if (lane >= static_cast<uint32_t>(off)) v += o;
    }
    return v;
}
__device__ __forceinline__ uint64_t pieces_of(const AttnArgs &a, uint32_t s) {
    const Shape h = shape_of(a, s);
    return static_cast<uint64_t>(h.blocks) * a.c.kv_heads * h.pieces;
}
__device__ __forceinline__ uint64_t total_pieces(const AttnArgs &a) {
    uint64_t n = 0;
    for (uint32_t s0 = 0; s0 < a.b.sequences; s0 += kWaveSize) {
        const uint32_t s = s0 + threadIdx.x % kWaveSize;
        if (s < a.b.sequences) n += pieces_of(a, s);
    }
    for (int off = kWaveSize / 2; off > 0; off >>= 1) n += __shfl_xor(n, off);
    return n;
}
__device__ __forceinline__ Place find_piece(const AttnArgs &a, uint64_t index) {
    uint64_t before = 0;
    for (uint32_t s0 = 0; s0 < a.b.sequences; s0 += kWaveSize) {
        const uint32_t s = s0 + threadIdx.x % kWaveSize;
        const uint64_t n = s < a.b.sequences ? pieces_of(a, s) : 0ull;
        const uint64_t end = before + scan64(n);
        const uint64_t past = __ballot(end > index);
        if (past) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            return {s0 + first, __shfl(end, first) - __shfl(n, first)};
        }
        before = __shfl(end, kWaveSize - 1);
    }
    return {a.b.sequences, before};
}

__device__ __forceinline__ uint64_t share(uint64_t total, uint32_t w) { return paged_share(total, kWorkers, w); }

// Half b (0: nibbles 0 .. 3, 1: 4 .. 7) pairs of a code word as f16: nibbles
// p and p + 4 in the two halves of a register.  1024 + code is the f16 with
// the code in its last bits.
__device__ __forceinline__ v2h codes2(uint32_t word, int p) {
    const uint32_t bits = ((word >> (4 * p)) & 0x000f000fu) | 0x64006400u;
    const v2h base = {static_cast<_Float16>(1024.0f), static_cast<_Float16>(1024.0f)};
    return __builtin_bit_cast(v2h, bits) - base;
}
__device__ __forceinline__ v8h codes8(uint32_t word) {
    const v2h a = codes2(word, 0), b = codes2(word, 1), c = codes2(word, 2), d = codes2(word, 3);
    return (v8h){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x as NP halves that add up to it.
template <int NP>
struct Halves {
    v8h p[NP];
};
template <int NP>
__device__ __forceinline__ Halves<NP> halves(const float x[8]) {
    Halves<NP> h;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const _Float16 hi = static_cast<_Float16>(x[i]);
        h.p[0][i] = hi;
        if constexpr (NP == 2) h.p[1][i] = static_cast<_Float16>(x[i] - static_cast<float>(hi));
    }
    return h;
}

__device__ __forceinline__ float across_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// What a lane reads of a step's two tiles.
template <int W>
struct Tiles {
    uint32_t k[2][W / 32], v[2][W / 32], ks[2][4 * (W / 64)], vs[2][4 * (W / 64)];
    bool ok[2];
};
template <int N>
__device__ __forceinline__ void load_words(uint32_t *dst, const uint8_t *src) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const v4u x = *reinterpret_cast<const v4u *>(src + 4 * i);
            dst[i] = x[0], dst[i + 1] = x[1], dst[i + 2] = x[2], dst[i + 3] = x[3];
        }
    } else {
        const v2u x = *reinterpret_cast<const v2u *>(src);
        dst[0] = x[0], dst[1] = x[1];
    }
}
template <int W>
__device__ __forceinline__ void load_tiles(const AttnArgs &a, uint32_t s, uint32_t head, uint32_t token, uint32_t lane,
                                           Tiles<W> &t) {
    constexpr int JW = W >= 128 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t slot = token + kPagedTile * i;
        uint32_t page = 0;
        t.ok[i] = paged_page(a.c, a.b, s, slot, page);
        const uint8_t *block =
            a.c.pool + paged_block_at(a.c, t.ok[i] ? page : 0u, (slot & (a.c.page_tokens - 1)) / kPagedTile, head);
#pragma unroll
        for (int j = 0; j < W / 32; j += JW) {
            load_words<JW>(t.k[i] + j, block + 4 * paged_word(W, lane, j));
            load_words<JW>(t.v[i] + j, block + paged_values_at(W) + 4 * paged_word(W, lane, j));
        }
        constexpr int G = W / 64;
        load_words<4 * G>(t.ks[i], block + paged_key_scales_at(W) + lane / 16 * (16 * G));
        load_words<4 * G>(t.vs[i], block + paged_value_scales_at(W) + lane / 16 * (16 * G));
    }
}

template <typename T, int W>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(AttnArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    constexpr int J = W / 32, G = W / 64, C = W / 16;
    constexpr int kPad = W + 4;
    __shared__ float merge_o[kWaves][kRows][kPad];
    __shared__ float2 merge_ml[kWaves][kRows];
    const uint32_t lane = threadIdx.x % kWaveSize;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const uint32_t n = lane % 16, g = lane / 16;
    const uint64_t total = total_pieces(a);
    const uint64_t begin = share(total, blockIdx.x), end = share(total, blockIdx.x + 1);
    if (begin >= end) return;
    Place at = find_piece(a, begin);
    for (uint64_t u = begin; u < end;) {
        // the block and head of piece u, and this worker's pieces of it
        Shape h = shape_of(a, at.seq);
        uint64_t in_seq = static_cast<uint64_t>(h.blocks) * a.c.kv_heads * h.pieces;
        while (u - at.before >= in_seq) {
            at.before += in_seq;
            ++at.seq;
            h = shape_of(a, at.seq);
            in_seq = static_cast<uint64_t>(h.blocks) * a.c.kv_heads * h.pieces;
        }
        const uint32_t s = at.seq;
        const PagedSequence q = paged_sequence(a.b, s);
        const uint64_t in = u - at.before;
        const uint32_t item = static_cast<uint32_t>(in / h.pieces), piece0 = static_cast<uint32_t>(in % h.pieces);
        const uint32_t block = item / a.c.kv_heads, head = item % a.c.kv_heads;
        const uint32_t count = static_cast<uint32_t>(min(static_cast<uint64_t>(h.pieces - piece0), end - u));
        const bool whole = piece0 == 0 && count == h.pieces;

        // this lane's query row (column n): token and head, its visible slots
        const uint64_t r = static_cast<uint64_t>(block) * kRows + n;
        const bool real = r < static_cast<uint64_t>(q.rows) * a.group;
        const uint32_t tok = real ? static_cast<uint32_t>(r / a.group) : 0u;
        const uint32_t qh = head * a.group + static_cast<uint32_t>(r % a.group);
        const uint32_t visible = real ? q.past + tok + 1 : 0u;
        const uint64_t last_row = min(static_cast<uint64_t>(block) * kRows + kRows, static_cast<uint64_t>(q.rows) * a.group) - 1;
        const uint32_t most = q.past + static_cast<uint32_t>(last_row / a.group) + 1;  // slots any row of the block sees
        const T *qp = static_cast<const T *>(a.query) + static_cast<size_t>(q.row + tok) * a.query_stride +
                      static_cast<size_t>(qh) * a.c.head_dim;

        Halves<NP> qf[J];
        float qsum[G], row_mul;
        {
            float x[J][8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t ch = 32 * j + 8 * g + i;
                    x[j][i] = real && ch < a.c.head_dim ? to_float(qp[ch]) : 0.0f;
                    top = fmaxf(top, fabsf(x[j][i]));
                }
            top = across_max(top);
            int e = 0;  // top < 2^e
            if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);
            e = max(e, -126);
            const float down = ldexpf(1.0f, -e);
            row_mul = a.scale * 1.44269504088896340736f * ldexpf(1.0f, e);
#pragma unroll
            for (int gg = 0; gg < G; ++gg) qsum[gg] = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[j][i] *= down;
                }
                qf[j] = halves<NP>(x[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) qsum[j / 2] += x[j][i];
            }
#pragma unroll
            for (int gg = 0; gg < G; ++gg) qsum[gg] = across_sum(qsum[gg]);
        }

        v4f acc[C];
        float low[G], sum = 0.0f, m = -INFINITY, ref = 0.0f;
        int vexp = -24;  // below every step that is not zero
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int gg = 0; gg < G; ++gg) low[gg] = 0.0f;

        const uint32_t t_end = min(most, (piece0 + count) * kPiece);
        for (uint32_t t0 = piece0 * kPiece + wave * kStep; t0 < t_end; t0 += kPiece) {
            Tiles<W> t;
            load_tiles<W>(a, s, head, t0, lane, t);
            // scores of the lane's 8 tokens
            float sc[8], step_top = 0.0f;
            bool see[8];
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                v4f d[G];
#pragma unroll
                for (int gg = 0; gg < G; ++gg) d[gg] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const v8h kc = codes8(t.k[i2][j]);
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        d[j / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qf[j].p[p], d[j / 2], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = 0.0f;
#pragma unroll
                    for (int gg = 0; gg < G; ++gg) {
                        const uint32_t w = t.ks[i2][i * G + gg];
                        x = fmaf(half_to_float(w & 0xffffu), d[gg][i], x);
                        x = fmaf(half_to_float(w >> 16), qsum[gg], x);
                    }
                    const uint32_t slot = t0 + kPagedTile * i2 + 4 * g + i;
                    see[4 * i2 + i] = t.ok[i2] && slot < visible;
                    sc[4 * i2 + i] = see[4 * i2 + i] ? x * row_mul : -INFINITY;
                    // tokens that no row sees may hold anything
                    const bool live = t.ok[i2] && slot < most;
#pragma unroll
                    for (int gg = 0; gg < G; ++gg) {
                        if (!live) t.vs[i2][i * G + gg] = 0;
                        step_top = fmaxf(step_top, half_to_float(t.vs[i2][i * G + gg] & 0xffffu));
                    }
                }
            }
            float mx = m;
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sc[i]);
            mx = across_max(mx);
            step_top = across_max(step_top);
            const int e = static_cast<int>(__builtin_bit_cast(uint32_t, step_top) >> 23) - 126;  // steps < 2^e
            const int ve = max(vexp, e);
            const float next = mx == -INFINITY ? 0.0f : mx + static_cast<float>(ve);
            if (__any(mx > m || ve > vexp)) {
                // nothing seen yet: sums of zeros, whatever the reference was
                const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref - next);
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] *= alpha;
#pragma unroll
                for (int gg = 0; gg < G; ++gg) low[gg] *= alpha;
                sum *= alpha;
                m = mx;
                vexp = ve;
                ref = next;
            }
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(sc[i] - ref);
                sum += p[i];
            }
            Halves<NP> pf[G];
#pragma unroll
            for (int gg = 0; gg < G; ++gg) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = t.vs[i / 4][(i % 4) * G + gg];
                    x[i] = p[i] * half_to_float(w & 0xffffu);
                    low[gg] = fmaf(p[i], half_to_float(w >> 16), low[gg]);
                }
                pf[gg] = halves<NP>(x);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int w = c / 2, b = (c % 2) * 2;
                const v2h x0 = codes2(t.v[0][w], b), x1 = codes2(t.v[0][w], b + 1);
                const v2h x2 = codes2(t.v[1][w], b), x3 = codes2(t.v[1][w], b + 1);
                const v8h vc = {x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
#pragma unroll
                for (int k = 0; k < NP; ++k)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pf[c / 4].p[k], acc[c], 0, 0, 0);
            }
        }

        // the four waves' results of the block: lane (g, n) has channels
        // 16 c + 4 g .. + 3 of row n
        sum = across_sum(sum);
#pragma unroll
        for (int gg = 0; gg < G; ++gg) low[gg] = across_sum(low[gg]);
        __syncthreads();  // the previous block's results are read
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const v4f o = acc[c] + low[c / 4];
            *reinterpret_cast<v4f *>(&merge_o[wave][n][16 * c + 4 * g]) = o;
        }
        if (g == 0) merge_ml[wave][n] = make_float2(m == -INFINITY ? -INFINITY : ref, sum);
        __syncthreads();
        const uint32_t part = paged_partial(total, kWorkers, u - piece0, blockIdx.x);
        for (uint32_t i = threadIdx.x; i < kRows * W; i += kThreads) {
            const uint32_t row = i / W, ch = i % W;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, merge_ml[w][row].x);
            const float base = top == -INFINITY ? 0.0f : top;
            float o = 0.0f, l = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(merge_ml[w][row].x - base);
                o = fmaf(merge_o[w][row][ch], f, o);
                l = fmaf(merge_ml[w][row].y, f, l);
            }
            const uint64_t rr = static_cast<uint64_t>(block) * kRows + row;
            if (rr >= static_cast<uint64_t>(q.rows) * a.group) continue;
            if (whole) {
                if (ch < a.c.head_dim) {
                    T *dst = static_cast<T *>(a.output) + (static_cast<size_t>(q.row) + rr / a.group) * a.output_stride +
                             static_cast<size_t>(head * a.group + rr % a.group) * a.c.head_dim;
                    dst[ch] = from_float<T>(l == 0.0f ? 0.0f : o / l);
                }
            } else {
                const size_t at_part = static_cast<size_t>(part) * kRows + row;
                a.part_o[at_part * W + ch] = o;
                if (ch == 0) a.part_ml[at_part] = make_float2(top, l);
            }
        }
        u += count;
    }
}

// Blocks that several workers shared: their partial sums joined.  grid (row
// blocks of the batch at most, KV heads).
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(AttnArgs a) {
    uint32_t s, block;
    if (!find_in(a.b, blockIdx.x, [&](uint32_t i) { return shape_of(a, i).blocks; }, s, block)) return;
    const uint32_t head = blockIdx.y;
    const uint64_t total = total_pieces(a);
    uint64_t before = 0;
    for (uint32_t s0 = 0; s0 < s; s0 += kWaveSize) {
        const uint32_t i = s0 + threadIdx.x % kWaveSize;
        uint64_t v = i < s ? pieces_of(a, i) : 0ull;
        for (int off = kWaveSize / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
        before += v;
    }
    const Shape h = shape_of(a, s);
    const PagedSequence q = paged_sequence(a.b, s);
    const uint64_t first = before + (static_cast<uint64_t>(block) * a.c.kv_heads + head) * h.pieces;
    const uint32_t w0 = paged_worker(total, kWorkers, first), w1 = paged_worker(total, kWorkers, first + h.pieces - 1);
    if (w0 == w1) return;  // one worker had it all, and wrote it
    const uint64_t rows = min(static_cast<uint64_t>(kRows), static_cast<uint64_t>(q.rows) * a.group - static_cast<uint64_t>(block) * kRows);
    for (uint32_t i = threadIdx.x; i < rows * W; i += kThreads) {
        const uint32_t row = i / W, ch = i % W;
        float top = -INFINITY;
        for (uint32_t w = w0; w <= w1; ++w)
            if (share(total, w) < share(total, w + 1))
                top = fmaxf(top, a.part_ml[static_cast<size_t>(paged_partial(total, kWorkers, first, w)) * kRows + row].x);
        const float base = top == -INFINITY ? 0.0f : top;
        float o = 0.0f, l = 0.0f;
        for (uint32_t w = w0; w <= w1; ++w) {
            if (share(total, w) >= share(total, w + 1)) continue;
            const size_t at = static_cast<size_t>(paged_partial(total, kWorkers, first, w)) * kRows + row;
            const float2 ml = a.part_ml[at];
            const float f = __builtin_amdgcn_exp2f(ml.x - base);
            o = fmaf(a.part_o[at * W + ch], f, o);
            l = fmaf(ml.y, f, l);
        }
        if (ch < a.c.head_dim) {
            const uint64_t rr = static_cast<uint64_t>(block) * kRows + row;
            T *dst = static_cast<T *>(a.output) + (static_cast<size_t>(q.row) + rr / a.group) * a.output_stride +
                     static_cast<size_t>(head * a.group + rr % a.group) * a.c.head_dim;
            dst[ch] = from_float<T>(l == 0.0f ? 0.0f : o / l);
        }
    }
}

size_t partial_bytes(uint32_t width) {
    return static_cast<size_t>(kWorkers) * 2 * kRows * (width * sizeof(float) + sizeof(float2));
}

template <typename T, int W>
hipError_t launch_width(const AttnArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attention_kernel<T, W>), dim3(kWorkers), dim3(kThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // a sequence's rows fill blocks but for its last one
    const uint64_t rows = static_cast<uint64_t>(a.b.tokens) * a.group;
    const uint64_t blocks = std::min<uint64_t>(rows, rows / kRows + std::min(a.b.sequences, a.b.tokens));
    if (blocks > 0x7fffffffu) return hipErrorInvalidValue;
    hipLaunchKernelGGL((paged_merge_kernel<T, W>), dim3(static_cast<uint32_t>(blocks), a.c.kv_heads), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_paged_attention(const AttnArgs &a, hipStream_t stream) {
    return a.c.width == 64    ? launch_width<T, 64>(a, stream)
           : a.c.width == 128 ? launch_width<T, 128>(a, stream)
                              : launch_width<T, 256>(a, stream);
}

// The request as the kernels take it (lock held): what a workspace is sized
// from and what a call runs on are checked alike.
ResidentPaged *attention_of(Context *ctx, const QwnHipPagedKvHandle *h, const QwnHipPagedAttentionRequest *r, AttnArgs &a) {
    if (!h || !r || !header_ok(*r) || !batch_of(r->batch, a.b) || r->dtype > QWN_HIP_DTYPE_BF16 || r->query_heads == 0 ||
        r->query_heads > 65535)
        return nullptr;
    ResidentPaged *rp = paged_of(ctx, *h);
    if (!rp || r->query_heads % rp->c.kv_heads) return nullptr;
    a.c = rp->c;
    a.query_heads = r->query_heads;
    a.group = r->query_heads / rp->c.kv_heads;
    const uint32_t channels = r->query_heads * rp->c.head_dim;
    a.query_stride = stride_or(r->query_stride, channels);
    a.output_stride = stride_or(r->output_stride, channels);
    return a.query_stride < channels || a.output_stride < channels ? nullptr : rp;
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API uint64_t qwn_hip_ext_paged_kv_attention_workspace_bytes(QwnCudaContextHandle *handle,
                                                                         QwnHipPagedKvHandle *h,
                                                                         const QwnHipPagedAttentionRequest *r) {
    Context *ctx = context_of(handle);
    if (!ctx) return 0;
    std::lock_guard<std::mutex> lock(ctx->mutex);
    AttnArgs a{};
    return attention_of(ctx, h, r, a) ? partial_bytes(a.c.width) : 0;
}

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_attention_device(QwnCudaContextHandle *handle, QwnHipPagedKvHandle *h,
                                                           const QwnHipPagedAttentionRequest *r, void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx) {
        set_error("invalid paged attention request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    AttnArgs a{};
    if (!attention_of(ctx, h, r, a) || !r->query || !r->output || !r->workspace) {
        set_error("invalid paged attention request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(r->workspace) & 15u) {
        set_error("paged attention workspace must be 16-byte aligned");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("paged attention device", device.error());
    a.query = r->query;
    a.output = r->output;
    a.scale = r->scale;
    a.part_ml = static_cast<float2 *>(r->workspace);
    a.part_o = reinterpret_cast<float *>(a.part_ml + static_cast<size_t>(kWorkers) * 2 * kRows);
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_paged_attention<float>(a, s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_paged_attention<f16>(a, s)
                                                         : launch_paged_attention<bf16>(a, s);
    if (e != hipSuccess) return hip_fail("paged attention launch", e);
    ctx->telemetry.kv_cache_kernel_count++;
    return QWN_CUDA_STATUS_OK;
}

}  // extern "C"
