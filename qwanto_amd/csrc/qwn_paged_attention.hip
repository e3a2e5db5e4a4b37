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
// products); f16 and bf16 ones take one.  With one product the codes go in
// where they lie in a word, as f16 of 2^-24 and 2^-20 times their value
// (qwn_paged.h): 5 instructions for 8 codes, where making them integers takes
// 11.  The elements that meet the larger ones are divided by 16 beforehand, the
// sums multiplied by 2^24 at the end.  (The matrix cores sum such operands to
// 2e-7 of their magnitudes, integers to 5e-8: fp32 takes integers, less 8 to
// halve what cancels, and so do f16's values.)  A probability that f16 rounds
// would count its error times the code, although codes are 7.5 +- 5 and the
// values they make around zero; the sum of the rounded weights, one more product
// with a row of ones, takes 8 times that error out again.
//
// Queries are scaled by a power of two
// per row to below 2^15, probabilities times steps by one per row and wave to
// below 2^11 where their largest was met (2^15 a little past it): f16 then has
// 25 binades and more below the largest, for the second halves as well.  The
// largest product is taken off before products become exponents: rounded, its
// exponent would be off by more than f16 holds where scores pass 2^27.
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_paged.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace qwn;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWaveSize;
constexpr uint32_t kRows = 16;                    // query rows of a block: the matrix cores' columns
constexpr uint32_t kStep = 32;                    // tokens of a wave's step
constexpr uint32_t kPiece = kStep * kWaves;       // tokens of a workgroup's step: the unit work is split in
constexpr uint32_t kWorkers = 768;                // workgroups at most: three of four waves on each CU
constexpr uint32_t kStart = 3;                    // pieces that a block's beginning and end cost as much as
// Contexts are not split up to so many slots, the second where blocks are many
// (64 sequences of 1024 tokens, 8 KV heads, 20 us whole and 28 split and merged),
// or fewer with eight waves each (8 of 1000 bf16 11.5 and 14.5, fp32 14.8 and
// 15.7), for 16-bit rows down to one sequence (of 700, 10.0 and 10.9; fp32 12.4
// and 11.2).
constexpr uint32_t kWholeSlots = 512, kWholeSlotsMany = 1024, kMany = 256, kSome = 16;

constexpr int kQueryBits = 15;                   // |query| < 2^15 in f16
constexpr int kWeightBits = 11;                  // probability times step < 2^11 of the largest met,
constexpr float kSlack = 4.0f;                   // and 2^4 more before the reference moves
// The largest product where none was seen: finite, and any exponents' factor
// (2^-100 and more) takes it past kSlack from every product.
constexpr float kNothing = -3.402823466e38f;

struct AttnArgs {
    PagedKv c;
    PagedBatch b;
    const void *query;
    void *output;
    float *part_o;       // [worker][2][kRows][width]
    float4 *part_ml;     // [worker][2][kRows]: largest product, sum, what makes products exponents
    uint32_t query_stride, output_stride, query_heads, group;
    uint32_t slots;      // of a sequence's row of the table
    uint32_t workers;    // workgroups of the launch
    bool whole;
    uint32_t parts;      // of a block's context in the block kernel, at most
    float scale;
};

// Work is a list: for each sequence, each block of kRows query rows (a row is a
// token and one of the query heads of a KV head), each KV head, kStart units
// for the block itself and one for each piece of kPiece tokens of its context.
// Worker w of W takes the w-th share of the list, whatever the lengths of the
// sequences.  (61 contexts of 1 to 8191 tokens, 32 heads, 8 KV heads: 30 us,
// 44 with pieces alone, many short blocks meeting in some workers.)  Where no
// context can be long (`whole`), a worker takes a block, and nothing is merged.
struct Shape {
    uint32_t blocks, pieces, units;  // of a sequence: row blocks; pieces and units of one block and head
};
__device__ __forceinline__ Shape shape_of(const AttnArgs &a, const PagedSequence &q) {
    Shape r;
    r.blocks = (q.rows * a.group + kRows - 1) / kRows;
    // slots past the table are attended to by none
    r.pieces = (min(q.past + q.rows, a.slots) + kPiece - 1) / kPiece;
    r.units = a.whole ? 1u : kStart + r.pieces;
    return r;
}
// Where a block and head stand among a sequence's items of the list.  Heads next
// to each other, on XCDs of their own, are best where blocks hardly differ.  In
// prompts, without cuts the longest contexts come first; where they are cut and a
// prompt has little before it, its first rows see little of the context and its
// last ones all: a share of several blocks has of both, the blocks of each head
// in turn from both ends (2048 tokens, fp32: 213 us, 253 in the rows' order; four
// of 512 behind 2048 407, and 393 with heads next to each other).
template <bool PROMPT>
__device__ __forceinline__ uint32_t item_of(const AttnArgs &a, const PagedSequence &q, uint32_t blocks, uint32_t block, uint32_t head) {
    if (PROMPT && !a.whole && q.past < q.rows)
        return head * blocks + (2 * block < blocks ? 2 * block : 2 * (blocks - 1 - block) + 1);
    return (PROMPT && a.whole ? blocks - 1 - block : block) * a.c.kv_heads + head;
}
template <bool PROMPT>
__device__ __forceinline__ void place_of(const AttnArgs &a, const PagedSequence &q, uint32_t blocks, uint32_t item, uint32_t &block,
                                         uint32_t &head) {
    if (PROMPT && !a.whole && q.past < q.rows) {
        const uint32_t place = item % blocks;
        head = item / blocks;
        block = place % 2 ? blocks - 1 - place / 2 : place / 2;
    } else {
        head = item % a.c.kv_heads;
        block = PROMPT && a.whole ? blocks - 1 - item / a.c.kv_heads : item / a.c.kv_heads;
    }
}
__device__ __forceinline__ PagedSequence lane_sequence(const AttnArgs &a, uint32_t s) {
    return s < a.b.sequences ? paged_sequence(a.b, s) : PagedSequence{};
}
__device__ __forceinline__ uint32_t units_of(const AttnArgs &a, const PagedSequence &q) {
    const Shape h = shape_of(a, q);
    return h.blocks * a.c.kv_heads * h.units;
}

// The list's length, and the first 64 sequences in the lanes: what most batches
// are found by without a second look.
struct List {
    PagedSequence q;           // of lane l: sequence l,
    uint32_t n, end;           // its units, and those of the sequences up to it
    uint32_t total;
};
__device__ __forceinline__ List list_of(const AttnArgs &a) {
    List l;
    const uint32_t lane = threadIdx.x % kWaveSize;
    l.q = lane_sequence(a, lane);
    l.n = units_of(a, l.q);
    l.end = wave_scan(l.n);
    l.total = lane_of(l.end, kWaveSize - 1);
    for (uint32_t s0 = kWaveSize; s0 < a.b.sequences; s0 += kWaveSize)
        l.total += lane_of(wave_scan(units_of(a, lane_sequence(a, s0 + lane))), kWaveSize - 1);
    return l;
}
// The sequence that holds unit `index` of the list, and the units before it.
__device__ __forceinline__ PagedSequence find_place(const AttnArgs &a, const List &l, uint32_t index, uint32_t &seq,
                                                    uint32_t &before) {
    PagedSequence q = l.q;
    uint32_t n = l.n, end = l.end;
    before = 0;
    for (uint32_t s0 = 0;; ) {
        const uint64_t past = __ballot(before + end > index);
        const int first = past ? __ffsll(static_cast<unsigned long long>(past)) - 1 : kWaveSize - 1;
        if (past || s0 + kWaveSize >= a.b.sequences) {  // the second only past the list's end
            seq = s0 + first;
            before += lane_of(end, first) - lane_of(n, first);
            return PagedSequence{lane_of(q.row, first), lane_of(q.rows, first), lane_of(q.past, first)};
        }
        before += lane_of(end, kWaveSize - 1);
        s0 += kWaveSize;
        q = lane_sequence(a, s0 + threadIdx.x % kWaveSize);
        n = units_of(a, q);
        end = wave_scan(n);
    }
}

// Workgroups that get work: all, or one for each unit.
__device__ __forceinline__ uint32_t workers_of(const AttnArgs &a, uint32_t total) { return min(total, a.workers); }

// A code word's 8 codes as f16, for one product with halves (WHOLE false):
// nibbles p and p + 4 as they lie, times 2^-24 (p even) or 2^-20; for two
// products (WHOLE): the codes less 8.  1024 + code is the f16 with the code in
// its last bits.
template <bool WHOLE>
__device__ __forceinline__ v2h codes2(uint32_t word, int p) {
    if constexpr (WHOLE) {
        const v2h base = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
        return __builtin_bit_cast(v2h, ((word >> (4 * p)) & 0x000f000fu) | 0x64006400u) - base;
    }
    return __builtin_bit_cast(v2h, (p >= 2 ? word >> 8 : word) & (p % 2 ? 0x00f000f0u : 0x000f000fu));
}
template <bool WHOLE>
__device__ __forceinline__ v8h codes8(uint32_t word) {
    const v2h a = codes2<WHOLE>(word, 0), b = codes2<WHOLE>(word, 1), c = codes2<WHOLE>(word, 2), d = codes2<WHOLE>(word, 3);
    return (v8h){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// What element i of an operand that meets codes8 is multiplied by, and what
// makes up for it together with the codes' own factor.
template <bool WHOLE>
__device__ constexpr float balance(int i) { return !WHOLE && (i >> 1) % 2 ? 0.0625f : 1.0f; }

__device__ __forceinline__ v2h to_halves(float a, float b) {
    return __builtin_convertvector((v2f){a, b}, v2h);
}
__device__ __forceinline__ float step_of(uint32_t w) { return half_to_float(w >> 16); }
__device__ __forceinline__ float least_of(uint32_t w) { return half_to_float(w & 0xffffu); }

// x as NP halves that add up to it.
template <int NP>
struct Halves {
    v8h p[NP];
};
template <int NP>
__device__ __forceinline__ Halves<NP> halves(const float x[8]) {
    Halves<NP> h;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const v2h hi = to_halves(x[i], x[i + 1]);
        h.p[0][i] = hi[0], h.p[0][i + 1] = hi[1];
        if constexpr (NP == 2) {
            const v2h lo = to_halves(x[i] - static_cast<float>(hi[0]), x[i + 1] - static_cast<float>(hi[1]));
            h.p[1][i] = lo[0], h.p[1][i + 1] = lo[1];
        }
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

// A step's tiles by their pages; ok: the table names them.
struct Pages {
    uint32_t page[2];
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
// The page of a slot, 0 and false where the table names none; s and slot are
// the same in every lane.
__device__ __forceinline__ bool page_at(const AttnArgs &a, uint32_t s, uint32_t slot, uint32_t &page) {
    const uint32_t at = slot >> a.c.page_shift;
    const bool in = at < a.b.table_stride;
    const int32_t p = scalar_load(a.b.table + static_cast<size_t>(s) * a.b.table_stride + (in ? at : 0u));
    const bool ok = in && p >= 0 && static_cast<uint32_t>(p) < a.c.pages;
    page = ok ? static_cast<uint32_t>(p) : 0u;
    return ok;
}
__device__ __forceinline__ Pages find_pages(const AttnArgs &a, uint32_t s, uint32_t token) {
    Pages p;
#pragma unroll
    for (int i = 0; i < 2; ++i) p.ok[i] = page_at(a, s, token + kPagedTile * i, p.page[i]);
    return p;
}
// The keys' half of a step's tiles, or the values'.
template <int W, bool KEYS>
__device__ __forceinline__ void load_tiles(const AttnArgs &a, const Pages &p, uint32_t head, uint32_t token, uint32_t lane,
                                           uint32_t (&codes)[2][W / 32], uint32_t (&scales)[2][W / 16]) {
    constexpr int JW = W >= 128 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t tile = ((token + kPagedTile * i) & (a.c.page_tokens - 1)) / kPagedTile;
        const uint8_t *block = a.c.pool + paged_block_at(a.c, p.page[i], tile, head);
#pragma unroll
        for (int j = 0; j < W / 32; j += JW)
            load_words<JW>(codes[i] + j, block + (KEYS ? 0u : paged_values_at(W)) + 4 * paged_word(W, lane, j));
        load_words<W / 16>(scales[i], block + (KEYS ? paged_key_scales_at(W) : paged_value_scales_at(W)) + lane / 16 * (W / 4));
    }
}

// What a row's products, of queries times the power of two `up`, are multiplied
// by to be exponents of 2: positive, the scale's sign is the queries'.  Below
// 2^-100 all scores are alike, as products are below 2^40.  Past fp32 the largest
// fp32 stands in its place: products that differ (by far more than 2^-120, of
// f16 minima and steps and a row's largest query) are further apart than any
// exponent with either.
__device__ __forceinline__ float exponents_of(float scale, int bits, float &up) {
    const float mul = fminf(ldexpf(fabsf(scale), bits) * 1.44269504088896340736f, 3.402823466e38f);
    const bool alike = mul < 0x1p-100f;
    up = alike ? 0.0f : copysignf(up, scale);
    return alike ? 1.0f : mul;
}

// The 8 channels of a query row from c0, zeros past the head's.
template <typename T>
__device__ __forceinline__ void load_query(const T *row, uint32_t c0, uint32_t n, float x[8]) {
    constexpr int VEC = 16 / sizeof(T);
    if (c0 + 8 <= n) {
#pragma unroll
        for (int h = 0; h < 8; h += VEC) {
            const Vec<T, VEC> v = load_vec<T, VEC>(row + c0 + h);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[h + i] = to_float(v.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = c0 + i < n ? to_float(row[c0 + i]) : 0.0f;
    }
}

// A worker goes through its pieces block by block; in a block its four waves
// take every fourth step of 32 tokens, each with its own maxima and sums, and
// meet in LDS at the end.  A step's keys are read again as soon as the scores
// are there, its values once they are used: the other half of the step's work
// hides each, in one set of registers.  Bound by HBM in the long run, by the
// searches and loads that a block starts with where contexts are short.
template <typename T, int W, bool PROMPT, int WAVES>
__global__ __launch_bounds__(WAVES * kWaveSize, W == 256 ? 1 : WAVES == 4 ? 3 : 2) void paged_attention_kernel(AttnArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    // Keys meet a few large products, in whole codes only for fp32.  Values meet
    // many: the sum of p * code as it lies less that of p * 8 leaves 2e-4 of an
    // output that 131000 tokens average to near nothing (2.9e-4 of error become
    // 3.7e-4, output's own rounding 2.1e-4), nothing next to bf16's rounding;
    // f16's in whole codes 49 us for 48.
    constexpr bool WHOLE = NP == 2, WHOLE_V = !std::is_same_v<T, bf16>;
    constexpr int J = W / 32, G = W / 64, C = W / 16;
    constexpr int kPad = W + 4;
    constexpr uint32_t kStride = WAVES * kStep;  // tokens of the workgroup's step: a piece, but where nothing is cut
    __shared__ float merge_o[WAVES][kRows][kPad];
    __shared__ float2 merge_ml[WAVES][kRows];  // largest product, sum
    __shared__ float merge_mul[kRows];
    const uint32_t lane = threadIdx.x % kWaveSize;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const uint32_t n = lane % 16, g = lane / 16;
    const List list = list_of(a);
    const uint32_t workers = workers_of(a, list.total);
    if (blockIdx.x >= workers) return;
    const uint32_t begin = static_cast<uint32_t>(paged_share(list.total, workers, blockIdx.x));
    const uint32_t end = static_cast<uint32_t>(paged_share(list.total, workers, blockIdx.x + 1));
    uint32_t s, before;
    PagedSequence q = find_place(a, list, begin, s, before);
    for (uint32_t u = begin; u < end;) {
        // the block and head of unit u, and this worker's pieces of it
        Shape h = shape_of(a, q);
        while (u - before >= h.blocks * a.c.kv_heads * h.units) {
            before += h.blocks * a.c.kv_heads * h.units;
            if (++s >= a.b.sequences) return;  // starts that do not ascend: the list's length has wrapped
            q = sequence_of(a.b, s);
            h = shape_of(a, q);
        }
        const uint32_t item = (u - before) / h.units, at = (u - before) % h.units;
        const uint32_t first = u - at + (a.whole ? 0u : kStart);  // the unit of its first piece
        if (u < first) u = min(first, end);
        if (u == end) break;
        uint32_t block, head;
        place_of<PROMPT>(a, q, h.blocks, item, block, head);
        const uint32_t piece0 = u - first;
        const uint32_t count = a.whole ? h.pieces : min(h.pieces - piece0, end - u);
        const uint32_t rows = min(kRows, q.rows * a.group - block * kRows);
        const uint32_t most = min(q.past + (block * kRows + rows - 1) / a.group + 1, a.slots);  // slots any row sees
        const uint32_t least_seen = q.past + block * kRows / a.group + 1;                        // slots every row sees
        // of this block's rows: a prompt's first ones see nothing of the sequence's others
        const uint32_t pieces = PROMPT ? (most + kPiece - 1) / kPiece : h.pieces;
        if (PROMPT && piece0 >= pieces) {
            u += count;
            continue;
        }
        const uint32_t t_end = min(most, (piece0 + count) * kPiece);
        uint32_t t0 = piece0 * kPiece + wave * kStep;
        uint32_t k[2][J], v[2][J], ks[2][4 * G], vs[2][4 * G];
        Pages pk = find_pages(a, s, t0), pv = pk;
        load_tiles<W, true>(a, pk, head, t0, lane, k, ks);
        load_tiles<W, false>(a, pv, head, t0, lane, v, vs);
        // where nothing follows a step's loads are issued again: how many are in
        // flight does not depend on a branch, and no wait is for more than it needs
        uint32_t next = t0 + kStride < t_end ? t0 + kStride : t0;
        Pages pn = find_pages(a, s, next);

        // this lane's query row (column n): token and head, its visible slots
        const bool real = n < rows;
        const uint32_t r = block * kRows + (real ? n : 0u), tok = r / a.group;
        const uint32_t visible = real ? q.past + tok + 1 : 0u;
        const T *qp = static_cast<const T *>(a.query) + static_cast<size_t>(q.row + tok) * a.query_stride +
                      static_cast<size_t>(head * a.group + r % a.group) * a.c.head_dim;
        Halves<NP> qf[J];
        float qsum[G], row_mul;
        {
            float x[J][8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j) load_query(qp, 32 * j + 8 * g, a.c.head_dim, x[j]);
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (!real) x[j][i] = 0.0f;
                    top = fmaxf(top, fabsf(x[j][i]));
                }
            top = across_max(top);
            int e = 0;  // top < 2^e
            if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);
            e = max(e, -100);
            float up = ldexpf(1.0f, kQueryBits - e);
            row_mul = exponents_of(a.scale, e - kQueryBits + (WHOLE ? 0 : 24), up);
#pragma unroll
            for (int gg = 0; gg < G; ++gg) qsum[gg] = 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[j][i] *= up;
                    qsum[j / 2] += x[j][i];
                    x[j][i] *= balance<WHOLE>(i);
                }
                qf[j] = halves<NP>(x[j]);
            }
#pragma unroll
            for (int gg = 0; gg < G; ++gg) {
                qsum[gg] = across_sum(qsum[gg]) * (WHOLE ? 1.0f : 0x1p-24f);
                if (top == INFINITY || !isfinite(a.scale)) qsum[gg] = __builtin_nanf("");  // the row is NaN, whatever the codes are
            }
        }

        v4f acc[C], weights[G];
        // m is of the products as they come, before row_mul: below 2^40
        float low[G], sum = 0.0f, m = kNothing, up_bits = 0.0f;
        uint32_t steps = 0;  // no step of a value met so far is larger: f16 bits above, 0xffff below
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int gg = 0; gg < G; ++gg) low[gg] = 0.0f, weights[gg] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

        for (; t0 < t_end; t0 += kStride) {
            float sc[8];
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                v4f d[G];
#pragma unroll
                for (int gg = 0; gg < G; ++gg) d[gg] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const v8h kc = codes8<WHOLE>(k[i2][j]);
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        d[j / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qf[j].p[p], d[j / 2], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = 0.0f;
#pragma unroll
                    for (int gg = 0; gg < G; ++gg) {
                        const uint32_t w = ks[i2][i * G + gg];
                        x = fmaf(step_of(w), d[gg][i], x);
                        x = fmaf(WHOLE ? fmaf(8.0f, step_of(w), least_of(w)) : least_of(w), qsum[gg], x);
                    }
                    sc[4 * i2 + i] = x;
                }
            }
            const Pages pg = pv;
            const uint32_t now = next;
            pk = pn;
            load_tiles<W, true>(a, pk, head, now, lane, k, ks);
            next = t0 + 2 * kStride < t_end ? t0 + 2 * kStride : now;
            pn = find_pages(a, s, next);
            uint32_t top = 0;
            if (t0 + kStep > least_seen || !pg.ok[0] || !pg.ok[1]) {  // not all tokens for all rows
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t slot = t0 + kPagedTile * (i / 4) + 4 * g + i % 4;
                    if (!pg.ok[i / 4] || slot >= visible) sc[i] = -INFINITY;
                    // tokens that no row sees may hold any (finite) numbers
#pragma unroll
                    for (int gg = 0; gg < G; ++gg)
                        if (pg.ok[i / 4] && slot < most) top = max(top, vs[i / 4][(i % 4) * G + gg]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8 * G; ++i) top = max(top, vs[i / (4 * G)][i % (4 * G)]);
            }
            float mx = sc[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
            // a new reference only where a score is well past the last one's or a
            // step larger: rare once a few steps are done
            if (__any((mx - m) * row_mul > kSlack || top > steps)) {
                mx = across_max(fmaxf(mx, m));
                top = max(top, steps);
                top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
                top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
                steps = top | 0xffffu;
                // steps < 2^e; 2^-24 is the smallest that is not zero
                const int e = max(-24, static_cast<int>(__builtin_bit_cast(uint32_t, step_of(top)) >> 23) - 126);
                const float bits = static_cast<float>(kWeightBits - e);
                const float alpha = __builtin_amdgcn_exp2f(fmaf(m - mx, row_mul, bits - up_bits));
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] *= alpha;
#pragma unroll
                for (int gg = 0; gg < G; ++gg) low[gg] *= alpha, weights[gg] *= alpha;
                sum *= alpha;
                m = mx;
                up_bits = bits;
            }
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i] - m, row_mul, up_bits));
                sum += p[i];
            }
            Halves<NP> pf[G];
#pragma unroll
            for (int gg = 0; gg < G; ++gg) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = vs[i / 4][(i % 4) * G + gg];
                    low[gg] = fmaf(p[i], fmaf(8.0f, step_of(w), least_of(w)), low[gg]);
                    x[i] = fmaf(p[i] * balance<WHOLE_V>(i), step_of(w), 0.0f);
                }
                pf[gg] = halves<NP>(x);
                if constexpr (!WHOLE_V) {
                    const _Float16 one = static_cast<_Float16>(1.0f), more = static_cast<_Float16>(16.0f);
                    weights[gg] = __builtin_amdgcn_mfma_f32_16x16x32_f16((v8h){one, one, more, more, one, one, more, more},
                                                                        pf[gg].p[0], weights[gg], 0, 0, 0);
                }
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int w = c / 2, b = (c % 2) * 2;
                const v2h x0 = codes2<WHOLE_V>(v[0][w], b), x1 = codes2<WHOLE_V>(v[0][w], b + 1);
                const v2h x2 = codes2<WHOLE_V>(v[1][w], b), x3 = codes2<WHOLE_V>(v[1][w], b + 1);
                const v8h vc = {x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
#pragma unroll
                for (int kk = 0; kk < NP; ++kk)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pf[c / 4].p[kk], acc[c], 0, 0, 0);
            }
            pv = pk;
            load_tiles<W, false>(a, pv, head, now, lane, v, vs);
        }

        // the four waves' results of the block: lane (g, n) has channels
        // 16 c + 4 g .. + 3 of row n
        sum = across_sum(sum);
#pragma unroll
        for (int gg = 0; gg < G; ++gg) low[gg] = across_sum(low[gg]);
        const float down = ldexpf(1.0f, -static_cast<int>(up_bits));  // the largest probability is 1 again
        __syncthreads();  // the previous block's results are read
        if (real) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const v4f o = WHOLE_V ? acc[c] + low[c / 4] : acc[c] * 0x1p24f - 8.0f * weights[c / 4] + low[c / 4];
                *reinterpret_cast<v4f *>(&merge_o[wave][n][16 * c + 4 * g]) = o * down;
            }
            if (g == 0) merge_ml[wave][n] = make_float2(m, sum * down);
            if (g == 0 && wave == 0) merge_mul[n] = row_mul;
        }
        __syncthreads();
        const bool whole = piece0 == 0 && count >= pieces;
        const uint32_t part = paged_partial(list.total, workers, first, blockIdx.x);
        for (uint32_t i = threadIdx.x; i < rows * W; i += WAVES * kWaveSize) {
            const uint32_t row = i / W, ch = i % W;
            float top = kNothing;
            const float mul = merge_mul[row];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top = fmaxf(top, merge_ml[w][row].x);
            float o = 0.0f, l = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f((merge_ml[w][row].x - top) * mul);
                o = fmaf(merge_o[w][row][ch], f, o);
                l = fmaf(merge_ml[w][row].y, f, l);
            }
            if (whole) {
                const uint32_t rr = block * kRows + row;
                T *dst = static_cast<T *>(a.output) + static_cast<size_t>(q.row + rr / a.group) * a.output_stride +
                         static_cast<size_t>(head * a.group + rr % a.group) * a.c.head_dim;
                if (ch < a.c.head_dim) dst[ch] = from_float<T>(l == 0.0f ? 0.0f : o / l);
            } else {
                const size_t at_part = static_cast<size_t>(part) * kRows + row;
                a.part_o[at_part * W + ch] = o;
                if (ch == 0) a.part_ml[at_part] = make_float4(top, l, mul, 0.0f);
            }
        }
        u += a.whole ? 1u : count;
    }
}

// Blocks that several workers shared: their partial sums joined.  grid (row
// blocks of the batch at most, KV heads, parts): part z takes rows z, z + parts,
// ... of a block.  W / 4 threads hold 4 channels each of a row; where a part has
// fewer rows than the workgroup has such groups, several groups share a row's
// partials and meet in LDS.  Parts as many as the GPU holds workgroups, and no
// more than rows: 4 sequences of 8 new tokens behind up to 30000 (8 KV heads, 4
// query heads each) 30 us with 16, 36 with 4; 61 of 2 behind 4000 29 and 25.
constexpr uint32_t kMergeGroups = 2048;
template <typename T, int W, bool PROMPT>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(AttnArgs a) {
    constexpr uint32_t kLanes = W / 4, kGroups = kThreads / kLanes;
    __shared__ v4f part_o[kGroups][kLanes];
    __shared__ float2 part_ml[kGroups];
    const List list = list_of(a);
    uint32_t s, block, before = 0;
    PagedSequence q;
    if (!find_in(a.b, blockIdx.x, [&](const PagedSequence &x) { return shape_of(a, x).blocks; }, s, block, q)) return;
    const uint32_t head = blockIdx.y;
    const uint32_t total = list.total, workers = workers_of(a, total);
    if (s < kWaveSize) {
        before = lane_of(list.end, s) - lane_of(list.n, s);
    } else {
        for (uint32_t s0 = 0; s0 < s; s0 += kWaveSize) {
            const uint32_t i = s0 + threadIdx.x % kWaveSize;
            before += lane_of(wave_scan(i < s ? units_of(a, paged_sequence(a.b, i)) : 0u), kWaveSize - 1);
        }
    }
    const Shape h = shape_of(a, q);
    const uint32_t first = before + item_of<PROMPT>(a, q, h.blocks, block, head) * h.units + kStart;
    const uint32_t all = min(kRows, q.rows * a.group - block * kRows);
    const uint32_t most = min(q.past + (block * kRows + all - 1) / a.group + 1, a.slots);
    const uint32_t pieces = PROMPT ? (most + kPiece - 1) / kPiece : h.pieces;
    if (first + h.pieces > total) return;  // starts that do not ascend: the list's length has wrapped
    const uint32_t w0 = paged_worker(total, workers, first), w1 = paged_worker(total, workers, first + pieces - 1);
    if (w0 == w1) return;  // one worker had it all, and wrote it
    const uint32_t p0 = paged_partial(total, workers, first, w0), n = w1 - w0 + 1;
    if (blockIdx.z >= all) return;
    const uint32_t rows = (all - blockIdx.z + gridDim.z - 1) / gridDim.z;
    uint32_t share = 1;  // groups of a row
    while (2 * share * rows <= kGroups) share *= 2;
    const uint32_t group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, mine = group % share;
    for (uint32_t r0 = 0; r0 < rows; r0 += kGroups / share) {
        const uint32_t r = r0 + group / share, row = blockIdx.z + r * gridDim.z;
        v4f o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        float top = kNothing, l = 0.0f, mul = 1.0f;
        if (r < rows) {
#pragma unroll 4
            for (uint32_t i = mine; i < n; i += share) {
                // the first worker's partial may be its second, the others' are their first
                const size_t at = static_cast<size_t>(i ? 2 * (w0 + i) : p0) * kRows + row;
                const float4 ml = a.part_ml[at];
                const v4f x = *reinterpret_cast<const v4f *>(a.part_o + at * W + 4 * lane);
                const float next = fmaxf(top, ml.x);
                mul = ml.z;
                const float f0 = __builtin_amdgcn_exp2f((top - next) * mul), f1 = __builtin_amdgcn_exp2f((ml.x - next) * mul);
                o = o * f0 + x * f1;
                l = l * f0 + ml.y * f1;
                top = next;
            }
        }
        if (share > 1) {  // then this loop is run once
            part_o[group][lane] = o;
            if (lane == 0) part_ml[group] = make_float2(top, l);
            __syncthreads();
            if (mine != 0) continue;
            for (uint32_t i = 1; i < share; ++i) top = fmaxf(top, part_ml[group + i].x);
            o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
            l = 0.0f;
            for (uint32_t i = 0; i < share; ++i) {
                const float f = __builtin_amdgcn_exp2f((part_ml[group + i].x - top) * mul);
                o += part_o[group + i][lane] * f;
                l += part_ml[group + i].y * f;
            }
        }
        if (r >= rows) continue;
        const uint32_t rr = block * kRows + row;
        T *dst = static_cast<T *>(a.output) + static_cast<size_t>(q.row + rr / a.group) * a.output_stride +
                 static_cast<size_t>(head * a.group + rr % a.group) * a.c.head_dim;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * lane + i < a.c.head_dim) dst[4 * lane + i] = from_float<T>(l == 0.0f ? 0.0f : o[i] / l);
    }
}

// ---- many query rows ----------------------------------------------------------
//
// Prompts: a workgroup takes a block of RW x RT x 16 query rows of one KV head
// and its whole context, in chunks of 64 tokens, every other chunk for each of
// its two halves of RW waves; a wave has RT tiles of 16 rows.  Here the products
// are as many as the reads are few, and unpacking per wave would cost more than
// the products: a half's threads bring the chunk's codes to f16 values once,
// step * code + minimum rounded once, in LDS and in the order of the matrix
// cores' operands, and every wave reads them from there.  Workgroups are numbered
// by blocks, then heads: a sequence's longest contexts come first for all heads
// (a prompt of 2048 tokens, 8 KV heads, 62 us; head by head 98), and with 8 heads
// each stays on one XCD's L2.  (bf16 rows only: the rounding of keys and values,
// 2^-12 of a value, is a sixteenth of the output's.)
// With two buffers a half unpacks the next chunk while it works on this one; of
// the two waves that a SIMD holds, the first half's unpacks before its products
// and the second's after them, so that one's vector instructions meet the
// other's matrix ones.  Of a round of 128 tokens, 2.5 us, the vector ALU
// (exponentials, unpacking) issues 57 %, the matrix cores work 30 % and LDS (every
// wave reads its whole chunk) 26 %: bound by how they overlap.
constexpr uint32_t kChunk = 64;
constexpr uint32_t kChunkTiles = kChunk / kPagedTile;
constexpr uint32_t kNoPage = 0xffffffffu;
// Where a launch has fewer blocks than half the CUs, a block's context is split
// among several workgroups, each with kPartRounds rounds at least, and merged
// after (32 heads of 128: 64 tokens behind 4032 25 us, 89 whole; 512 behind 7680
// 103 us, 169 whole).  Workgroups that follow each other on a CU do not pay for
// the merge: with twice kBlockGroups the second takes 116 us and four prompts of
// 152 blocks 70, 59 whole.  Eight rounds at least: the first takes 33 us.
constexpr uint32_t kBlockGroups = 256, kBlockPartsMost = 8, kPartRounds = 4;
constexpr int kBlockWaves = 4;
constexpr int kRowBits = 8;  // probabilities up to 2^8 of the largest met, and kSlack more
constexpr float kFarRef = 0x1p12f;  // exponents up to here are rounded by 2^-12 at most

// A lane's words of one tile's keys and values, and the scales that go with them.
template <int W>
struct TileWords {
    uint32_t k[W / 32], v[W / 32], ks[W / 64], vs[W / 16];
};
template <int W>
__device__ __forceinline__ void load_tile(const AttnArgs &a, uint32_t page, uint32_t slot, uint32_t head, uint32_t lane, TileWords<W> &t) {
    constexpr int JW = W >= 128 ? 4 : 2;
    const uint8_t *block = a.c.pool + paged_block_at(a.c, page, (slot & (a.c.page_tokens - 1)) / kPagedTile, head);
#pragma unroll
    for (int j = 0; j < W / 32; j += JW) {
        load_words<JW>(t.k + j, block + 4 * paged_word(W, lane, j));
        load_words<JW>(t.v + j, block + paged_values_at(W) + 4 * paged_word(W, lane, j));
    }
#pragma unroll
    for (int j = 0; j < W / 64; ++j)
        t.ks[j] = reinterpret_cast<const uint32_t *>(block + paged_key_scales_at(W))[lane % 16 * (W / 64) + j];
    load_words<W / 16>(t.vs, block + paged_value_scales_at(W) + lane / 16 * (W / 4));
}

// Nibbles p and p + 4 of a word as step * code + minimum, of one or of two tokens.
__device__ __forceinline__ v2h values2(uint32_t word, int p, v2h step, v2h least) {
    const v2h base = {static_cast<_Float16>(1024.0f), static_cast<_Float16>(1024.0f)};
    const v2h code = __builtin_bit_cast(v2h, ((word >> (4 * p)) & 0x000f000fu) | 0x64006400u) - base;
    const v2h top = {static_cast<_Float16>(65504.0f), static_cast<_Float16>(65504.0f)};
    return __builtin_elementwise_min(__builtin_elementwise_fma(code, step, least), top);  // a step rounded up may pass f16
}
__device__ __forceinline__ v2h both(uint32_t bits) { return __builtin_bit_cast(v2h, bits); }

// The tile in LDS: keys [j][lane][8 halves], values [c][lane][half of a pair of
// tiles][4 halves].
template <int W>
__device__ __forceinline__ void unpack_tile(const TileWords<W> &t, uint32_t tile, uint32_t lane, v4u *keys, v2u *values) {
#pragma unroll
    for (int j = 0; j < W / 32; ++j) {
        const uint32_t w = t.ks[j / 2];
        const v2h step = both(__builtin_amdgcn_perm(w, w, 0x03020302u)), least = both(__builtin_amdgcn_perm(w, w, 0x01000100u));
        v4u o;
#pragma unroll
        for (int p = 0; p < 4; ++p) o[p] = __builtin_bit_cast(uint32_t, values2(t.k[j], p, step, least));
        keys[(tile * (W / 32) + j) * kWaveSize + lane] = o;
    }
#pragma unroll
    for (int g = 0; g < W / 64; ++g) {
        v2h step[2], least[2];  // of tokens 0, 1 and 2, 3
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t a = t.vs[2 * h * (W / 64) + g], b = t.vs[(2 * h + 1) * (W / 64) + g];
            step[h] = both(__builtin_amdgcn_perm(b, a, 0x07060302u));
            least[h] = both(__builtin_amdgcn_perm(b, a, 0x05040100u));
        }
#pragma unroll
        for (int w = 2 * g; w < 2 * g + 2; ++w)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                v2u o;
#pragma unroll
                for (int h = 0; h < 2; ++h) o[h] = __builtin_bit_cast(uint32_t, values2(t.v[w], 2 * c + h, step[h], least[h]));
                values[((tile / 2 * (W / 16) + 2 * w + c) * kWaveSize + lane) * 2 + tile % 2] = o;
            }
    }
}

__device__ __forceinline__ uint32_t block_parts(const AttnArgs &a, uint32_t rounds) {
    return min(a.parts, (rounds + kPartRounds - 1) / kPartRounds);
}

template <typename T, int W, int RW, int RT, int BUFFERS>
__global__ __launch_bounds__(2 * RW * kWaveSize, 2) void paged_block_attention_kernel(AttnArgs a) {
    constexpr int J = W / 32, C = W / 16;
    constexpr uint32_t kBlockRows = RW * RT * 16;
    constexpr uint32_t kTilesOfWave = kChunkTiles / RW;
    // of each half: the chunk's keys, then its values
    extern __shared__ v4u chunk[];
    constexpr uint32_t kOperands = kChunkTiles * J * kWaveSize;  // 16-byte pieces of keys, and of values
    const uint32_t lane = threadIdx.x % kWaveSize, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const uint32_t rw = wave % RW, half = wave / RW, n = lane % 16, g = lane / 16;
    uint32_t s, at;
    PagedSequence q;
    const uint32_t head = blockIdx.x % a.c.kv_heads, index = blockIdx.x / a.c.kv_heads;
    if (!find_in(a.b, index, [&](const PagedSequence &x) { return (x.rows * a.group + kBlockRows - 1) / kBlockRows; }, s, at, q))
        return;
    const uint32_t all = q.rows * a.group, blocks = (all + kBlockRows - 1) / kBlockRows;
    const uint32_t block = blocks - 1 - at;  // a sequence's longest contexts first
    const uint32_t row0 = block * kBlockRows, last = min(row0 + kBlockRows, all) - 1;
    const uint32_t most = min(q.past + last / a.group + 1, a.slots);
    const uint32_t chunks = (most + kChunk - 1) / kChunk, all_rounds = (chunks + 1) / 2;
    const uint32_t parts = block_parts(a, all_rounds);
    if (blockIdx.y >= parts) return;
    const uint32_t from = all_rounds * blockIdx.y / parts, rounds = all_rounds * (blockIdx.y + 1) / parts;
    v4u *mine = chunk + half * BUFFERS * 2 * kOperands;  // this half's buffers: keys, then values

    // the tiles this wave brings: rw, rw + RW, ... of its half's chunk.  A lane
    // holds the page of one tile of 64, and the next 64 are on their way: looking
    // a chunk's pages up in the table, a round's wait each, was a fifth of the time
    TileWords<W> words[kTilesOfWave];
    uint32_t pages[kChunkTiles], next_ok = 0;  // of the chunk to be brought next: bit i, its tile i has a page
    constexpr uint32_t kAllTiles = (1u << kChunkTiles) - 1;
    auto load_window = [&](uint32_t tile) {
        const uint32_t i = ((tile + lane) * kPagedTile) >> a.c.page_shift;
        const int32_t p = i < a.b.table_stride ? a.b.table[static_cast<size_t>(s) * a.b.table_stride + i] : -1;
        return p >= 0 && static_cast<uint32_t>(p) < a.c.pages ? static_cast<uint32_t>(p) : kNoPage;
    };
    uint32_t window_tile = 2 * from * kChunkTiles / kWaveSize * kWaveSize;
    uint32_t window = load_window(window_tile), next_window = load_window(window_tile + kWaveSize);
    // the wave's rows and their queries, on their way while the first pages are
    // looked up
    const uint32_t w_row0 = row0 + rw * RT * 16;
    uint32_t visible[RT];
    Vec<T, 8> raw[RT][J];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const uint32_t r = w_row0 + t * 16 + n;
        const uint32_t rr = min(r, last), tok = rr / a.group;
        visible[t] = r <= last ? min(q.past + tok + 1, a.slots) : 0u;
        const T *qp = static_cast<const T *>(a.query) + static_cast<size_t>(q.row + tok) * a.query_stride +
                      static_cast<size_t>(head * a.group + rr % a.group) * a.c.head_dim;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint32_t c0 = 32 * j + 8 * g;
            if (a.c.head_dim == W || c0 + 8 <= a.c.head_dim) {
                raw[t][j] = load_vec<T, 8>(qp + c0);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) raw[t][j].v[e] = c0 + e < a.c.head_dim ? qp[c0 + e] : from_float<T>(0.0f);
            }
        }
    }
    auto look_up = [&](uint32_t t0) {
        if (t0 / kPagedTile >= window_tile + kWaveSize) {
            window = next_window;
            window_tile += kWaveSize;
            next_window = load_window(window_tile + kWaveSize);
        }
        next_ok = 0;
#pragma unroll
        for (uint32_t i = 0; i < kChunkTiles; ++i) {
            const uint32_t p = lane_of(window, (t0 / kPagedTile + i) % kWaveSize);
            next_ok |= p != kNoPage ? 1u << i : 0u;
            pages[i] = p != kNoPage ? p : 0u;
        }
    };
    auto bring = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < kTilesOfWave; ++i) {
            // pages[rw + RW i], by constant indexes
            uint32_t page = 0;
#pragma unroll
            for (uint32_t k = 0; k < kChunkTiles; ++k) page = k == rw + RW * i ? pages[k] : page;
            load_tile<W>(a, page, t0 + (rw + RW * i) * kPagedTile, head, lane, words[i]);
        }
    };
    look_up((2 * from + half) * kChunk);
    uint32_t now = next_ok;  // of the chunk that is worked on
    bring((2 * from + half) * kChunk);
    v8h qf[RT][J];
    float mul[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(to_float(raw[t][j].v[e])));
        top = across_max(top);
        int e = 0;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);
        e = max(e, -100);
        float up = ldexpf(1.0f, -e);                        // |query| < 1
        mul[t] = exponents_of(a.scale, e, up);
        if (top == INFINITY || !isfinite(a.scale)) up = __builtin_nanf("");  // the row is NaN, whatever the keys are
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = to_float(raw[t][j].v[k]) * up;
            qf[t][j] = halves<1>(x).p[0];
        }
    }
    const uint32_t w_last = min(w_row0 + RT * 16 - 1, last);
    const bool idle = w_row0 > last;
    const uint32_t w_most = idle ? 0u : min(q.past + w_last / a.group + 1, a.slots);   // slots any row of the wave sees
    const uint32_t w_least = idle ? 0u : min(q.past + w_row0 / a.group + 1, a.slots);  // slots every one sees

    // m is of the products as they come, before mul; ref its exponent less kRowBits
    v4f acc[RT][C], sum[RT];
    float m[RT], ref[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        sum[t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f}, m[t] = kNothing, ref[t] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[t][c] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    }

    // chunk r of this half from the registers into LDS, chunk r + 1 on its way
    auto unpack = [&](uint32_t r) {
        v4u *keys = mine + (r % BUFFERS) * 2 * kOperands;
        look_up((2 * (r + 1) + half) * kChunk);
#pragma unroll
        for (uint32_t i = 0; i < kTilesOfWave; ++i)
            unpack_tile<W>(words[i], rw + RW * i, lane, keys, reinterpret_cast<v2u *>(keys + kOperands));
    };
    auto work = [&](uint32_t r, uint32_t seen) {
        const uint32_t t0 = (2 * r + half) * kChunk;
        if (t0 >= w_most) return;
        const v4u *keys = mine + (r % BUFFERS) * 2 * kOperands, *values = keys + kOperands;
        v4f sc[RT][kChunkTiles];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (uint32_t i = 0; i < kChunkTiles; ++i) {
                const v8h kc = __builtin_bit_cast(v8h, keys[(i * J + j) * kWaveSize + lane]);
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        kc, qf[t][j], j == 0 ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : sc[t][i], 0, 0, 0);
            }
        const bool masked = t0 + kChunk > w_least || seen != kAllTiles;
        v8h pf[RT][kChunkTiles / 2];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if (masked) {
#pragma unroll
                for (uint32_t i = 0; i < kChunkTiles; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((seen >> i) & 1u) || t0 + i * kPagedTile + 4 * g + e >= visible[t]) sc[t][i][e] = -INFINITY;
            }
            float mx = sc[t][0][0];
#pragma unroll
            for (uint32_t i = 0; i < kChunkTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[t][i][e]);
            if (__any((mx - m[t]) * mul[t] > kSlack)) {  // or nothing seen so far
                mx = across_max(fmaxf(mx, m[t]));
                const float moved = mx == kNothing ? 0.0f : fmaf(mx, mul[t], -static_cast<float>(kRowBits));
                const float alpha = __builtin_amdgcn_exp2f((m[t] - mx) * mul[t]);
#pragma unroll
                for (int c = 0; c < C; ++c) acc[t][c] *= alpha;
                sum[t] *= alpha;
                m[t] = mx;
                ref[t] = moved;
            }
            // a far reference is rounded by more than f16 has room for: then the
            // largest product is taken off first (for all rows 60.8 us for 58.2)
            float less = ref[t];
            if (__any(fabsf(less) > kFarRef)) {
#pragma unroll
                for (uint32_t i = 0; i < kChunkTiles; ++i) sc[t][i] -= m[t];
                less = -static_cast<float>(kRowBits);
            }
#pragma unroll
            for (uint32_t i = 0; i < kChunkTiles / 2; ++i) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    p[e] = __builtin_amdgcn_exp2f(fmaf(sc[t][2 * i + e / 4][e % 4], mul[t], -less));
                pf[t][i] = halves<1>(p).p[0];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kChunkTiles / 2; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const v8h vc = __builtin_bit_cast(v8h, values[(i * C + c) * kWaveSize + lane]);
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pf[t][i], acc[t][c], 0, 0, 0);
            }
        // the sum of the probabilities, as they were rounded: a product with ones
        const _Float16 one = static_cast<_Float16>(1.0f);
#pragma unroll
        for (uint32_t i = 0; i < kChunkTiles / 2; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t)
                sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16((v8h){one, one, one, one, one, one, one, one}, pf[t][i], sum[t], 0, 0, 0);
    };

    if constexpr (BUFFERS == 2) {
        unpack(from);
        uint32_t next = next_ok;
        bring((2 * (from + 1) + half) * kChunk);
        for (uint32_t r = from; r < rounds; ++r) {
            lds_barrier();  // chunk r is there, and the buffer of the one before is free
            if (half == 0) {
                unpack(r + 1);
                bring((2 * (r + 2) + half) * kChunk);
            }
            work(r, now);
            if (half == 1) {
                unpack(r + 1);
                bring((2 * (r + 2) + half) * kChunk);
            }
            now = next;
            next = next_ok;
        }
    } else {
        for (uint32_t r = from; r < rounds; ++r) {
            lds_barrier();
            unpack(r);
            lds_barrier();
            bring((2 * (r + 1) + half) * kChunk);
            work(r, now);
            now = next_ok;
        }
    }

    // the halves meet: the second one's sums through LDS, a wave's rows in its
    // own part of it
    lds_barrier();
    constexpr uint32_t kSumLanes = kWaveSize + 1;  // float4s of a register quadruple, kept off one bank
    constexpr uint32_t kSums = C * kSumLanes + kWaveSize;
    v4f *sums = reinterpret_cast<v4f *>(chunk) + rw * RT * kSums;
    if (half == 1) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int c = 0; c < C; ++c) sums[t * kSums + c * kSumLanes + lane] = acc[t][c];
            sums[t * kSums + C * kSumLanes + lane] = (v4f){m[t], sum[t][0], 0.0f, 0.0f};
        }
    }
    lds_barrier();
    if (half == 1) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const v4f other = sums[t * kSums + C * kSumLanes + lane];
        const float top = fmaxf(m[t], other[0]);
        const float f0 = __builtin_amdgcn_exp2f((m[t] - top) * mul[t]), f1 = __builtin_amdgcn_exp2f((other[0] - top) * mul[t]);
        const float l = sum[t][0] * f0 + other[1] * f1, inv = l == 0.0f ? 0.0f : 1.0f / l;
        const uint32_t r = w_row0 + t * 16 + n;
        if (r > last) continue;
        T *dst = static_cast<T *>(a.output) + static_cast<size_t>(q.row + r / a.group) * a.output_stride +
                 static_cast<size_t>(head * a.group + r % a.group) * a.c.head_dim;
        const size_t at_part = (static_cast<size_t>(blockIdx.x) * a.parts + blockIdx.y) * kBlockRows + r - row0;
        if (parts > 1 && g == 0) a.part_ml[at_part] = make_float4(top, l, mul[t], 0.0f);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const v4f o = acc[t][c] * f0 + sums[t * kSums + c * kSumLanes + lane] * f1;
            const uint32_t ch = 16 * c + 4 * g;
            if (parts > 1) {
                *reinterpret_cast<v4f *>(a.part_o + at_part * W + ch) = o;
                continue;
            }
            Vec<T, 4> y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.v[e] = from_float<T>(o[e] * inv);
            if (a.c.head_dim == W || ch + 4 <= a.c.head_dim) {
                store_vec<T, 4>(dst + ch, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ch + e < a.c.head_dim) dst[ch + e] = y.v[e];
            }
        }
    }
}

// The parts of the blocks whose contexts were split.  grid (KV heads of blocks at
// most, row groups): W / 4 threads a row.
template <typename T, int W, uint32_t ROWS>
__global__ __launch_bounds__(kThreads) void paged_block_merge_kernel(AttnArgs a) {
    constexpr uint32_t kLanes = W / 4, kGroups = kThreads / kLanes;
    uint32_t s, at;
    PagedSequence q;
    const uint32_t head = blockIdx.x % a.c.kv_heads, index = blockIdx.x / a.c.kv_heads;
    if (!find_in(a.b, index, [&](const PagedSequence &x) { return (x.rows * a.group + ROWS - 1) / ROWS; }, s, at, q)) return;
    const uint32_t all = q.rows * a.group, block = (all + ROWS - 1) / ROWS - 1 - at;
    const uint32_t row0 = block * ROWS, last = min(row0 + ROWS, all) - 1;
    const uint32_t most = min(q.past + last / a.group + 1, a.slots);
    const uint32_t parts = block_parts(a, ((most + kChunk - 1) / kChunk + 1) / 2);
    if (parts == 1) return;
    const uint32_t lane = threadIdx.x % kLanes, r = blockIdx.y * kGroups + threadIdx.x / kLanes, row = row0 + r;
    if (row > last) return;
    const size_t first = static_cast<size_t>(blockIdx.x) * a.parts * ROWS + r;
    float2 ml[kBlockPartsMost];
    v4f x[kBlockPartsMost];
    float top = kNothing, mul = 1.0f;
#pragma unroll
    for (uint32_t i = 0; i < kBlockPartsMost; ++i)
        if (i < parts) {
            const float4 part = a.part_ml[first + i * ROWS];
            ml[i] = make_float2(part.x, part.y);
            mul = part.z;
            x[i] = *reinterpret_cast<const v4f *>(a.part_o + (first + i * ROWS) * W + 4 * lane);
            top = fmaxf(top, ml[i].x);
        }
    v4f o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kBlockPartsMost; ++i)
        if (i < parts) {
            const float f = __builtin_amdgcn_exp2f((ml[i].x - top) * mul);
            o += x[i] * f;
            l += ml[i].y * f;
        }
    T *dst = static_cast<T *>(a.output) + static_cast<size_t>(q.row + row / a.group) * a.output_stride +
             static_cast<size_t>(head * a.group + row % a.group) * a.c.head_dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (4 * lane + e < a.c.head_dim) dst[4 * lane + e] = from_float<T>(l == 0.0f ? 0.0f : o[e] / l);
}

// Rows of the block kernel's blocks.
constexpr uint32_t block_rows_of(uint32_t width) { return kBlockWaves * (width == 256 ? 1u : 2u) * 16; }

// Partial rows that a workspace holds: two blocks of each worker, or a part of a
// block of each of the block kernel's workgroups.
size_t partial_rows(uint32_t width) {
    return std::max<size_t>(static_cast<size_t>(kWorkers) * 2 * kRows, static_cast<size_t>(kBlockGroups) * block_rows_of(width));
}
size_t partial_bytes(uint32_t width) { return partial_rows(width) * (width * sizeof(float) + sizeof(float4)); }

// Whether a batch's sequences bring rows as prompts do (of 8 KV heads: 16
// sequences of 3000 tokens with 64 rows each 70 us in the block kernel and 53 in
// blocks of 16, with 80 rows 70 and 66, with 124 72 and 88; 64 of 1000 with 80
// rows 64 and 78), and is for the block kernel: more than a few short ones (a
// prompt of 128 tokens 13 and 9, of 256 16 and 12; 8 of 64 behind 192 16 and 20).
bool many_rows(const AttnArgs &a) { return static_cast<uint64_t>(a.b.tokens) * a.group >= 80ull * a.b.sequences; }
bool block_rows(const AttnArgs &a) {
    return many_rows(a) && (static_cast<uint64_t>(a.b.tokens) * a.group * a.c.kv_heads > 8192 || a.slots > kWholeSlots);
}

template <typename T, int W, int RW, int RT, int BUFFERS>
hipError_t launch_block(AttnArgs a, hipStream_t stream) {
    constexpr uint32_t kBlockRows = RW * RT * 16;
    static_assert(kBlockRows == block_rows_of(W), "the workspace is sized by it");
    constexpr size_t chunks = 2 * BUFFERS * 2 * kChunk * W * 2;
    constexpr size_t sums = static_cast<size_t>(RW) * RT * (W / 16 * (kWaveSize + 1) + kWaveSize) * 16;
    constexpr size_t lds = chunks > sums ? chunks : sums;
    static_assert(lds <= 160 * 1024, "a workgroup's LDS");
    const void *kernel = reinterpret_cast<const void *>(&paged_block_attention_kernel<T, W, RW, RT, BUFFERS>);
    hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return e;
    // at most one block of each sequence is not full; of one sequence no workgroup is
    // without work, as one is enough to send two others to the same CU
    const uint64_t rows = static_cast<uint64_t>(a.b.tokens) * a.group, used = std::min(a.b.sequences, a.b.tokens);
    const uint32_t blocks = static_cast<uint32_t>((rows + used * (kBlockRows - 1)) / kBlockRows);
    a.parts = std::max(1u, std::min(kBlockPartsMost, kBlockGroups / (blocks * a.c.kv_heads)));
    hipLaunchKernelGGL((paged_block_attention_kernel<T, W, RW, RT, BUFFERS>), dim3(blocks * a.c.kv_heads, a.parts),
                       dim3(2 * RW * kWaveSize), lds, stream, a);
    if ((e = hipGetLastError()) != hipSuccess || a.parts == 1 || a.slots <= 2 * kPartRounds * kChunk) return e;
    hipLaunchKernelGGL((paged_block_merge_kernel<T, W, kBlockRows>), dim3(blocks * a.c.kv_heads, kBlockRows / (kThreads / (W / 4))),
                       dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

template <typename T, int W, bool PROMPT>
hipError_t launch_blocks(AttnArgs a, uint32_t blocks, hipStream_t stream) {
    const uint32_t groups = blocks * a.c.kv_heads;
    constexpr bool kEight = !PROMPT && W != 256;  // of 256 channels they would not have the registers
    const bool eight = kEight && groups < kMany;
    const bool longer = groups >= kMany || (eight && (sizeof(T) == 2 || groups >= kSome));
    a.whole = a.slots <= (longer ? kWholeSlotsMany : kWholeSlots);
    a.workers = a.whole ? groups : W == 256 ? kWorkers / 3 : kWorkers;  // of 256 channels: one on each CU
    if constexpr (kEight) {
        // few blocks that are not cut: eight waves each (one sequence of 334 tokens,
        // 2 KV heads, bf16 7.9 us, with four 8.4; fp32 9.4 and 9.7)
        if (a.whole && eight) {
            hipLaunchKernelGGL((paged_attention_kernel<T, W, false, 8>), dim3(a.workers), dim3(8 * kWaveSize), 0, stream, a);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((paged_attention_kernel<T, W, PROMPT, kWaves>), dim3(a.workers), dim3(kThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.whole) return e;
    // rows of a sequence, about
    const uint32_t each = static_cast<uint32_t>((static_cast<uint64_t>(a.b.tokens) * a.group + a.b.sequences - 1) / a.b.sequences);
    const uint32_t parts = std::min({kRows, each, std::max(3u, kMergeGroups / (blocks * a.c.kv_heads))});
    hipLaunchKernelGGL((paged_merge_kernel<T, W, PROMPT>), dim3(blocks, a.c.kv_heads, parts), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

template <typename T, int W>
hipError_t launch_width(AttnArgs a, uint32_t blocks, hipStream_t stream) {
    // f16 rows are left to blocks of 16, whose values are exact: keys and values
    // rounded to f16 would cost more than the output's own rounding (error 3.5 to
    // 4.5e-4, there 2.9e-4, of which the output's 2.1e-4; four prompts of 512 tokens
    // behind 2048 276 us for 134)
    if constexpr (std::is_same_v<T, bf16>) {
        if (block_rows(a)) return launch_block<T, W, kBlockWaves, W == 256 ? 1 : 2, W == 256 ? 1 : 2>(a, stream);
    }
    return many_rows(a) ? launch_blocks<T, W, true>(a, blocks, stream) : launch_blocks<T, W, false>(a, blocks, stream);
}
template <typename T>
hipError_t launch_paged_attention(const AttnArgs &a, uint32_t blocks, hipStream_t stream) {
    return a.c.width == 64    ? launch_width<T, 64>(a, blocks, stream)
           : a.c.width == 128 ? launch_width<T, 128>(a, blocks, stream)
                              : launch_width<T, 256>(a, blocks, stream);
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
    const uint64_t channels = static_cast<uint64_t>(r->query_heads) * a.c.head_dim, size = dtype_bytes(r->dtype);
    const Rows in = row_block(r->query, a.b.tokens, channels, a.query_stride, size),
               out = row_block(r->output, a.b.tokens, channels, a.output_stride, size),
               work = list_of_bytes(r->workspace, partial_bytes(a.c.width));
    if (overlaps_any(out, {in, work}) || overlap(work, in) || overlaps_batch(out, a.b) || overlaps_batch(work, a.b)) {
        set_error("paged attention: the output or the workspace overlaps an input or each other");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    // row blocks and pieces of the batch at most: counted in 32 bits
    const uint64_t rows = static_cast<uint64_t>(a.b.tokens) * a.group;
    const uint64_t blocks = std::min<uint64_t>(rows, rows / kRows + std::min(a.b.sequences, a.b.tokens));
    const uint64_t slots = std::min<uint64_t>(static_cast<uint64_t>(a.b.table_stride) << a.c.page_shift, 0x7fffff80u);
    if (rows > 0x7fffffffu || blocks * a.c.kv_heads > 0x7fffffffu ||
        blocks * a.c.kv_heads > 0x7fffffffull / (kStart + (slots + kPiece - 1) / kPiece)) {
        set_error("paged attention: %u tokens of %u heads over %llu slots are too many for one call", a.b.tokens,
                  r->query_heads, static_cast<unsigned long long>(slots));
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    a.slots = static_cast<uint32_t>(slots);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("paged attention device", device.error());
    a.query = r->query;
    a.output = r->output;
    a.scale = r->scale;
    a.part_ml = static_cast<float4 *>(r->workspace);
    a.part_o = reinterpret_cast<float *>(a.part_ml + partial_rows(a.c.width));
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_paged_attention<float>(a, static_cast<uint32_t>(blocks), s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_paged_attention<f16>(a, static_cast<uint32_t>(blocks), s)
                                                         : launch_paged_attention<bf16>(a, static_cast<uint32_t>(blocks), s);
    if (e != hipSuccess) return hip_fail("paged attention launch", e);
    ctx->telemetry.kv_cache_kernel_count++;
    return QWN_CUDA_STATUS_OK;
}

}  // extern "C"
