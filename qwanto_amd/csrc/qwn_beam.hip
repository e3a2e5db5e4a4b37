// Beams: the best continuations of each sequence's beams over the vocabulary
// (qwn_hip_ext_beam_select_device), and what the beams keep following them
// (qwn_hip_ext_paged_kv_beam_advance_device).
#include "qwn_context.h"
#include "qwn_device.h"
#include "qwn_hip_ext.h"
#include "qwn_overlap.h"
#include "qwn_paged.h"
#include "qwn_paged_batch.h"
#include "qwn_types.h"

#include <algorithm>

namespace {

using namespace qwn;

// ---- selection --------------------------------------------------------------

constexpr uint32_t kThreads = 256;
constexpr uint32_t kBeamsMost = QWN_HIP_BEAM_MAX_BEAMS, kCountMost = QWN_HIP_BEAM_MAX_COUNT;
constexpr uint32_t kNone = 0xffffffffu;
constexpr int kLoads = 4;               // vectors of 16 bytes that a thread takes of a row
template <typename T>
constexpr uint32_t kSlice = kThreads * kLoads * (16 / sizeof(T));  // tokens of the vocabulary a workgroup takes

// Candidates in order: a larger value, then the larger place, is the larger key;
// the value 0 is none.  Of a row, values are fp32 logits and places its tokens from the last; of a
// sequence, 64-bit sums, and places the beams from the last, then the logits (sums of one beam may
// be one number where they are not), then the tokens from the last.
__device__ __forceinline__ uint32_t ordered(float v) {  // 0 for -inf and NaN, which are no candidates
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 is 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t ord) {
    return __builtin_bit_cast(float, (ord & 0x80000000u) ? ord & 0x7fffffffu : ~ord);
}
__device__ __forceinline__ uint64_t ordered(double v) {
    if (!(v > -INFINITY)) return 0;
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return (b >> 63) ? ~b : (b | 1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t ord) {
    return __builtin_bit_cast(double, (ord >> 63) ? ord & ~(1ull << 63) : ~ord);
}
struct Key {
    uint64_t value, place;  // ordered bits
};
constexpr uint32_t kTokenBits = 24, kTokens = 1u << kTokenBits;  // of a place in a sequence: above them 32 of the logit, then the beam
__device__ __forceinline__ uint64_t place_of(uint32_t beam, uint32_t logit, uint32_t token) {
    return static_cast<uint64_t>(kBeamsMost - 1 - beam) << (kTokenBits + 32) | static_cast<uint64_t>(logit) << kTokenBits | (kTokens - 1 - token);
}
__device__ __forceinline__ uint32_t beam_of(uint64_t place) { return kBeamsMost - 1 - static_cast<uint32_t>(place >> (kTokenBits + 32)); }
__device__ __forceinline__ uint32_t token_of(uint64_t place) { return kTokens - 1 - (static_cast<uint32_t>(place) & (kTokens - 1)); }
__device__ __forceinline__ bool larger(const Key &a, const Key &b) {
    return a.value > b.value || (a.value == b.value && a.place > b.place);
}

// The count-th largest of 64 numbers, each the largest of 4 of the workgroup's; 0
// where fewer are not 0.  Every wave searches for itself.
__device__ __forceinline__ uint32_t find_bound(const uint32_t *numbers, uint32_t count) {
    const uint4 x = reinterpret_cast<const uint4 *>(numbers)[threadIdx.x % kWaveSize];
    const uint32_t most = max(max(x.x, x.y), max(x.z, x.w));
    uint32_t bound = 0;
#pragma unroll 4
    for (uint32_t bit = 1u << 31; bit; bit >>= 1)
        if (static_cast<uint32_t>(__popcll(__ballot(most >= (bound | bit)))) >= count) bound |= bit;
    return bound;
}

// The `count` largest of the workgroup's candidates, N a thread, largest first, in
// list[0 .. count); the value 0 where there are fewer.  key(i): the thread's i-th;
// reaches(i, bound): whether its value's upper bits, of a number that does not
// decrease with the value, are bound or more; top: the largest of them, 0 for none.
// The result does not fall below the count-th largest of 64 of these, and few candidates
// are as large; of those, each one's place is the number that are larger.  Where
// they are more than kFound (many are alike), the largest are taken out one by one.
// (The bound from all 256 threads' numbers, each one's place counted: 4 beams 35 us for 11.)
constexpr uint32_t kFound = 512;
constexpr uint32_t kLeast = 0x00100000u;  // below what any number's upper bits are ordered as, above none's
struct Selection {
    alignas(16) uint32_t tops[kThreads];  // read four at a time
    Key found[kFound];
    Key list[kCountMost];
    Key best[kThreads / kWaveSize];
    uint32_t held;
};
template <int N, typename R, typename K>
__device__ __forceinline__ void select_keys(Selection &s, uint32_t count, uint32_t top, R reaches, K key) {
    const uint32_t tid = threadIdx.x;
    s.tops[tid] = top;
    if (tid == 0) s.held = 0;
    lds_barrier();
    for (uint32_t i = tid; i < count; i += kThreads) s.list[i] = Key{0, 0};
    const uint32_t bound = max(kLeast, find_bound(s.tops, count));
    if (top >= bound) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (reaches(i, bound)) {
                const uint32_t to = atomicAdd(&s.held, 1u);
                if (to < kFound) s.found[to] = key(i);
            }
    }
    lds_barrier();
    const uint32_t n = s.held;
    if (n <= kFound) {
        for (uint32_t e = tid; e < n; e += kThreads) {
            const Key mine = s.found[e];
            uint32_t place = 0;
            for (uint32_t i = 0; i < n; ++i) place += larger(s.found[i], mine) ? 1u : 0u;
            if (place < count) s.list[place] = mine;
        }
        lds_barrier();
        return;
    }
    Key last{~0ull, ~0ull};
#pragma unroll 1
    for (uint32_t k = 0; k < count; ++k) {
        Key best{0, 0};
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            if (!reaches(i, bound)) continue;
            const Key x = key(i);
            if (larger(last, x) && larger(x, best)) best = x;
        }
#pragma unroll
        for (int off = kWaveSize / 2; off > 0; off >>= 1) {
            const Key o{__shfl_xor(best.value, off), __shfl_xor(best.place, off)};
            if (larger(o, best)) best = o;
        }
        if (tid % kWaveSize == 0) s.best[tid / kWaveSize] = best;
        lds_barrier();
        best = s.best[0];
#pragma unroll
        for (uint32_t w = 1; w < kThreads / kWaveSize; ++w)
            if (larger(s.best[w], best)) best = s.best[w];
        if (tid == 0) s.list[k] = best;
        last = best;
        lds_barrier();  // `best` is read
    }
}

struct SelectArgs {
    const void *logits;
    const float *scores;
    float *values, *next_scores;
    int32_t *parents, *tokens, *next_parents, *next_tokens;
    float2 *sums;        // [rows][parts]: the largest logit of a part, the sum of exp(logit - it)
    uint64_t *keys;      // [rows][parts][count]
    uint32_t beams, vocab, count, in_stride, parts, end_count;
    int32_t end_tokens[4];
};

// grid (parts of the vocabulary, rows): a part's largest logits and its share of
// the sum, in one pass over them.  Bound by HBM where rows are many, 64 rows of 151936 bf16
// logits 8.1 us, 2.4 TB/s, a part's selection at its end included; few by load and selection,
// 4 rows 4.4.
template <typename T>
__global__ __launch_bounds__(kThreads) void beam_rows_kernel(SelectArgs a) {
    constexpr int VEC = 16 / sizeof(T), N = kLoads * VEC;
    __shared__ Selection select;
    __shared__ float2 red[kThreads / kWaveSize];
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * kSlice<T>, tid = threadIdx.x;
    const T *in = static_cast<const T *>(a.logits) + static_cast<size_t>(r) * a.in_stride;
    float x[N];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
        const uint32_t v = v0 + (tid + kThreads * k) * VEC;
        if (v + VEC <= a.vocab) {
            const Vec<T, VEC> t = load_vec<T, VEC>(in + v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[k * VEC + i] = to_float(t.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[k * VEC + i] = v + i < a.vocab ? to_float(in[v + i]) : -INFINITY;
        }
    }
    constexpr float kLowest = -3.402823466e38f;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = fmaxf(x[i], -INFINITY);  // NaN counts as -inf
        top = fmaxf(top, x[i]);
    }
    const float m = fmaxf(wave_max_all(top), kLowest);
    // logits are few steps of fp32 below m where they count: the difference and its
    // product are rounded by 2^-24 of at most 40
    constexpr float kLog2e = 1.44269504088896340736f;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f((x[i] - m) * kLog2e);
    s = wave_sum_all(s);
    if (tid % kWaveSize == 0) red[tid / kWaveSize] = make_float2(m, s);
    select_keys<N>(select, a.count, ordered(top), [&](int i, uint32_t bound) { return x[i] >= fmaxf(unordered(bound), kLowest); },
                   [&](int i) {
                       const uint32_t v = v0 + (tid + kThreads * (i / VEC)) * VEC + i % VEC;
                       return Key{ordered(x[i]), ~static_cast<uint64_t>(v)};
                   });
    const size_t part = static_cast<size_t>(r) * a.parts + blockIdx.x;
    for (uint32_t i = tid; i < a.count; i += kThreads)
        a.keys[part * a.count + i] = select.list[i].value << 32 | static_cast<uint32_t>(~select.list[i].place);
    if (tid == 0) {
        float most = red[0].x, sum = 0.0f;
        for (uint32_t w = 1; w < kThreads / kWaveSize; ++w) most = fmaxf(most, red[w].x);
        for (uint32_t w = 0; w < kThreads / kWaveSize; ++w) sum += red[w].y * __builtin_amdgcn_exp2f((red[w].x - most) * kLog2e);
        a.sums[part] = make_float2(most > kLowest || sum > 0.0f ? most : -INFINITY, sum);  // else nothing but -inf and NaN
    }
}

// grid (sequences): the rows' sums, and the largest of their parts' candidates.  One
// workgroup's latency: parts, selection, order, 5.7 us for 1 as for 16 sequences.
__global__ __launch_bounds__(kThreads) void beam_sequences_kernel(SelectArgs a) {
    constexpr int N = 8;                 // keys of a thread in a round, one more of what is left of the round before
    __shared__ Selection select;
    __shared__ double base[kBeamsMost], most[kBeamsMost];  // of a beam: its score less the logarithm of its sum, -inf: no
                                                           // candidates; its largest logit
    const uint32_t tid = threadIdx.x, lane = tid % kWaveSize, wave = tid / kWaveSize, row0 = blockIdx.x * a.beams;
    const uint32_t of_row = a.parts * a.count, all = a.beams * of_row;
    const uint64_t *keys = a.keys + static_cast<size_t>(row0) * of_row;
    uint64_t next[N];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t i = i0 + tid + kThreads * e;
            next[e] = i < all ? keys[i] : 0u;
        }
    };
    load(0);
    for (uint32_t b = wave; b < a.beams; b += kThreads / kWaveSize) {
        const float2 *sums = a.sums + static_cast<size_t>(row0 + b) * a.parts;
        const float score = a.scores[row0 + b];
        const float2 mine = lane < a.parts ? sums[lane] : make_float2(-INFINITY, 0.0f);
        float m = mine.x;
        for (uint32_t i = lane + kWaveSize; i < a.parts; i += kWaveSize) m = fmaxf(m, sums[i].x);
        m = wave_max_all(m);
        auto share = [&](float2 x) {
            return x.x > -INFINITY ? static_cast<double>(x.y) * exp(static_cast<double>(x.x) - static_cast<double>(m)) : 0.0;
        };
        double s = share(mine);
        for (uint32_t i = lane + kWaveSize; i < a.parts; i += kWaveSize) s += share(sums[i]);
        s = wave_sum_f64(s);
        if (lane == 0) {
            base[b] = isfinite(m) && isfinite(score) ? static_cast<double>(score) - log(s) : -INFINITY;
            most[b] = m;
        }
    }
    lds_barrier();
    for (uint32_t i0 = 0; i0 < all; i0 += N * kThreads) {
        double v[N + 1];
        uint64_t place[N + 1], top = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t b = min((i0 + tid + kThreads * e) / of_row, a.beams - 1);
            v[e] = next[e] ? base[b] + (static_cast<double>(unordered(static_cast<uint32_t>(next[e] >> 32))) - most[b]) : -INFINITY;
            place[e] = place_of(b, static_cast<uint32_t>(next[e] >> 32), static_cast<uint32_t>(next[e]));
        }
        v[N] = -INFINITY;
        if (i0 > 0 && tid < a.count && select.list[tid].value) {
            v[N] = unordered(select.list[tid].value);
            place[N] = select.list[tid].place;
        }
        if (i0 + N * kThreads < all) load(i0 + N * kThreads);
#pragma unroll
        for (int e = 0; e <= N; ++e) top = max(top, ordered(v[e]));
        if (i0 > 0) lds_barrier();  // the list is read
        select_keys<N + 1>(select, a.count, static_cast<uint32_t>(top >> 32), [&](int i, uint32_t bound) { return static_cast<uint32_t>(ordered(v[i]) >> 32) >= bound; },
                           [&](int i) { return Key{ordered(v[i]), place[i]}; });
    }
    // the list is one wave's: place, and place among those that go on
    if (wave > 0) return;
    const size_t out = static_cast<size_t>(blockIdx.x) * a.count, out_next = static_cast<size_t>(blockIdx.x) * a.beams;
    float value = -INFINITY;
    int32_t parent = -1, token = -1;
    const bool real = lane < a.count && select.list[lane].value;
    if (real) {
        const uint64_t at = select.list[lane].place;
        value = static_cast<float>(unordered(select.list[lane].value));
        parent = static_cast<int32_t>(row0 + beam_of(at));
        token = static_cast<int32_t>(token_of(at));
    }
    if (lane < a.count) {
        a.values[out + lane] = value;
        a.parents[out + lane] = parent;
        a.tokens[out + lane] = token;
    }
    if (!a.next_scores) return;
    bool goes = real;
    for (uint32_t i = 0; i < a.end_count; ++i) goes = goes && token != a.end_tokens[i];
    const uint64_t on = __ballot(goes);
    const uint32_t to = __popcll(on & ((1ull << lane) - 1)), n = __popcll(on);
    if (goes && to < a.beams) {
        a.next_scores[out_next + to] = value;
        a.next_parents[out_next + to] = parent;
        a.next_tokens[out_next + to] = token;
    }
    if (lane >= n && lane < a.beams) {
        a.next_scores[out_next + lane] = -INFINITY;
        a.next_parents[out_next + lane] = -1;
        a.next_tokens[out_next + lane] = -1;
    }
}

uint32_t parts_of(uint32_t vocab, uint32_t slice) { return (vocab + slice - 1) / slice; }
// sums, then keys: of the type with the most parts
uint64_t sums_bytes(uint64_t rows, uint64_t parts) { return (rows * parts * sizeof(float2) + 15) / 16 * 16; }

template <typename T>
hipError_t launch_select(SelectArgs a, uint32_t sequences, void *workspace, hipStream_t stream) {
    const uint32_t rows = sequences * a.beams;
    a.parts = parts_of(a.vocab, kSlice<T>);
    a.sums = static_cast<float2 *>(workspace);
    a.keys = reinterpret_cast<uint64_t *>(static_cast<uint8_t *>(workspace) + sums_bytes(rows, a.parts));
    hipLaunchKernelGGL(beam_rows_kernel<T>, dim3(a.parts, rows), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(beam_sequences_kernel, dim3(sequences), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

bool select_sizes(uint32_t sequences, uint32_t beams, uint32_t vocab, uint32_t count) {
    return sequences > 0 && beams > 0 && beams <= kBeamsMost && static_cast<uint64_t>(sequences) * beams <= 65535 && vocab > 0 &&
           vocab <= kTokens && count > 0 && count <= kCountMost;
}

// ---- what the beams keep ------------------------------------------------------

constexpr uint32_t kCachesMost = QWN_HIP_BEAM_MAX_CACHES;

struct AdvanceArgs {
    const int32_t *parents, *past, *table, *spare, *tokens, *history;
    int32_t *past_out, *table_out, *spare_out, *history_out;
    uint32_t beams, page_shift, table_stride, added, history_length;
};
struct CopyArgs {
    AdvanceArgs a;
    PagedKv c;
    uint8_t *pools[kCachesMost];
};

// Where row r of its sequence goes on from, and its length then; false: from
// none, nothing of it changes.
struct Goes {
    uint32_t parent;   // row
    uint32_t length;
    bool token;        // not from itself for want of a parent
};
__device__ __forceinline__ bool goes_on(const AdvanceArgs &a, uint32_t row0, uint32_t r, Goes &g) {
    const int32_t p = a.parents[r];
    g.token = p >= static_cast<int32_t>(row0) && p < static_cast<int32_t>(row0 + a.beams) && a.past[p] >= 0;
    g.parent = g.token ? static_cast<uint32_t>(p) : r;
    const int32_t past = a.past[g.parent];
    if (past < 0) return false;
    g.length = static_cast<uint32_t>(min(static_cast<int64_t>(past) + a.added, static_cast<int64_t>(0x7fffffff)));
    return true;
}
__device__ __forceinline__ int32_t page_of(const AdvanceArgs &a, uint32_t row, uint32_t at) {
    return at < a.table_stride ? a.table[static_cast<size_t>(row) * a.table_stride + at] : -1;
}

// What the rows of a sequence are to each other: a lane a row (lanes past them: none).
struct Kin {
    bool goes;        // the lane's row is one, and goes on
    bool later;       // not its parent's first child
    Goes g;
    uint64_t laters, childless;
};
__device__ __forceinline__ Kin kin_of(const AdvanceArgs &a, uint32_t row0, uint32_t lane) {
    Kin k{};
    const bool row = lane < a.beams;
    k.goes = row && goes_on(a, row0, row0 + lane, k.g);
    const uint32_t mine = k.goes ? k.g.parent - row0 : kNone;
    uint64_t parents = 0;
    for (uint32_t b = 0; b < a.beams; ++b) {
        const uint32_t p = lane_of(mine, static_cast<int>(b));
        if (b < lane && p == mine) k.later = k.goes;
        if (p != kNone) parents |= 1ull << p;
    }
    k.laters = __ballot(k.later);
    k.childless = __ballot(row && !((parents >> lane) & 1ull));
    return k;
}

// The n-th of some bits (from 0); none past the last.
__device__ __forceinline__ uint32_t nth_of(uint64_t bits, uint32_t n) {
    for (; n > 0 && bits; --n) bits &= bits - 1;
    return bits ? __ffsll(static_cast<unsigned long long>(bits)) - 1 : kNone;
}
// The spare that the lane's row has afterwards.  Pages in use are left by rows that nothing
// goes on from, where they have a length and a page that has not just become full.  A
// row that copies takes the one of the row that has its place among the childless, if it
// left one, else the first that nobody took so, in order; those that are left then go to rows that
// begin a page (of other lengths: of one length there are none left).  So a page in use is
// lost only where no row has room for it.
__device__ __forceinline__ int32_t spare_of(const AdvanceArgs &a, const Kin &k, uint32_t row0, uint32_t lane) {
    const bool row = lane < a.beams;
    const uint32_t slots = (1u << a.page_shift) - 1;
    const int32_t past = row ? a.past[row0 + lane] : -1;
    const int64_t length = static_cast<int64_t>(past) + a.added;
    const int32_t page = past >= 0 && (length & slots) && length >> a.page_shift < a.table_stride
                             ? page_of(a, row0 + lane, static_cast<uint32_t>(length >> a.page_shift)) : -1;
    const bool copies = k.later && (k.g.length & slots),
               begins = k.goes && !(k.g.length & slots) && k.g.length >> a.page_shift < a.table_stride;  // else the table has no place for a page
    const uint64_t below = (1ull << lane) - 1, all_copy = __ballot(copies), left = __ballot(((k.childless >> lane) & 1) && page >= 0);
    // by place: the lane's row as one that copies, and as one that leaves its page
    const uint32_t giver = nth_of(k.childless, __popcll(k.laters & below)), taker = nth_of(k.laters, __popcll(k.childless & below));
    const bool served = copies && giver != kNone && (left >> giver & 1), gives = taker != kNone && (all_copy >> taker & 1);
    // in order: who has none yet, then who begins a page; of what is left
    const uint64_t free = __ballot((left >> lane & 1) && !gives), want = __ballot(copies && !served), later_want = __ballot(begins);
    const uint32_t place = begins ? __popcll(want) + __popcll(later_want & below) : __popcll(want & below);
    const uint32_t from = served ? giver : nth_of(free, place);
    const int32_t taken = __shfl(page, static_cast<int>(from == kNone ? 0u : from));
    const int32_t spare = row ? a.spare[row0 + lane] : -1;
    return copies || begins ? (from == kNone ? -1 : taken) : spare;
}

// The slots of the parent's page in use to the row's spare, in one cache; the first
// of a row's workgroups writes its length and the spare it gets.  Bytes bound it.
__device__ __forceinline__ void copy_pages(const CopyArgs &args, uint32_t r, uint32_t cache) {
    const AdvanceArgs &a = args.a;
    const uint32_t row0 = r / a.beams * a.beams, lane = threadIdx.x % kWaveSize;
    const Kin k = kin_of(a, row0, lane);
    const int b = static_cast<int>(r - row0);
    const bool goes = lane_of(k.goes, b), later = lane_of(k.later, b);
    const uint32_t parent = lane_of(k.g.parent, b), length = lane_of(k.g.length, b);
    const uint32_t full = length >> a.page_shift, used = length & ((1u << a.page_shift) - 1);
    const int32_t spare = a.spare[r];
    if (cache == 0 && threadIdx.x < kWaveSize) {
        const int32_t next = spare_of(a, k, row0, lane);
        if (lane == static_cast<uint32_t>(b)) {
            a.past_out[r] = goes ? static_cast<int32_t>(length) : a.past[r];
            a.spare_out[r] = next;
        }
    }
    if (!goes || !later || used == 0 || !args.pools[cache]) return;
    const PagedKv &c = args.c;
    const int32_t from = page_of(a, parent, full);
    if (from < 0 || static_cast<uint32_t>(from) >= c.pages || spare < 0 || static_cast<uint32_t>(spare) >= c.pages || from == spare) return;
    const uint32_t tiles = (used + kPagedTile - 1) / kPagedTile, words = tiles * (paged_block_bytes(c.width) / 16);
    for (uint32_t i = threadIdx.x; i < c.kv_heads * words; i += kThreads) {
        const uint32_t head = i / words, w = i % words;
        uint8_t *pool = args.pools[cache];
        reinterpret_cast<uint4 *>(pool + paged_block_at(c, static_cast<uint32_t>(spare), 0, head))[w] =
            reinterpret_cast<const uint4 *>(pool + paged_block_at(c, static_cast<uint32_t>(from), 0, head))[w];
    }
}

// A thread moves a column of the table or of the histories in all of the
// sequence's rows, reading all of them first, so that they may be in place.
__device__ __forceinline__ void move_columns(const AdvanceArgs &a, uint32_t sequence, uint32_t group, uint32_t table_groups) {
    const uint32_t row0 = sequence * a.beams, lane = threadIdx.x % kWaveSize;
    const Kin k = kin_of(a, row0, lane);
    const bool table = group < table_groups;
    const uint32_t column = (table ? group : group - table_groups) * kThreads + threadIdx.x;
    const uint32_t stride = table ? a.table_stride : a.history_length;
    const bool in = column < stride;
    const int32_t *from = table ? a.table : a.history;
    int32_t *to = table ? a.table_out : a.history_out;
    int32_t v[kBeamsMost];
#pragma unroll
    for (uint32_t b = 0; b < kBeamsMost; ++b) {
        v[b] = 0;
        if (b >= a.beams) continue;
        const bool goes = lane_of(k.goes, b), later = lane_of(k.later, b), token = lane_of(k.g.token, b);
        const uint32_t parent = goes ? lane_of(k.g.parent, b) : row0 + b, length = lane_of(k.g.length, b);
        if (in) v[b] = from[static_cast<size_t>(parent) * stride + column];
        if (!goes) continue;
        if (table) {
            const uint32_t full = length >> a.page_shift, used = length & ((1u << a.page_shift) - 1);
            if (column == full && (used == 0 || later)) v[b] = a.spare[row0 + b];
            if (column > full) v[b] = -1;
        } else if (token && a.tokens && column == length) {
            v[b] = a.tokens[row0 + b];
        }
    }
    if (!in) return;
#pragma unroll
    for (uint32_t b = 0; b < kBeamsMost; ++b)
        if (b < a.beams) to[static_cast<size_t>(row0 + b) * stride + column] = v[b];
}

// grid: workgroups from `first` on of those that copy (a row and a cache each, at
// least one cache), then of those that move (a sequence, and 256 columns).  4 rows 4.2 us, a
// launch and three loads one after the other; 64 rows of 28 caches 10.9, copies of up to 18 KB each.
__global__ __launch_bounds__(kThreads) void beam_advance_kernel(CopyArgs args, uint32_t first, uint32_t copies, uint32_t rows,
                                                                uint32_t groups, uint32_t table_groups) {
    const uint32_t i = first + blockIdx.x;
    if (i < copies) {
        copy_pages(args, i % rows, i / rows);
    } else {
        move_columns(args.a, (i - copies) / groups, (i - copies) % groups, table_groups);
    }
}

}  // namespace

extern "C" {

QWN_CUDA_ABI_API uint64_t qwn_hip_ext_beam_select_workspace_bytes(uint32_t sequences, uint32_t beams, uint32_t vocab,
                                                                  uint32_t count) {
    if (!select_sizes(sequences, beams, vocab, count)) return 0;
    const uint64_t rows = static_cast<uint64_t>(sequences) * beams, parts = parts_of(vocab, kSlice<float>);
    return sums_bytes(rows, parts) + rows * parts * count * sizeof(uint64_t);
}

QWN_CUDA_ABI_API int qwn_hip_ext_beam_select_device(QwnCudaContextHandle *handle, const QwnHipBeamSelectRequest *r, void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || !r || !header_ok(*r) || r->sequences == 0 || r->beams == 0 || r->vocab == 0 || r->count == 0 || !r->logits || !r->scores ||
        !r->values || !r->parents || !r->tokens || !r->workspace || (reinterpret_cast<uintptr_t>(r->workspace) & 15u) ||
        r->dtype > QWN_HIP_DTYPE_BF16 || r->end_count > 4 || !r->next_scores != !r->next_parents || !r->next_scores != !r->next_tokens) {
        set_error("invalid beam selection request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    if (!select_sizes(r->sequences, r->beams, r->vocab, r->count)) {
        set_error("unsupported beam selection: %u sequences of %u beams, %u candidates of %u tokens", r->sequences, r->beams, r->count,
                  r->vocab);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    SelectArgs a{};
    a.in_stride = stride_or(r->in_stride, r->vocab);
    if (a.in_stride < r->vocab) {
        set_error("beam selection request: a row stride is shorter than its row");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t rows = static_cast<uint64_t>(r->sequences) * r->beams, found = static_cast<uint64_t>(r->sequences) * r->count;
    const Rows logits = row_block(r->logits, rows, r->vocab, a.in_stride, dtype_bytes(r->dtype)), scores = list_of_bytes(r->scores, 4 * rows);
    const Rows outs[7] = {list_of_bytes(r->workspace, qwn_hip_ext_beam_select_workspace_bytes(r->sequences, r->beams, r->vocab, r->count)),
                          list_of_bytes(r->values, 4 * found),      list_of_bytes(r->parents, 4 * found),
                          list_of_bytes(r->tokens, 4 * found),      list_of_bytes(r->next_parents, 4 * rows),
                          list_of_bytes(r->next_tokens, 4 * rows),  list_of_bytes(r->next_scores, 4 * rows)};
    bool bad = false;
    for (int i = 0; i < 7; ++i) {
        bad = bad || overlap(outs[i], logits) || (overlap(outs[i], scores) && !(i == 6 && in_place(outs[i], scores)));
        for (int k = 0; k < i; ++k) bad = bad || overlap(outs[i], outs[k]);
    }
    if (bad) {
        set_error("beam selection request: an output or the workspace overlaps an input or another output");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("beam selection device", device.error());
    a.logits = r->logits;
    a.scores = r->scores;
    a.values = r->values;
    a.parents = r->parents;
    a.tokens = r->tokens;
    a.next_scores = r->next_scores;
    a.next_parents = r->next_parents;
    a.next_tokens = r->next_tokens;
    a.beams = r->beams;
    a.vocab = r->vocab;
    a.count = r->count;
    a.end_count = r->end_count;
    std::copy(r->end_tokens, r->end_tokens + 4, a.end_tokens);
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    const hipError_t e = r->dtype == QWN_HIP_DTYPE_F32   ? launch_select<float>(a, r->sequences, r->workspace, s)
                         : r->dtype == QWN_HIP_DTYPE_F16 ? launch_select<f16>(a, r->sequences, r->workspace, s)
                                                         : launch_select<bf16>(a, r->sequences, r->workspace, s);
    return e == hipSuccess ? QWN_CUDA_STATUS_OK : hip_fail("beam selection launch", e);
}

QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_beam_advance_device(QwnCudaContextHandle *handle, const QwnHipPagedKvHandle *caches,
                                                              uint32_t count, const QwnHipBeamAdvanceRequest *r, void *stream) {
    Context *ctx = context_of(handle);
    if (!ctx || (count && !caches) || !r || !header_ok(*r) || r->sequences == 0 || r->beams == 0 || r->table_stride == 0 || !r->parents ||
        !r->past || !r->past_out || !r->page_table || !r->page_table_out || !r->spare || !r->spare_out || !r->history != !r->history_out ||
        (r->history && r->history_length == 0) || r->page_tokens < kPagedTile || r->page_tokens > 1024 ||
        (r->page_tokens & (r->page_tokens - 1)) || r->added > 0x7fffffffu) {
        set_error("invalid beam advance request");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    const uint64_t rows = static_cast<uint64_t>(r->sequences) * r->beams;
    const uint64_t table_groups = (static_cast<uint64_t>(r->table_stride) + kThreads - 1) / kThreads;
    const uint64_t history_groups = r->history ? (static_cast<uint64_t>(r->history_length) + kThreads - 1) / kThreads : 0;
    const uint64_t groups = table_groups + history_groups;
    if (r->beams > kBeamsMost || rows > 65535 || count > kCachesMost || rows * std::max(1u, count) + r->sequences * groups > 0xffffffffu / kThreads) {
        set_error("unsupported beam advance: %u sequences of %u beams, %u caches", r->sequences, r->beams, count);
        return QWN_CUDA_STATUS_UNSUPPORTED;
    }
    const Rows table = row_block(r->page_table, rows, r->table_stride, r->table_stride, 4),
               history = row_block(r->history, rows, r->history_length, r->history_length, 4);
    const Rows lists[4] = {list_of_bytes(r->parents, 4 * rows), list_of_bytes(r->past, 4 * rows), list_of_bytes(r->spare, 4 * rows),
                           list_of_bytes(r->tokens, 4 * rows)};
    const Rows outs[4] = {row_block(r->page_table_out, rows, r->table_stride, r->table_stride, 4),
                          row_block(r->history_out, rows, r->history_length, r->history_length, 4), list_of_bytes(r->past_out, 4 * rows),
                          list_of_bytes(r->spare_out, 4 * rows)};
    bool bad = false;
    for (int i = 0; i < 4; ++i) {
        for (const Rows &x : lists) bad = bad || overlap(outs[i], x);
        for (int k = 0; k < i; ++k) bad = bad || overlap(outs[i], outs[k]);
        bad = bad || (overlap(outs[i], table) && !(i == 0 && in_place(outs[i], table))) ||
              (overlap(outs[i], history) && !(i == 1 && in_place(outs[i], history)));
    }
    if (bad) {
        set_error("beam advance request: an output overlaps an input or another output");
        return QWN_CUDA_STATUS_INVALID_ARGUMENT;
    }
    std::lock_guard<std::mutex> lock(ctx->mutex);
    CopyArgs c{};
    for (uint32_t i = 0; i < count; ++i) {
        ResidentPaged *rp = paged_of(ctx, caches[i]);
        if (!rp) {
            set_error("paged KV-cache handle is not resident in this context");
            return QWN_CUDA_STATUS_INVALID_ARGUMENT;
        }
        if (i == 0) c.c = rp->c;
        if (rp->c.page_tokens != r->page_tokens || rp->c.pages != c.c.pages || rp->c.kv_heads != c.c.kv_heads || rp->c.width != c.c.width) {
            set_error("beam advance request: the caches are not of one shape, or not of pages of %u tokens", r->page_tokens);
            return QWN_CUDA_STATUS_INVALID_ARGUMENT;
        }
        c.pools[i] = rp->c.pool;
    }
    DeviceScope device(ctx->device);
    if (device.error() != hipSuccess) return hip_fail("beam advance device", device.error());
    AdvanceArgs &a = c.a;
    a.parents = r->parents;
    a.past = r->past;
    a.past_out = r->past_out;
    a.table = r->page_table;
    a.table_out = r->page_table_out;
    a.spare = r->spare;
    a.spare_out = r->spare_out;
    a.tokens = r->tokens;
    a.history = r->history;
    a.history_out = r->history_out;
    a.beams = r->beams;
    while ((1u << a.page_shift) < r->page_tokens) ++a.page_shift;
    a.table_stride = r->table_stride;
    a.added = r->added;
    a.history_length = r->history_length;
    hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
    // the copies read the tables as they were: a launch of their own where these are in place
    const uint32_t copies = static_cast<uint32_t>(rows * std::max(1u, count)), moves = static_cast<uint32_t>(r->sequences * groups);
    const bool in_two = r->page_table_out == r->page_table;
    auto launch = [&](uint32_t first, uint32_t n) {
        hipLaunchKernelGGL(beam_advance_kernel, dim3(n), dim3(kThreads), 0, s, c, first, copies, static_cast<uint32_t>(rows),
                           static_cast<uint32_t>(groups), static_cast<uint32_t>(table_groups));
        return hipGetLastError();
    };
    hipError_t e = launch(0, in_two ? copies : copies + moves);
    if (e == hipSuccess && in_two) e = launch(copies, moves);
    if (e != hipSuccess) return hip_fail("beam advance launch", e);
    ctx->telemetry.kv_cache_kernel_count++;
    return QWN_CUDA_STATUS_OK;
}

}  // extern "C"
