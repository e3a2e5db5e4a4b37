// The paged 4-bit KV cache: where a code and a scale lie, and which tokens of
// a ragged batch a workgroup takes.  Plain C++ as well as device code, so
// that the addressing is checked on the host.
//
// A page holds page_tokens slots in tiles of 16.  Of each tile the pool keeps
// one block per KV head, everything that attention reads of these 16 tokens
// next to each other (2304 bytes at 128 channels):
//
//   keys    [load][lane 64][JW words]   lane 16 g + n: token n, word j the
//           channels 32 j + 8 g .. + 7; element i of the 8 in nibble
//           (i >> 1) | (i & 1) << 2
//   values  [load][lane 64][JW words]   lane 16 g + n: tokens 4 g .. 4 g + 3 of
//           the channels 32 w + n (low byte pairs) and 32 w + 16 + n
//   key scales, value scales            [token][group] f16 minimum, f16 step (the upper half)
//
// with JW = 4 words (2 at 64 channels) of the head's channels / 32, so that a
// wave's load of 16 bytes a lane is one contiguous kilobyte and each word is
// one lane's share of a v_mfma_f32_16x16x32_f16 operand: nibbles b and b + 4
// are the two halves of one register.  As they lie there, nibble 0 or 1 of a
// half is an f16 of 2^-24 or 2^-20 times its code, a number below the normal
// ones that the matrix cores take as it is.  Heads of 32 to 256 channels are stored
// as 64, 128 or 256; the channels past head_dim are zeros.
#pragma once

#include <cstddef>
#include <cstdint>

#if defined(__HIPCC__)
#define QWN_HD __host__ __device__ __forceinline__
#else
#define QWN_HD inline
#endif

namespace qwn {

constexpr uint32_t kPagedTile = 16;    // slots of a tile
constexpr uint32_t kPagedGroup = 64;   // channels that share a step and a minimum
constexpr uint32_t kPagedUnit = 4;     // slots that share a word of values

struct PagedKv {
    uint32_t pages = 0;
    uint32_t page_tokens = 0;    // 1 << page_shift
    uint32_t page_shift = 0;
    uint32_t kv_heads = 0;
    uint32_t head_dim = 0;
    uint32_t width = 0;          // head_dim as stored: 64, 128 or 256
    uint32_t rope_dims = 0;
    uint8_t *pool = nullptr;
    double *freqs = nullptr;     // [rope_dims / 2]: theta^(-2 i / rope_dims)
    uint64_t bytes = 0;
};

QWN_HD uint32_t paged_width(uint32_t head_dim) { return head_dim <= 64 ? 64u : head_dim <= 128 ? 128u : 256u; }
QWN_HD uint32_t paged_codes_bytes(uint32_t width) { return kPagedTile * width / 2; }
QWN_HD uint32_t paged_scales_bytes(uint32_t width) { return kPagedTile * (width / kPagedGroup) * 4; }
QWN_HD uint32_t paged_block_bytes(uint32_t width) { return 2 * (paged_codes_bytes(width) + paged_scales_bytes(width)); }
QWN_HD uint32_t paged_values_at(uint32_t width) { return paged_codes_bytes(width); }
QWN_HD uint32_t paged_key_scales_at(uint32_t width) { return 2 * paged_codes_bytes(width); }
QWN_HD uint32_t paged_value_scales_at(uint32_t width) { return 2 * paged_codes_bytes(width) + paged_scales_bytes(width); }

// Byte of the block of (page, tile of the page, head).
QWN_HD size_t paged_block_at(const PagedKv &c, uint32_t page, uint32_t tile, uint32_t head) {
    return ((static_cast<size_t>(page) * c.kv_heads + head) * (c.page_tokens / kPagedTile) + tile) *
           paged_block_bytes(c.width);
}

// Word of lane `lane`'s word j within the codes of a block.
QWN_HD uint32_t paged_word(uint32_t width, uint32_t lane, uint32_t j) {
    const uint32_t jw = width >= 128 ? 4u : 2u;
    return ((j / jw) * 64 + lane) * jw + j % jw;
}
// Word and bit of a key's code, of a value's.
QWN_HD uint32_t paged_key_word(uint32_t width, uint32_t token, uint32_t channel) {
    return paged_word(width, channel % 32 / 8 * 16 + token, channel / 32);
}
QWN_HD uint32_t paged_key_bit(uint32_t channel) { return 4 * (((channel & 7u) >> 1) | ((channel & 1u) << 2)); }
QWN_HD uint32_t paged_value_word(uint32_t width, uint32_t token, uint32_t channel) {
    return paged_word(width, token / kPagedUnit * 16 + channel % 16, channel / 32);
}
QWN_HD uint32_t paged_value_bit(uint32_t token, uint32_t channel) {
    return 4 * (((channel / 16 & 1u) << 1) | ((token & 3u) >> 1) | ((token & 1u) << 2));
}

// A ragged batch as the device reads it.
struct PagedBatch {
    uint32_t sequences = 0;
    uint32_t tokens = 0;
    uint32_t table_stride = 0;
    const int32_t *starts = nullptr;
    const int32_t *past = nullptr;
    const int32_t *table = nullptr;
};

// Rows and cached tokens of sequence s: none where the starts or the length
// do not lie in the batch.
struct PagedSequence {
    uint32_t row = 0, rows = 0, past = 0;
};
QWN_HD PagedSequence paged_rows(const PagedBatch &b, int32_t r0, int32_t r1, int32_t past) {
    PagedSequence q;
    if (r0 < 0 || r1 <= r0 || static_cast<uint32_t>(r1) > b.tokens || past < 0) return q;
    q.row = static_cast<uint32_t>(r0);
    q.rows = static_cast<uint32_t>(r1 - r0);
    q.past = static_cast<uint32_t>(past);
    return q;
}

QWN_HD PagedSequence paged_sequence(const PagedBatch &b, uint32_t s) {
    return paged_rows(b, b.starts[s], b.starts[s + 1], b.past[s]);
}

// Page of a slot of sequence s; false where the table names none of the pool.
QWN_HD bool paged_page(const PagedKv &c, const PagedBatch &b, uint32_t s, uint32_t slot, uint32_t &page) {
    const uint32_t i = slot >> c.page_shift;
    if (i >= b.table_stride) return false;
    const int32_t p = b.table[static_cast<size_t>(s) * b.table_stride + i];
    page = static_cast<uint32_t>(p);
    return p >= 0 && page < c.pages;
}

// Aligned groups of 4 slots that the new tokens of a sequence reach, and the
// most of them that a batch can have: one for each token, and for long runs
// one for 4 tokens and a group cut at either end.
QWN_HD uint32_t paged_units(const PagedSequence &q) {
    return q.rows ? (q.past + q.rows - 1) / kPagedUnit - q.past / kPagedUnit + 1 : 0u;
}
inline uint32_t paged_units_most(uint32_t sequences, uint32_t tokens) {
    const uint64_t runs = static_cast<uint64_t>(tokens) / kPagedUnit + 2ull * sequences;
    return static_cast<uint32_t>(runs < tokens ? runs : tokens);
}

// Attention splits a list of `total` units of work among `workers`: worker w
// takes units paged_share(w) .. paged_share(w + 1) - 1, and paged_worker is the
// one that takes a unit.
QWN_HD uint64_t paged_share(uint64_t total, uint32_t workers, uint32_t w) { return total * w / workers; }
QWN_HD uint32_t paged_worker(uint64_t total, uint32_t workers, uint64_t unit) {
    return static_cast<uint32_t>(((unit + 1) * workers - 1) / total);
}
// A block of work is `start` units for its beginning, that no worker does
// anything for, and one for each of its pieces, the first of them unit `first`.
// Of a block whose pieces no worker has all of, worker w's partial sums: each
// worker keeps two, of a block that it begins in the middle of (or at its first
// piece) and of one that it does not come to the end of.
QWN_HD uint32_t paged_partial(uint64_t total, uint32_t workers, uint64_t first, uint32_t w) {
    return 2 * w + (paged_share(total, workers, w) < first ? 1u : 0u);
}

}  // namespace qwn
