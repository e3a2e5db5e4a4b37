// Checks of the paged cache's addressing and work split on the host; prints
// the first that fails, or "ok".
#include "qwn_paged.h"

#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <utility>
#include <vector>

using namespace qwn;

#define CHECK(c)                                             \
    do {                                                     \
        if (!(c)) {                                          \
            std::printf("line %d: %s\n", __LINE__, #c);      \
            return 1;                                        \
        }                                                    \
    } while (0)

static int layout() {
    for (uint32_t d : {1u, 2u, 32u, 64u, 65u, 80u, 96u, 128u, 192u, 256u}) {
        const uint32_t w = paged_width(d);
        CHECK(w >= d && (w == 64 || w == 128 || w == 256));
        // every code of a tile has 4 bits of its own within the codes
        for (int value = 0; value < 2; ++value) {
            std::set<uint32_t> bits;
            for (uint32_t t = 0; t < kPagedTile; ++t)
                for (uint32_t c = 0; c < w; ++c) {
                    const uint32_t word = value ? paged_value_word(w, t, c) : paged_key_word(w, t, c);
                    const uint32_t bit = value ? paged_value_bit(t, c) : paged_key_bit(c);
                    CHECK(word * 4 + 4 <= paged_codes_bytes(w) && bit <= 28 && bit % 4 == 0);
                    CHECK(bits.insert(word * 32 + bit).second);
                }
            CHECK(bits.size() * 4 == paged_codes_bytes(w) * 8);
        }
        // a lane's words lie next to each other, 16 bytes (8) a load
        for (uint32_t lane = 0; lane < 64; ++lane)
            for (uint32_t j = 0; j < w / 32; ++j)
                if (j % (w >= 128 ? 4 : 2)) CHECK(paged_word(w, lane, j) == paged_word(w, lane, j - 1) + 1);
        CHECK(paged_value_scales_at(w) + paged_scales_bytes(w) == paged_block_bytes(w) && paged_block_bytes(w) % 16 == 0);
        // blocks of pages, heads and tiles fill the pool without overlap
        PagedKv c;
        c.pages = 3;
        c.page_tokens = 64;
        c.page_shift = 6;
        c.kv_heads = 3;
        c.width = w;
        std::set<size_t> at;
        for (uint32_t p = 0; p < 3; ++p)
            for (uint32_t h = 0; h < 3; ++h)
                for (uint32_t t = 0; t < 4; ++t) at.insert(paged_block_at(c, p, t, h));
        CHECK(at.size() == 36 && *at.rbegin() + paged_block_bytes(w) == paged_block_at(c, 3, 0, 0));
        size_t next = 0;
        for (size_t b : at) {
            CHECK(b == next);
            next += paged_block_bytes(w);
        }
    }
    PagedKv big;
    big.page_tokens = 1024;
    big.page_shift = 10;
    big.kv_heads = 8;
    big.width = 128;
    CHECK(paged_block_at(big, 100000, 0, 0) == 100000ull * 8 * 64 * 2304);  // past 32 bits
    return 0;
}

static int pages() {
    PagedKv c;
    c.pages = 4;
    c.page_tokens = 16;
    c.page_shift = 4;
    const int32_t starts[] = {0, 1, 1, 3, 2, -1, 9}, past[] = {0, 5, -1, 7, 0, 2147483647};
    const int32_t table[] = {0, 3, 4, -1, 2147483647, -2147483647, 1, 1};
    PagedBatch b;
    b.sequences = 6;
    b.tokens = 8;
    b.table_stride = 8;
    b.starts = starts;
    b.past = past;
    b.table = table;
    uint32_t page = 0;
    const bool want[] = {true, true, false, false, false, false, true, true};
    for (uint32_t i = 0; i < 8; ++i)
        for (uint32_t t : {16 * i, 16 * i + 15}) {
            CHECK(paged_page(c, b, 0, t, page) == want[i]);
            if (want[i]) CHECK(page == static_cast<uint32_t>(table[i]));
        }
    CHECK(!paged_page(c, b, 0, 128, page) && !paged_page(c, b, 0, 0xffffffffu, page));
    CHECK(paged_sequence(b, 0).rows == 1 && paged_sequence(b, 0).row == 0);
    CHECK(paged_sequence(b, 1).rows == 0);   // no rows
    CHECK(paged_sequence(b, 2).rows == 0);   // a negative length
    CHECK(paged_sequence(b, 3).rows == 0);   // descending
    CHECK(paged_sequence(b, 4).rows == 0);   // descending below zero
    CHECK(paged_sequence(b, 5).rows == 0);   // from a negative start past the rows
    return 0;
}

static int units() {
    std::srand(1);
    for (int round = 0; round < 20000; ++round) {
        const uint32_t s = 1 + std::rand() % 6;
        uint32_t tokens = 0, count = 0;
        for (uint32_t i = 0; i < s; ++i) {
            PagedSequence q;
            q.past = std::rand() % 20;
            q.rows = std::rand() % 3 ? std::rand() % 12 : 0;
            std::set<uint32_t> groups;
            for (uint32_t r = 0; r < q.rows; ++r) groups.insert((q.past + r) / kPagedUnit);
            CHECK(groups.size() == paged_units(q));
            tokens += q.rows;
            count += paged_units(q);
        }
        CHECK(count <= paged_units_most(s, tokens) || tokens == 0);
    }
    return 0;
}

// Workers write the partial sums of the blocks they have parts of; the merge
// reads those of each block's workers: the same ones, each written once.
static int split() {
    std::srand(2);
    for (int round = 0; round < 6000; ++round) {
        const uint32_t start = std::rand() % 4;
        std::vector<uint64_t> first, pieces;
        uint64_t total = 0;
        for (int i = 1 + std::rand() % 12; i > 0; --i) {
            first.push_back(total + start);   // the first piece's unit
            pieces.push_back(1 + std::rand() % (std::rand() % 2 ? 3 : 90));
            total += start + pieces.back();
        }
        uint32_t workers = 1 + std::rand() % 40;
        if (workers > total) workers = static_cast<uint32_t>(total);
        std::map<uint32_t, std::pair<size_t, uint32_t>> written;  // partial -> (block, worker)
        std::vector<int> whole(first.size(), 0);
        for (uint32_t w = 0; w < workers; ++w) {
            const uint64_t b = paged_share(total, workers, w), e = paged_share(total, workers, w + 1);
            CHECK(b < e);
            for (uint64_t u = b; u < e; ++u) CHECK(paged_worker(total, workers, u) == w);
            for (size_t i = 0; i < first.size(); ++i) {
                const uint64_t from = first[i] > b ? first[i] : b;
                const uint64_t to = first[i] + pieces[i] < e ? first[i] + pieces[i] : e;
                if (from >= to) continue;
                if (to - from == pieces[i]) {
                    ++whole[i];
                } else {
                    CHECK(written.insert({paged_partial(total, workers, first[i], w), {i, w}}).second);
                }
            }
        }
        CHECK(paged_share(total, workers, workers) == total);
        for (size_t i = 0; i < first.size(); ++i) {
            const uint32_t w0 = paged_worker(total, workers, first[i]);
            const uint32_t w1 = paged_worker(total, workers, first[i] + pieces[i] - 1);
            if (w0 == w1) {
                CHECK(whole[i] == 1);
                continue;
            }
            CHECK(whole[i] == 0);
            for (uint32_t w = w0; w <= w1; ++w) {
                const uint32_t part = paged_partial(total, workers, first[i], w);
                CHECK(w == w0 || part == 2 * w);   // what the merge takes for granted
                const auto it = written.find(part);
                CHECK(it != written.end() && it->second.first == i && it->second.second == w);
                written.erase(it);
            }
        }
        CHECK(written.empty());
    }
    return 0;
}

int main() {
    if (layout() || pages() || units() || split()) return 1;
    std::puts("ok");
    return 0;
}
