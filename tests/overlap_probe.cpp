// Buffers that share a byte, against a count of their bytes.
#include "qwn_overlap.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace qwn;

namespace {

char memory[4096];

bool share(const Rows &a, const Rows &b) {
    if (a.none() || b.none()) return false;
    std::vector<char> used(sizeof(memory), 0);
    const auto at = [](const Rows &r, uint64_t i) { return r.at() + i * r.stride - reinterpret_cast<uintptr_t>(memory); };
    for (uint64_t i = 0; i < a.rows; ++i)
        for (uint64_t k = 0; k < a.width; ++k) used[at(a, i) + k] = 1;
    for (uint64_t i = 0; i < b.rows; ++i)
        for (uint64_t k = 0; k < b.width; ++k)
            if (used[at(b, i) + k]) return true;
    return false;
}

void expect(bool got, bool want, const char *what, const Rows &a, const Rows &b) {
    if (got == want) return;
    const auto p = [](const Rows &r) { return static_cast<long>(r.at() - reinterpret_cast<uintptr_t>(memory)); };
    std::printf("%s: %ld %lu x %lu / %lu and %ld %lu x %lu / %lu: %d\n", what, p(a), a.rows, a.width, a.stride, p(b), b.rows, b.width,
                b.stride, got);
    std::exit(1);
}

}  // namespace

int main() {
    std::srand(1);
    const auto any = [](uint64_t n) { return static_cast<uint64_t>(std::rand()) % n; };
    uint64_t met = 0;
    for (int i = 0; i < 300000; ++i) {
        Rows r[2];
        const uint64_t shared = 1 + any(24);
        for (Rows &x : r) {
            x.data = any(50) ? memory + any(300) : nullptr;
            x.rows = any(12);
            x.stride = any(2) ? shared : 1 + any(24);
            x.width = any(4) ? any(x.stride + 1) : x.stride;
            if (x.rows == 1 && any(2)) x.stride = 0;   // of one row it does not matter
        }
        const bool want = share(r[0], r[1]);
        met += want;
        expect(overlap(r[0], r[1]), want, "overlap", r[0], r[1]);
        expect(overlap(r[1], r[0]), want, "overlap", r[1], r[0]);
        expect(overlaps_any(r[0], {Rows{}, r[1]}), want, "any", r[0], r[1]);
    }
    if (met < 30000 || met > 270000) return std::printf("%lu of the pairs share a byte\n", met), 1;
    const Rows a = row_block(memory, 4, 3, 8, 2), b = row_block(memory + 6, 4, 5, 8, 2), c = row_block(memory + 6, 4, 6, 8, 2);
    if (a.width != 6 || a.stride != 16 || overlap(a, b) || !overlap(a, c) || overlap(a, list_of_bytes(memory + 54, 100)) ||
        !overlap(a, list_of_bytes(memory + 53, 1)) || !in_place(a, a) || in_place(a, b))
        return std::printf("columns of one buffer\n"), 1;
    std::printf("ok\n");
    return 0;
}
