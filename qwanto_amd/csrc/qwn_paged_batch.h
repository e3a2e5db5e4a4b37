// Host state of a paged KV cache, and the search of a ragged batch by the
// workgroups that work on it.
#pragma once

#include "qwn_context.h"
#include "qwn_hip_ext.h"
#include "qwn_internal.h"
#include "qwn_overlap.h"
#include "qwn_paged.h"

namespace qwn {

// The cache of a handle this context issued (lock held); null otherwise.
ResidentPaged *paged_of(Context *ctx, const QwnHipPagedKvHandle &h);

// A caller's batch as kernels take it; false where it is not one.
bool batch_of(const QwnHipPagedBatch *b, PagedBatch &out);

// Whether what a call writes would change the batch that it reads.
inline bool overlaps_batch(const Rows &out, const PagedBatch &b) {
    const uint64_t n = b.sequences;
    return overlaps_any(out, {list_of_bytes(b.starts, 4 * (n + 1)), list_of_bytes(b.past, 4 * n),
                              list_of_bytes(b.table, 4 * n * b.table_stride)});
}

// A read of what no kernel of the call writes, at an address that every lane
// shares: through the scalar cache, apart from the vector loads in flight.
template <typename T>
__device__ __forceinline__ T scalar_load(const T *p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) T *>(reinterpret_cast<uintptr_t>(p));
}

// A sequence that every lane asks for.
__device__ __forceinline__ PagedSequence sequence_of(const PagedBatch &b, uint32_t s) {
    return paged_rows(b, scalar_load(b.starts + s), scalar_load(b.starts + s + 1), scalar_load(b.past + s));
}

// Inclusive sum over the wave's lanes (row shifts, then the rows' totals).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
    return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = scan_step<0x111, 0xf>(v);   // row_shr:1
    v = scan_step<0x112, 0xf>(v);
    v = scan_step<0x114, 0xf>(v);
    v = scan_step<0x118, 0xf>(v);
    v = scan_step<0x142, 0xa>(v);   // row_bcast:15 into rows 1, 3
    return scan_step<0x143, 0xc>(v);  // row_bcast:31 into rows 2, 3
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// The sequence whose units (weight(q) of them) hold number `index`, counted
// over the sequences in order, and its number within the sequence; false past
// the last.  Every wave searches for itself, 64 sequences a step.
template <typename W>
__device__ __forceinline__ bool find_in(const PagedBatch &b, uint32_t index, W weight, uint32_t &seq, uint32_t &at,
                                        PagedSequence &q) {
    const uint32_t lane = threadIdx.x % kWaveSize;
    for (uint32_t s0 = 0; s0 < b.sequences; s0 += kWaveSize) {
        const uint32_t s = s0 + lane;
        const PagedSequence mine = s < b.sequences ? paged_sequence(b, s) : PagedSequence{};
        const uint32_t n = weight(mine), end = wave_scan(n);
        const uint64_t past = __ballot(end > index);
        if (past) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = s0 + first;
            at = index - (lane_of(end, first) - lane_of(n, first));
            if (at >= lane_of(n, first)) return false;  // starts that do not ascend: the sums have wrapped
            q = PagedSequence{lane_of(mine.row, first), lane_of(mine.rows, first), lane_of(mine.past, first)};
            return true;
        }
        index -= lane_of(end, kWaveSize - 1);
    }
    return false;
}

__device__ __forceinline__ bool find_unit(const PagedBatch &b, uint32_t index, uint32_t &seq, uint32_t &at, PagedSequence &q) {
    return find_in(b, index, [](const PagedSequence &x) { return paged_units(x); }, seq, at, q);
}

}  // namespace qwn
