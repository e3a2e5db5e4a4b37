// Host state of a paged KV cache, and the search of a ragged batch by the
// workgroups that work on it.
#pragma once

#include "qwn_context.h"
#include "qwn_hip_ext.h"
#include "qwn_internal.h"
#include "qwn_paged.h"

namespace qwn {

// The cache of a handle this context issued (lock held); null otherwise.
ResidentPaged *paged_of(Context *ctx, const QwnHipPagedKvHandle &h);

// A caller's batch as kernels take it; false where it is not one.
bool batch_of(const QwnHipPagedBatch *b, PagedBatch &out);

__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {  // inclusive
    const uint32_t lane = threadIdx.x % kWaveSize;
#pragma unroll
    for (int off = 1; off < kWaveSize; off <<= 1) {
        const uint32_t o = __shfl_up(v, off);
        if (lane >= static_cast<uint32_t>(off)) v += o;
    }
    return v;
}

// The sequence whose units (weight(s) of them) hold number `index`, counted
// over the sequences in order, and its number within the sequence; false past
// the last.  Every wave searches for itself, 64 sequences a step.
template <typename W>
__device__ __forceinline__ bool find_in(const PagedBatch &b, uint32_t index, W weight, uint32_t &seq, uint32_t &at) {
    const uint32_t lane = threadIdx.x % kWaveSize;
    for (uint32_t s0 = 0; s0 < b.sequences; s0 += kWaveSize) {
        const uint32_t s = s0 + lane;
        const uint32_t n = s < b.sequences ? weight(s) : 0u;
        const uint32_t end = wave_scan(n);
        const uint64_t past = __ballot(end > index);
        if (past) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = s0 + first;
            at = index - (__shfl(end, first) - __shfl(n, first));
            seq = __builtin_amdgcn_readfirstlane(seq);
            at = __builtin_amdgcn_readfirstlane(at);
            return true;
        }
        index -= __shfl(end, kWaveSize - 1);
    }
    return false;
}

__device__ __forceinline__ bool find_unit(const PagedBatch &b, uint32_t index, uint32_t &seq, uint32_t &at) {
    return find_in(b, index, [&](uint32_t s) { return paged_units(paged_sequence(b, s)); }, seq, at);
}

}  // namespace qwn
