// paged.cuh -- what the kernels over a paged K/V cache share: the cache as a kernel sees it, where a token of a ragged
// batch sits, and the checks of a descriptor (paged_kv.cu has the code).
#pragma once

#include "tc_common.cuh"

namespace tc {

// Pools [numPages][pageRows][nKV][hd] (int8: scales [numPages][pageRows][nKV]); row r of sequence b is row r % pageRows of page
// pages[b][r / pageRows].  Sequence b has lens[b] rows, the last of them those of its new tokens, which are rows starts[b] ..
// starts[b + 1] - 1 of the call's token arrays (starts null: perSeq tokens each).
struct PagedView {
    const int32_t *pages;
    const uint32_t *lens, *starts;
    uint32_t batch, pagesPerSeq, numPages, pageRows, nKV, tokens, perSeq;
    unsigned int *err;
};

int pagedCheck(const tc_paged_kv *c, const char *what);  // TC_OK or an error with its text set
PagedView pagedView(const tc_paged_kv *c, unsigned int *err);

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t seqStart(const PagedView &v, uint32_t b) { return v.starts != nullptr ? __ldg(v.starts + b) : b * v.perSeq; }

// The sequence of token t, found by a group of G lanes that work on the same token (starts ascend: the last b with starts[b] <= t),
// and the token's position in it.  False: the token lies behind the last sequence (or ahead of the first).  A position before the first row is negative.
template <uint32_t G>
__device__ __forceinline__ bool findToken(const PagedView &v, uint32_t t, uint32_t &seq, int64_t &pos) {
    uint32_t b = 0, end;
    if (v.starts == nullptr) {
        b = t / v.perSeq;
        end = (b + 1u) * v.perSeq;
    } else {
        const uint32_t lane = threadIdx.x & 31u, i = lane & (G - 1u);
        const uint32_t mask = (G == 32 ? 0xffffffffu : ((1u << (G & 31u)) - 1u) << (lane & ~(G - 1u)));
        uint32_t n = v.batch;
        while (n > 1u) {
            const uint32_t step = (n + G - 1u) / G, at = i * step;
            const uint32_t hits = __popc(__ballot_sync(mask, at < n && __ldg(v.starts + b + at) <= t) & mask);
            const uint32_t off = (hits ? hits - 1u : 0u) * step;
            b += off;
            n = min(step, n - off);
        }
        end = __ldg(v.starts + b + 1u);
        if (t >= end || (b == 0u && t < __ldg(v.starts))) return false;
    }
    seq = b;
    pos = static_cast<int64_t>(__ldg(v.lens + b)) - static_cast<int64_t>(end - t);
    return true;
}

// The pool row of row `pos` of sequence `seq`; false where the table has no page for it or the pool no such page.
__device__ __forceinline__ bool pagedRow(const PagedView &v, uint32_t seq, int64_t pos, size_t &row) {
    if (pos < 0) return false;
    const uint64_t slot = static_cast<uint64_t>(pos) / v.pageRows;
    if (slot >= v.pagesPerSeq) return false;
    const int32_t page = __ldg(v.pages + static_cast<size_t>(seq) * v.pagesPerSeq + slot);
    if (static_cast<uint32_t>(page) >= v.numPages) return false;  // (negative ones too)
    row = static_cast<size_t>(page) * v.pageRows + static_cast<size_t>(static_cast<uint64_t>(pos) - slot * v.pageRows);
    return true;
}
#endif

}  // namespace tc
