// The paged cache and a batch of new tokens as the kernels see them.
#pragma once

#include "q4b_kernels.h"

namespace q4b {

// codes in the status word for descriptors that do not hold together (q4b_sync: bad argument); the codes of expired
// waits are smaller
enum : uint32_t { kBadDescriptor = 0x1000u, kBadPage = kBadDescriptor | 1u, kBadLength = kBadDescriptor | 2u,
                  kBadBegin = kBadDescriptor | 3u };

// Only a word that holds nothing is written: the code of an expired wait stays (q4b_sync has more to put right after
// one), however close behind it the descriptor's comes.
__host__ __device__ inline void report(uint32_t *status, uint32_t code) {
#ifdef __CUDA_ARCH__
    atomicCAS(status, 0u, code);
#else
    if (*status == 0) *status = code;  // the index arithmetic below is checked on the host too
#endif
}

// Rows [begin, begin + count) belong to sequence s; its last row sits at place length - 1.
struct SequenceRows {
    uint32_t begin, count, length;
};
// The descriptor's numbers held to what the buffers have, whatever they say.  The length of a sequence that brings no token
// is used for nothing and may be anything.
__host__ __device__ inline SequenceRows sequence_rows(const BatchView &batch, uint32_t page_tokens, uint32_t s, uint32_t *status) {
    SequenceRows rows;
    const uint32_t from = batch.begin[s], to = batch.begin[s + 1];
    rows.begin = from < batch.tokens ? from : batch.tokens;
    const uint32_t end = to < batch.tokens ? to : batch.tokens;
    rows.count = end > rows.begin ? end - rows.begin : 0;
    if (to < from || to > batch.tokens) report(status, kBadBegin);
    const uint64_t room = (uint64_t)batch.table_stride * page_tokens;
    rows.length = batch.lengths[s];
    if (rows.length > room || rows.length > 0x7fffffffu) {
        if (rows.count != 0) report(status, kBadLength);
        rows.length = room < 0x7fffffffu ? (uint32_t)room : 0x7fffffffu;
    }
    return rows;
}

constexpr uint32_t kGroupKeys = 16;  // keys that attention takes together: the rows of one matrix product

// The groups of keys that a run of rows of one sequence may see: [0, sink) and [first, end).
struct Groups {
    uint32_t sink, first, end;
    __host__ __device__ inline uint32_t count() const { return sink + (end - first) == 0 ? 1u : sink + (end - first); }  // an empty unit still answers
    __host__ __device__ inline uint32_t at(uint32_t i) const { return i < sink ? i : first + (i - sink); }
};
// rows from token `token0` to `token1` (inclusive) of the sequence's new ones
template <uint32_t KEYS = kGroupKeys>
__host__ __device__ inline Groups groups_of(const SequenceRows &rows, uint32_t token0, uint32_t token1, uint32_t window,
                                            uint32_t sinks) {
    Groups g;
    const int64_t low = (int64_t)rows.length - rows.count + token0, high = (int64_t)rows.length - rows.count + token1;
    g.end = high < 0 ? 0u : (uint32_t)(high / KEYS) + 1;
    g.first = 0;
    g.sink = 0;
    if (window != 0 && low - (int64_t)window + 1 > 0) {
        const uint32_t first = (uint32_t)((low - (int64_t)window + 1) / KEYS);
        g.first = first < g.end ? first : g.end;
        const uint32_t sink = (uint32_t)(((uint64_t)sinks + KEYS - 1) / KEYS);
        g.sink = sink < g.first ? sink : g.first;
    }
    return g;
}

// the sequence of a row, found by the whole warp: the number of sequences that end at or before it
__device__ inline uint32_t sequence_of_row(const BatchView &batch, uint32_t row, uint32_t lane) {
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < batch.sequences; s0 += 32) {
        const bool ended = s0 + lane < batch.sequences && batch.begin[s0 + lane + 1] <= row;
        before += __popc(__ballot_sync(0xffffffffu, ended));
    }
    return before;
}

}  // namespace q4b
