// One token per row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// All three cuts keep a prefix of the order (largest logit first, the lowest index first among equals), so each is ONE
// composite number c = (ordered bits of the logit, complement of the index): an element stays when its own composite is
// at least the cut.  The token is then the first index at which the running sum of the kept weights
// exp((logit - largest) / temperature) passes uniform x total.  A row is never sorted.
//
// A row is spread over a cluster of 1 to 8 thread blocks.  Few rows are kept in shared memory after their one trip from
// HBM; with many rows in flight the passes read them again from L2 instead, which leaves room for two thread blocks
// per SM whose passes hide each other's waits (256 rows of 248,320 fp32 logits: 190 us against 282 us on chip; 18 rows the
// other way, 31 us on chip against 35 us, with top-p 72 us against 80 us).
//   extremes  the largest and the smallest finite logit (greedy ends here)
//   counts    2048 bins, linear in the distance to the largest logit: linear bins spread a row evenly, where bins of
//             the float's own bits would put most of it into a few and serialise the atomics.  With top-p alone the same
//             pass adds up all weights
//   few stay  (the usual case: the bins down to the border hold at most 2048 elements): these are gathered in the first
//             block of the cluster, sorted there, and everything else happens in that block
//   many stay the border's bin alone is gathered and ranked and gives the cut.  For top-p the counts only bracket the
//             border (a bin's weights differ by a per cent); the bracket is binned once more, now by exact weights
//   token     sums of kept weights per 128 words of the row, then within the one that the target falls into
//   A rare rest (both cuts deep in the row, thousands of equal logits at a border) goes through find_cut, which cuts the
//   span in question into 2048 again and again.
// Weights are integers in units of 2^-42 of the largest one's: sums are exact in any order of the atomics, so equal
// inputs give equal tokens.  What decides between neighbours of a border is the error of a running sum, so a weight is
// made to 2^-31, not to fp32's 2^-24 (whose argument alone would be off by 2^-24 x distance), whatever the logits' type:
// the distance and its product with log2(e) / temperature as unevaluated pairs of floats, a table of 2^(-j / 256), a cubic
// for the rest.  In fp64 the same pass is bound by the fp64 pipe and takes twice as long.
//
// Measured on B200 (248,320 logits a row): one fp32 row 10 us when greedy, 18 us with a top-k below 200, 29 to 61 us without
// one; 33 fp16 rows by top-p 95 us; 256 fp32 rows, the whole distribution, 190 us = 1.34 TB/s.  No unit is full in either of
// the last two: 55 instructions per logit take 58% of the issue slots (ALU 46%, FMA 26%, DRAM 18%) and waits for loads and
// barriers show at 43% of the warps; by top-p 134 instructions per logit take 51%, and barriers between a row's phases most.
#include "q4b_kernels.h"

#include <cooperative_groups.h>
#include <cmath>

namespace q4b {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kMostWarps = 32;
constexpr uint32_t kBins = 2048;           // at most: a thread of the cluster for each
constexpr uint32_t kMostBlocks = 8;        // thread blocks of a row
constexpr uint32_t kListed = 2048;         // elements that one block puts in order
constexpr uint32_t kTileRows4 = 4;         // 16-byte words of a tile: 4 per lane of a warp
constexpr uint32_t kTileWords = 32 * kTileRows4;
constexpr uint32_t kSliceBytes = 160 * 1024;  // of a row that a thread block may keep in shared memory
constexpr uint64_t kOne = 1ull << 42;      // the largest logit's weight

struct SampleShared {
    uint2 power[256];                      // 2^(-j / 256): in units of 2^-31 as an integer, and as a float's bits
    float high[kMostBlocks], low[kMostBlocks];
    uint64_t total[kMostBlocks];
    uint64_t parts[3][kMostBlocks];        // sums of the blocks' shares of the bins
    uint64_t warp_values[kMostWarps];
    float warp_high[kMostWarps], warp_low[kMostWarps];
    uint32_t first, listed, own_listed, low_bin, high_bin, low_before, found_count, fine_bin, fine_count;
    uint64_t found_before, cut;
    uint64_t span_low[kMostBlocks], span_high[kMostBlocks];
    uint32_t count[kBins];
    union {
        uint64_t list[kListed];            // composites
        uint64_t mass[kBins];
    };
    uint2 queue[16][64];                   // per warp: values and indices that wait for 31 others
    uint64_t sums[kListed];                // their weights; before that, what this block puts on the list
};

// 2^(-j / 256), by repeated multiplication in fp64 (256 roundings of 2^-53 each)
struct PowerTable {
    uint2 entry[256];
};
constexpr uint32_t float_bits(double x) {  // of 2^30 < x <= 2^31, rounded
    if (x >= 2147483648.0) return (158u << 23);
    return (157u << 23) | ((uint32_t)((x - 1073741824.0) / 128.0 + 0.5) & 0x7fffffu) +
                              (((uint32_t)((x - 1073741824.0) / 128.0 + 0.5) >> 23) << 23);
}
constexpr PowerTable make_powers() {
    PowerTable table = {};
    double value = 2147483648.0;
    for (int j = 0; j < 256; ++j) {
        table.entry[j].x = (uint32_t)(value + 0.5);
        table.entry[j].y = float_bits(value);
        value *= 0.997296056085470126;  // 2^(-1 / 256)
    }
    return table;
}
__device__ const PowerTable kPowers = make_powers();

__device__ inline float as_float(float x) { return x; }
__device__ inline float as_float(__half x) { return __half2float(x); }
__device__ inline float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// NaN counts as -infinity, both zeros are one number: in a composite; comparisons, weights (a NaN's is 0) and bins (the
// last) see to it by themselves
__device__ inline float tidy(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ inline uint64_t composite(float x, uint32_t index) {
    const uint32_t bits = __float_as_uint(tidy(x));
    const uint32_t ordered = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (uint64_t)ordered << 32 | (uint32_t)~index;
}
__device__ inline float logit_of(uint64_t c) {
    const uint32_t ordered = (uint32_t)(c >> 32);
    return __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
}
__device__ inline uint32_t index_of(uint64_t c) { return ~(uint32_t)c; }

__device__ inline uint64_t warp_sum(uint64_t x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ inline uint64_t warp_max(uint64_t x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, x, d);
        x = y > x ? y : x;
    }
    return x;
}
__device__ inline uint64_t warp_inclusive(uint64_t x) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= (uint32_t)d) x += y;
    }
    return x;
}
// the same in every thread of the block; `scratch` is free again afterwards
__device__ inline uint64_t block_max(uint64_t x, uint64_t *scratch) {
    x = warp_max(x);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = warp_max((threadIdx.x & 31) < blockDim.x / 32 ? scratch[threadIdx.x & 31] : 0);
    __syncthreads();
    return x;
}
// sum over the block, and (in `before`) over the threads in front of this one
__device__ inline uint64_t block_scan(uint64_t x, uint64_t *scratch, uint64_t &before) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t inclusive = warp_inclusive(x);
    if (lane == 31) scratch[warp] = inclusive;
    __syncthreads();
    const uint64_t warps = warp_inclusive(lane < blockDim.x / 32 ? scratch[lane] : 0);
    const uint64_t total = __shfl_sync(0xffffffffu, warps, 31);
    before = inclusive - x + (warp > 0 ? __shfl_sync(0xffffffffu, warps, warp - 1) : 0);
    __syncthreads();
    return total;
}
__device__ inline uint64_t block_sum(uint64_t x, uint64_t *scratch) {
    uint64_t before;
    return block_scan(x, scratch, before);
}

// This block's part of the row: `head` single values up to a 16-byte boundary, whole words, `tail` single values.
template <typename T>
struct Slice {
    const T *data;
    uint32_t begin, size, head, words, tail;
    static constexpr uint32_t kWord = 16 / sizeof(T);
    __device__ inline float at(uint32_t i) const { return as_float(data[i]); }
    __device__ inline uint32_t tiles() const { return (words + kTileWords - 1) / kTileWords; }
    __device__ inline void split(uint32_t skew) {
        head = min(size, skew == 0 ? 0u : (16u - skew) / (uint32_t)sizeof(T));
        words = (size - head) / kWord;
        tail = size - head - words * kWord;
    }
    // f(value, index within the slice) for the values of one tile, as a warp.  One word's code, not sixteen: a pass is
    // short, and the instructions of longer loops took more time to arrive than to run.
    template <typename F> __device__ inline void tile(uint32_t t, F f) const {
        const uint4 *const from = reinterpret_cast<const uint4 *>(data + head);
        uint32_t w = t * kTileWords + (threadIdx.x & 31);
        uint4 next = w < words ? from[w] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (uint32_t r = 0; r < kTileRows4; ++r, w += 32) {
            const uint4 word = next;
            if (r + 1 < kTileRows4 && w + 32 < words) next = from[w + 32];
            if (w < words) {
                const T *x = reinterpret_cast<const T *>(&word);
#pragma unroll
                for (uint32_t j = 0; j < kWord; ++j) f(as_float(x[j]), head + w * kWord + j);
            }
        }
    }
    // f over the values of a tile that may be `bound` or more (a NaN may), as a warp: they are collected and f runs for 32 at
    // a time, so a pass over a row of which little matters costs a comparison per value and f for those that do
    template <typename F> __device__ inline void tile_above(uint32_t t, float bound, uint2 *queue, F f) const {
        const uint4 *const from = reinterpret_cast<const uint4 *>(data + head);
        const uint32_t lane = threadIdx.x & 31, below = (1u << lane) - 1;
        uint32_t w = t * kTileWords + lane, waiting = 0;
        uint4 next = w < words ? from[w] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (uint32_t r = 0; r < kTileRows4; ++r, w += 32) {
            const uint4 word = next;
            const bool here = w < words;
            if (r + 1 < kTileRows4 && w + 32 < words) next = from[w + 32];
            const T *x = reinterpret_cast<const T *>(&word);
#pragma unroll
            for (uint32_t j = 0; j < kWord; ++j) {
                const float value = as_float(x[j]);
                const bool takes = here && !(value < bound);
                const uint32_t mask = __ballot_sync(0xffffffffu, takes);
                if (mask == 0) continue;
                if (takes) queue[waiting + __popc(mask & below)] = make_uint2(__float_as_uint(value), head + w * kWord + j);
                waiting += __popc(mask);
                if (waiting >= 32) {
                    __syncwarp();
                    const uint2 own = queue[lane], rest = queue[32 + lane];
                    __syncwarp();
                    waiting -= 32;
                    if (lane < waiting) queue[lane] = rest;
                    f(__uint_as_float(own.x), own.y);
                }
            }
        }
        __syncwarp();
        if (lane < waiting) f(__uint_as_float(queue[lane].x), queue[lane].y);
        __syncwarp();
    }
    // the same over the whole slice, as a block
    template <typename F> __device__ inline void each_above(float bound, uint2 *queue, F f) const {
        const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
        for (uint32_t t = warp; t < tiles(); t += (blockDim.x / 32)) tile_above(t, bound, queue, f);
        if (warp == 0 && lane < head + tail) {
            const uint32_t i = lane < head ? lane : size - tail + (lane - head);
            if (!(at(i) < bound)) f(at(i), i);
        }
    }
    // f over the whole slice, as a block
    template <typename F> __device__ inline void each(F f) const {
        const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
        for (uint32_t t = warp; t < tiles(); t += (blockDim.x / 32)) tile(t, f);
        if (warp == 0 && lane < head + tail) {
            const uint32_t i = lane < head ? lane : size - tail + (lane - head);
            f(at(i), i);
        }
    }
};

// Weights by the distance to the largest logit: about 45 instructions, which are what a pass costs, in one chain from the
// logit to the weight.  Without a branch in it several values' chains run side by side; with two the pass took 70 clocks
// per 32 values and scheduler, each chain waiting for the one before.
struct Weigh {
    const uint2 *power;
    float high, rate, rate_low;  // log2(e) / temperature = rate + rate_low; all finite
    float shrink;                // 1, or less where the largest logit is infinite
    __device__ inline void set(float largest, float temperature) {
        const double exact = 1.4426950408889634074 / (double)temperature;
        high = largest;
        shrink = 1.0f;
        rate = fminf((float)exact, 3.0e38f);
        rate_low = rate < 3.0e38f ? (float)(exact - (double)rate) : 0.0f;
        if (largest == INFINITY) {  // its equals share everything: they become the largest number, all else is halved and far away
            shrink = 0.5f;
            high = 3.402823466e38f;
            rate = 1.0f;
            rate_low = 0.0f;
        }
    }
    // of distance + distance_low >= 0; beyond 2^-43, overflow and NaN are nothing
    __device__ inline uint64_t at(float distance, float distance_low) const {
        const float y = distance * rate;
        const float y_low = fmaf(distance, rate_low, fmaf(distance, rate, -y)) + distance_low * rate;
        const float shifted = fmaf(y, 256.0f, 12582912.0f);  // 1.5 x 2^23: the nearest whole number of 1/256
        const uint32_t k = __float_as_uint(shifted) - 0x4b400000u;
        const float rest = fmaf(shifted - 12582912.0f, -1.0f / 256.0f, y) + y_low;
        const float q = rest * -0.693147180559945309f;
        const float more = q * fmaf(q, fmaf(q, 0.16666667f, 0.5f), 1.0f);  // 2^-rest - 1; q^4 / 24 < 2^-42
        const uint2 base = power[k & 255u];
        const uint32_t value = base.x + __float_as_uint(fmaf(__uint_as_float(base.y), more, 12582912.0f)) - 0x4b400000u;
        const uint32_t n = k >> 8 & 63u;
        const uint64_t weight = (((uint64_t)value << 11) + ((1ull << n) >> 1)) >> n;
        return y < 43.0f ? weight : 0;
    }
    __device__ inline uint64_t of(float x) const {
        float own;  // at most the largest (an infinity), a NaN stays one
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(own) : "f"(x * shrink), "f"(high));
        const float d = high - own;
        // d + low = high - x exactly, for 16-bit logits too: next to a large one a tiny one's bits end up beyond fp32's, and
        // leaving them out (2^-22 of a weight) saves 0.6 us of 95 for 33 rows
        const float back = high - d;
        const float low = (high - (d + back)) + (back - own);
        return at(d, low);
    }
};
// The bin of a distance, before it is cut off to a whole number.
__device__ inline float place_of(float x, float high, float to_bin, float last) {
    return x == high ? 0.0f : fminf((high - x) * to_bin, last);  // NaN (0 x infinity) is the last bin
}
__device__ inline uint32_t whole(float v) { return __float_as_uint(__fadd_rd(v, 8388608.0f)) & 0x7fffffu; }

// The sum of a value over the threads of the blocks in front of this one, and over those in front of this thread in its own;
// `all` is the sum over the cluster.  `slot` separates what is exchanged between two cluster barriers; the caller's
// barrier comes between tell_parts and sum_parts.
__device__ inline uint64_t tell_parts(cg::cluster_group &cluster, SampleShared &sh, uint32_t slot, uint64_t value) {
    uint64_t before;
    const uint64_t sum = block_scan(value, sh.warp_values, before);
    if (threadIdx.x < cluster.num_blocks()) cluster.map_shared_rank(&sh, threadIdx.x)->parts[slot][cluster.block_rank()] = sum;
    return before;
}
__device__ inline uint64_t sum_parts(cg::cluster_group &cluster, const SampleShared &sh, uint32_t slot, uint64_t &all) {
    uint64_t before = 0;
    all = 0;
    for (uint32_t r = 0; r < cluster.num_blocks(); ++r) {
        if (r < cluster.block_rank()) before += sh.parts[slot][r];
        all += sh.parts[slot][r];
    }
    return before;
}
// This thread's bin over the whole cluster: block r of n has bins [r, r + 1) x bins / n.
__device__ inline uint32_t my_bin(cg::cluster_group &cluster, uint32_t bins) {
    const uint32_t each = bins / cluster.num_blocks();
    return threadIdx.x < each ? cluster.block_rank() * each + threadIdx.x : 0xffffffffu;
}
template <typename V, typename F>
__device__ inline V over_blocks(cg::cluster_group &cluster, SampleShared &sh, bool any, F f) {
    V each[kMostBlocks], sum = 0;  // a round trip for all of them, not one each
#pragma unroll
    for (uint32_t r = 0; r < kMostBlocks; ++r) each[r] = any && r < cluster.num_blocks() ? f(cluster.map_shared_rank(&sh, r)) : 0;
#pragma unroll
    for (uint32_t r = 0; r < kMostBlocks; ++r) sum += each[r];
    return sum;
}
__device__ inline uint32_t count_of(cg::cluster_group &cluster, SampleShared &sh, uint32_t bin) {
    return over_blocks<uint32_t>(cluster, sh, bin != 0xffffffffu, [&](const SampleShared *other) { return other->count[bin]; });
}
__device__ inline uint64_t mass_of(cg::cluster_group &cluster, SampleShared &sh, uint32_t bin) {
    return over_blocks<uint64_t>(cluster, sh, bin != 0xffffffffu, [&](const SampleShared *other) { return other->mass[bin]; });
}
__device__ inline uint64_t reach_of(float share, uint64_t total) {
    const double reach = ceil((double)fmaxf(share, 0.0f) * (double)total);
    return reach < 1.0 ? 1ull : (uint64_t)reach;
}

// The elements that `wanted` names, as composites in the list of the cluster's first block; how many there are, or
// 0xffffffff when they are too many for it; `bound` is less than any of them, or -infinity (COLLECT: `wanted` is long
// and some per cent of the row pass the bound).  A block lists its own first: a place in another block's list is a round trip.
template <bool COLLECT, typename T, typename F>
__device__ uint32_t gather(cg::cluster_group &cluster, SampleShared &sh, const Slice<T> &slice, float bound, F wanted) {
    if (threadIdx.x == 0) sh.own_listed = 0;
    __syncthreads();
    auto list = [&](float x, uint32_t i) {
        if (wanted(x, i)) {
            const uint32_t place = atomicAdd(&sh.own_listed, 1u);
            if (place < kListed) sh.sums[place] = composite(x, slice.begin + i);
        }
    };
    if (COLLECT) slice.each_above(bound, sh.queue[threadIdx.x >> 5], list);
    else slice.each([&](float x, uint32_t i) { if (!(x < bound)) list(x, i); });
    __syncthreads();
    const uint32_t own = sh.own_listed, blocks = cluster.num_blocks(), rank = cluster.block_rank();
    if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->span_high[rank] = own;
    cluster.sync();
    uint32_t before = 0, all = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
        const uint32_t count = (uint32_t)sh.span_high[r];
        if (r < rank) before += count;
        all += count;
    }
    if (all > kListed) {
        cluster.sync();
        return 0xffffffffu;
    }
    SampleShared *leader = cluster.map_shared_rank(&sh, 0);
    for (uint32_t i = threadIdx.x; i < own; i += blockDim.x) leader->list[before + i] = sh.sums[i];
    if (rank == 0 && threadIdx.x == 0) sh.listed = all;
    cluster.sync();
    return all;
}

// The composite of the last element that stays, over the whole cluster, in every case.  By count: the `wanted`-th element
// of those at or above `floor`.  By mass: the first at which the running weight reaches `wanted`.
template <bool MASS, typename T>
__device__ __noinline__ uint64_t find_cut(cg::cluster_group &cluster, SampleShared &sh, const Slice<T> &slice, const Weigh &weigh,
                             float high, float to_bin, uint32_t bins, uint64_t floor, uint64_t wanted) {
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    bool by_distance = true;
    uint64_t span_low = floor, span_high = ~0ull;  // composites still in question, and how they are cut into bins
    uint32_t shift = 0;
    uint64_t before = 0;                           // count or mass above the span
    auto bin_of = [&](float x, uint64_t c) -> uint32_t {
        return by_distance ? whole(place_of(x, high, to_bin, (float)(bins - 1))) : (uint32_t)((span_high - c) >> shift);
    };
    auto in_span = [&](uint64_t c) { return c >= span_low && c <= span_high; };
    for (;;) {
        for (uint32_t b = threadIdx.x; b < kBins; b += blockDim.x) {
            sh.count[b] = 0;
            if (MASS) sh.mass[b] = 0;
        }
        __syncthreads();
        slice.each([&](float x, uint32_t i) {
            const uint64_t c = composite(x, slice.begin + i);
            if (!in_span(c)) return;
            const uint32_t b = bin_of(x, c);
            atomicAdd(&sh.count[b], 1u);
            if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)weigh.of(x));
        });
        cluster.sync();
        const uint32_t bin = my_bin(cluster, bins), number = count_of(cluster, sh, bin);
        const uint64_t own = MASS ? mass_of(cluster, sh, bin) : number;
        uint64_t running = tell_parts(cluster, sh, 0, own), all;
        cluster.sync();  // the bins have been read everywhere: the list may take their place
        running += before + sum_parts(cluster, sh, 0, all);
        if (before + all < wanted) {  // everything stays
            cluster.sync();
            return floor;
        }
        if (own != 0 && running < wanted && running + own >= wanted) {
            for (uint32_t r = 0; r < blocks; ++r) {
                SampleShared *other = cluster.map_shared_rank(&sh, r);
                other->low_bin = bin;
                other->found_count = number;
                other->found_before = running;
            }
        }
        cluster.sync();
        const uint32_t border = sh.low_bin, border_count = sh.found_count;
        before = sh.found_before;
        if (border_count <= kListed) {
            // gather the bin in the first block and rank it there
            gather<false>(cluster, sh, slice, -INFINITY, [&](float x, uint32_t i) {
                const uint64_t c = composite(x, slice.begin + i);
                return in_span(c) && bin_of(x, c) == border;
            });
            if (rank == 0) {
                const uint32_t n = sh.listed;
                if (MASS) {
                    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) sh.sums[i] = weigh.of(logit_of(sh.list[i]));
                    __syncthreads();
                }
                for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
                    const uint64_t c = sh.list[i];
                    uint64_t above = before;
                    for (uint32_t j = 0; j < n; ++j) {
                        if (sh.list[j] > c) above += MASS ? sh.sums[j] : 1u;
                    }
                    const uint64_t mine = MASS ? sh.sums[i] : 1u;
                    if (above < wanted && above + mine >= wanted) {
                        for (uint32_t r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->cut = c;
                    }
                }
            }
            cluster.sync();
            return sh.cut;
        }
        // too many for that: what span do they cover?
        uint64_t c_low = ~0ull, c_high = 0;
        slice.each([&](float x, uint32_t i) {
            const uint64_t c = composite(x, slice.begin + i);
            if (!in_span(c) || bin_of(x, c) != border) return;
            c_low = c < c_low ? c : c_low;
            c_high = c > c_high ? c : c_high;
        });
        c_low = ~block_max(~c_low, sh.warp_values);
        c_high = block_max(c_high, sh.warp_values);
        if (threadIdx.x < blocks) {
            SampleShared *other = cluster.map_shared_rank(&sh, threadIdx.x);
            other->span_low[rank] = c_low;
            other->span_high[rank] = c_high;
        }
        cluster.sync();
        span_low = ~0ull;
        span_high = 0;
        for (uint32_t r = 0; r < blocks; ++r) {
            span_low = sh.span_low[r] < span_low ? sh.span_low[r] : span_low;
            span_high = sh.span_high[r] > span_high ? sh.span_high[r] : span_high;
        }
        by_distance = false;
        const uint32_t bits = 64 - __clzll((long long)(span_high - span_low)), room = 31 - __clz(bins);
        shift = bits > room ? bits - room : 0;  // bins 0 .. (span >> shift) < bins
    }
}

// Largest first (or smallest, for UP), over the next power of two of n; the caller has filled the rest with the least.
template <bool UP, typename V>
__device__ void block_sort(V *values, uint32_t n) {
    uint32_t size = 32;
    while (size < n) size *= 2;
    for (uint32_t k = 2; k <= size; k *= 2) {
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            for (uint32_t pair = threadIdx.x; pair < size / 2; pair += blockDim.x) {
                const uint32_t i = 2 * pair - (pair & (j - 1)), other = i + j;
                const V x = values[i], y = values[other];
                if ((x > y) == (((i & k) == 0) != UP ? false : true)) {
                    values[i] = y;
                    values[other] = x;
                }
            }
            __syncthreads();
        }
    }
}

// The same for at most an element per thread, which gets the one of its place: by exchanges within the warps as far as
// those reach.  `size` is the power of two that values[0, size) is filled to.
__device__ inline uint64_t thread_sort(uint64_t *values, uint32_t size) {
    const uint32_t i = threadIdx.x;
    uint64_t own = i < size ? values[i] : 0;
#pragma unroll 1
    for (uint32_t k = 2; k <= size; k *= 2) {
#pragma unroll 1
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            uint64_t other;
            if (j >= 32) {
                __syncthreads();
                values[i] = own;
                __syncthreads();
                other = values[i ^ j];
            } else {
                other = __shfl_xor_sync(0xffffffffu, own, j);
            }
            const bool larger = ((i & j) == 0) == ((i & k) == 0);
            own = (own > other) == larger ? own : other;
        }
    }
    return own;
}

__device__ inline uint64_t target_of(float uniform, uint64_t total) {
    const double aim = uniform > 0.0f ? floor((double)uniform * (double)total) : 0.0;
    const uint64_t target = aim < (double)total ? (uint64_t)aim : total - 1;
    return target < total ? target : total - 1;
}

// All that matter are in this block's list: cut them, draw, and answer.  `mass` is the sum that top-p is a share of, or 0
// where it is the sum of the first k.
__device__ __noinline__ void finish_list(const SampleArgs &p, uint32_t row, SampleShared &sh, const Weigh &weigh, uint32_t k,
                                         float share, uint64_t mass, uint64_t least, float uniform) {
    const uint32_t n = sh.listed;
    uint32_t size = 32;
    while (size < n) size *= 2;
    for (uint32_t i = n + threadIdx.x; i < size; i += blockDim.x) sh.list[i] = 0;
    __syncthreads();
    if (n > blockDim.x) block_sort<false>(sh.list, n);
    const uint32_t first = k != 0 && k < n ? k : n;
    if (n <= blockDim.x) {
        const uint32_t i = threadIdx.x;
        const uint64_t own = thread_sort(sh.list, size);
        const uint64_t weight = i < n ? weigh.of(logit_of(own)) : 0;
        uint64_t above;
        const uint64_t sum_first = block_scan(i < first ? weight : 0, sh.warp_values, above);
        bool stays = i < first && weight >= least;
        if (share < 1.0f) stays = stays && above < reach_of(share, mass != 0 ? mass : sum_first);
        const uint64_t total = block_sum(stays ? weight : 0, sh.warp_values);
        const uint32_t m = (uint32_t)__syncthreads_count(stays);  // a prefix
        const uint32_t index = index_of(own);
        if (i < m) {
            sh.sums[i] = weight;
            sh.count[i] = index;
        }
        __syncthreads();
        if (!stays) return;
        uint64_t running = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < m; ++j)
            if (sh.count[j] < index) running += sh.sums[j];
        const uint64_t target = target_of(uniform, total);
        if (running <= target && running + weight > target) {
            p.tokens[row] = index;
            if (p.probabilities != nullptr) p.probabilities[row] = (float)((double)weight / (double)total);
        }
        return;
    }
    // in order: running weights, each thread a run of neighbours
    const uint32_t each = kListed / blockDim.x, i0 = threadIdx.x * each;
    uint64_t sum = 0, running;
    for (uint32_t i = i0; i < min(n, i0 + each); ++i) sum += weigh.of(logit_of(sh.list[i]));
    block_scan(sum, sh.warp_values, running);
    for (uint32_t i = i0; i < min(n, i0 + each); ++i) {
        running += weigh.of(logit_of(sh.list[i]));
        sh.sums[i] = running;
    }
    __syncthreads();
    auto weight_of = [&](uint32_t i) { return sh.sums[i] - (i > 0 ? sh.sums[i - 1] : 0); };
    const uint64_t wanted = share < 1.0f ? reach_of(share, mass != 0 ? mass : sh.sums[first - 1]) : ~0ull;
    uint32_t stay = 0;  // how many stay: a prefix
    for (uint32_t i = i0; i < min(first, i0 + each); ++i) {
        if (sh.sums[i] - weight_of(i) < wanted && weight_of(i) >= least) ++stay;
    }
    const uint32_t m = (uint32_t)block_sum(stay, sh.warp_values);
    const uint64_t total = sh.sums[m - 1];
    // by index: (index, place in the order) as one number
    uint32_t *const by_index = sh.count;
    size = 32;
    while (size < m) size *= 2;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x)
        by_index[i] = i < m ? index_of(sh.list[i]) << 11 | i : 0xffffffffu;
    __syncthreads();
    block_sort<true>(by_index, m);
    sum = 0;
    for (uint32_t i = i0; i < min(m, i0 + each); ++i) sum += weight_of(by_index[i] & (kListed - 1));
    block_scan(sum, sh.warp_values, running);
    const uint64_t target = target_of(uniform, total);
    for (uint32_t i = i0; i < min(m, i0 + each); ++i) {
        const uint32_t place = by_index[i] & (kListed - 1);
        const uint64_t weight = weight_of(place);
        if (running <= target && running + weight > target) {
            p.tokens[row] = index_of(sh.list[place]);
            if (p.probabilities != nullptr) p.probabilities[row] = (float)((double)weight / (double)total);
        }
        running += weight;
    }
}

template <typename T, bool ON_CHIP, int THREADS>
__global__ void __launch_bounds__(THREADS, ON_CHIP ? 1 : 1024 / THREADS)
sample_kernel(const __grid_constant__ SampleArgs p, uint32_t slice_size) {
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint8_t sample_smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(sample_smem);
    uint64_t *const tiles = reinterpret_cast<uint64_t *>(sample_smem + sizeof(SampleShared));
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    // asked for first, needed late
    const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.0f;
    const uint32_t asked_k = p.top_k != nullptr ? p.top_k[row] : 0;
    const float share = p.top_p != nullptr ? p.top_p[row] : 1.0f;
    const float floor_p = p.min_p != nullptr ? p.min_p[row] : 0.0f;
    const float uniform = p.uniform[row];

    Slice<T> slice;
    slice.begin = min(rank * slice_size, p.vocab);
    slice.size = min(slice_size, p.vocab - slice.begin);
    slice.data = static_cast<const T *>(p.logits) + (size_t)row * p.ld + slice.begin;
    const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(slice.data) & 15u);
    slice.split(skew);
    cg::cluster_group::arrival_token running_token = cluster.barrier_arrive();

    // ---- load: extremes on the way ----
    float high = -INFINITY, low = INFINITY;  // first of what this thread reads
    const bool binned = asked_k != 0 || share < 1.0f;  // the smallest only spaces the bins
    auto look = [&](float x, uint32_t) {
        high = fmaxf(high, x);
        if (binned && x > -INFINITY) low = fminf(low, x);
    };
    {
        // the copy starts at the same place within 16 bytes as the original, so whole words move
        uint8_t *held = reinterpret_cast<uint8_t *>(tiles + slice.tiles() + 2);
        held += ((16u - (uint32_t)(reinterpret_cast<uintptr_t>(held) & 15u)) & 15u) + skew;
        T *const copy = reinterpret_cast<T *>(held);
        const uint4 *const from = reinterpret_cast<const uint4 *>(slice.data + slice.head);
        uint4 *const to = reinterpret_cast<uint4 *>(copy + slice.head);
        constexpr uint32_t kAtOnce = ON_CHIP ? 8 : 6;  // words on their way per thread
#pragma unroll 1
        for (uint32_t w0 = threadIdx.x; w0 < slice.words; w0 += kAtOnce * blockDim.x) {
            uint4 word[kAtOnce];
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u)
                if (w0 + u * blockDim.x < slice.words) word[u] = ON_CHIP ? __ldcs(from + w0 + u * blockDim.x) : from[w0 + u * blockDim.x];
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u) {
                if (w0 + u * blockDim.x < slice.words) {
                    if (ON_CHIP) to[w0 + u * blockDim.x] = word[u];
                    const T *x = reinterpret_cast<const T *>(&word[u]);
#pragma unroll
                    for (uint32_t j = 0; j < Slice<T>::kWord; ++j) look(as_float(x[j]), 0);
                }
            }
        }
        if (threadIdx.x < slice.head + slice.tail) {
            const uint32_t i = threadIdx.x < slice.head ? threadIdx.x : slice.size - slice.tail + threadIdx.x - slice.head;
            if (ON_CHIP) copy[i] = slice.data[i];
            look(slice.at(i), 0);
        }
        if (ON_CHIP) slice.data = copy;
    }
    const float own_high = high;
    for (uint32_t j = threadIdx.x; j < 256; j += blockDim.x) sh.power[j] = kPowers.entry[j];
    for (uint32_t b = threadIdx.x; b < kBins; b += blockDim.x) sh.count[b] = 0;
    if (threadIdx.x == 0) {
        sh.listed = 0;
        sh.first = 0xffffffffu;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
    }
    if (lane == 0) {
        sh.warp_high[warp] = high;
        sh.warp_low[warp] = low;
    }
    __syncthreads();
    cluster.barrier_wait(static_cast<cg::cluster_group::arrival_token &&>(running_token));  // every block of the cluster runs
    if (warp == 0) {
        high = lane < blockDim.x / 32 ? sh.warp_high[lane] : -INFINITY;
        low = lane < blockDim.x / 32 ? sh.warp_low[lane] : INFINITY;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
        }
        if (lane < blocks) {
            SampleShared *other = cluster.map_shared_rank(&sh, lane);
            other->high[rank] = high;
            other->low[rank] = low;
        }
    }
    cluster.sync();
    high = sh.high[0];
    low = sh.low[0];
    for (uint32_t r = 1; r < blocks; ++r) {
        high = fmaxf(high, sh.high[r]);
        low = fminf(low, sh.low[r]);
    }
    if (high == -INFINITY) {
        if (rank == 0 && threadIdx.x == 0) {
            p.tokens[row] = 0xffffffffu;
            if (p.probabilities != nullptr) p.probabilities[row] = 0.0f;
        }
        return;
    }
    if (!(temperature > 0.0f)) {
        uint32_t first = 0xffffffffu;
        slice.each([&](float x, uint32_t i) {
            if (x == high) first = min(first, slice.begin + i);
        });
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0 && first != 0xffffffffu) atomicMin(&cluster.map_shared_rank(&sh, 0)->first, first);
        cluster.sync();
        if (rank == 0 && threadIdx.x == 0) {
            p.tokens[row] = sh.first;
            if (p.probabilities != nullptr) p.probabilities[row] = 1.0f;
        }
        return;
    }
    Weigh weigh;
    weigh.power = sh.power;
    weigh.set(high, temperature);
    const uint32_t bins = min(kBins, blocks * blockDim.x);
    const float last_bin = (float)(bins - 1), to_bin = last_bin / fmaxf(high - low, 1e-30f);
    const uint32_t k = asked_k < p.vocab ? asked_k : 0;
    // the least weight that stays, in units (a NaN is none)
    const uint64_t least = floor_p > 0.0f ? (uint64_t)ceil((double)fminf(floor_p, 1.0f) * (double)kOne) : 0;

    // less than every value whose place is below `end`: the place's roundings and the value's own are 2^-22 of them
    auto value_below = [&](float end) {
        if (end > last_bin) return -INFINITY;
        if (high == INFINITY) return high;
        return high - end / to_bin * 1.000001f - fabsf(high) * 1e-6f;
    };

    uint64_t cut = 0;
    // Collecting pays while a third of the row or less is collected; at a half it takes longer than not asking.
    bool sparse = false;
    if (k != 0 && k <= kListed / 2) {
        // ---- few by count ----
        // The k-th largest of the threads' own maxima is at most the k-th largest of all, and hardly smaller while k is a
        // fraction of the threads: bins of one element per thread tell how far down the list has to go.
        if (own_high > -INFINITY) atomicAdd(&sh.count[whole(place_of(own_high, high, to_bin, last_bin))], 1u);
        if (threadIdx.x == 0) sh.found_count = 0;
        cluster.sync();
        const uint32_t bin = my_bin(cluster, bins), number = count_of(cluster, sh, bin);
        uint64_t before = tell_parts(cluster, sh, 0, number), all;
        cluster.sync();  // the bins have been read everywhere
        before += sum_parts(cluster, sh, 0, all);
        if (number != 0 && before < k && before + number >= k) {
            for (uint32_t r = 0; r < blocks; ++r) {
                SampleShared *other = cluster.map_shared_rank(&sh, r);
                other->high_bin = bin;
                other->found_count = 1;
            }
        }
        cluster.sync();
        if (sh.found_count != 0) {  // fewer threads than k otherwise
            const float end = (float)(sh.high_bin + 1);
            if (gather<false>(cluster, sh, slice, value_below(end),
                              [&](float x, uint32_t) { return place_of(x, high, to_bin, last_bin) < end; }) <= kListed) {
                if (rank == 0) finish_list(p, row, sh, weigh, k, share, 0, least, uniform);
                return;
            }
        }
        for (uint32_t b = threadIdx.x; b < bins; b += blockDim.x) sh.count[b] = 0;
        __syncthreads();
    }
    if (k != 0 || share < 1.0f) {
        // ---- counts ----
        const bool add = k == 0;  // top-p alone is a share of everything
        uint64_t mine = 0;
        auto count = [&](float x) { atomicAdd(&sh.count[whole(place_of(x, high, to_bin, last_bin))], 1u); };
        if (add) {
            slice.each([&](float x, uint32_t) {
                count(x);
                mine += weigh.of(x);
            });
            mine = block_sum(mine, sh.warp_values);
            if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->total[rank] = mine;
        } else {
            slice.each([&](float x, uint32_t) { count(x); });
        }
        if (threadIdx.x == 0) {
            sh.low_bin = sh.high_bin = bins - 1;
            sh.found_count = sh.fine_count = 0;  // elements down to the end of the bracket, or in its bin; 0: nobody found it
        }
        cluster.sync();
        uint64_t everything = 0, wanted = k;
        if (add) {
            for (uint32_t r = 0; r < blocks; ++r) everything += sh.total[r];
            wanted = reach_of(share, everything);
        }
        // By weight a bin of n elements holds between n times the weight at its far edge and n times that at its near one
        // (the edges moved out by the rounding of a place: two units in the last of 2048).  [low_bin, high_bin] is where
        // the border may lie; by count both are its bin.
        const uint32_t bin = my_bin(cluster, bins), number = count_of(cluster, sh, bin);
        uint64_t far = number, near = number;
        if (add) {
            const float b = (float)bin, width = 1.0f / to_bin;
            uint64_t least_of = b < last_bin ? weigh.at((b + 1.001f) * width, 0.0f) : 0;
            least_of -= least_of > 0 ? (least_of >> 28) + 1 : 0;  // and by a weight's own error
            uint64_t most_of = b > 0.0f ? weigh.at((b - 0.001f) * width, 0.0f) : kOne;
            far = number * least_of;
            near = number * (most_of + (most_of >> 28) + 1);
        }
        uint64_t far_before = tell_parts(cluster, sh, 0, far), near_before = 0, number_before = 0, all_of;
        if (add) {
            near_before = tell_parts(cluster, sh, 1, near);
            number_before = tell_parts(cluster, sh, 2, number);
        }
        cluster.sync();  // the bins have been read everywhere
        far_before += sum_parts(cluster, sh, 0, all_of);
        if (add) {
            near_before += sum_parts(cluster, sh, 1, all_of);
            number_before += sum_parts(cluster, sh, 2, all_of);
        } else {
            near_before = number_before = far_before;
        }
        const bool is_low = near_before < wanted && near_before + near >= wanted;
        const bool is_high = far_before < wanted && far_before + far >= wanted;
        if (number != 0 && (is_low || is_high)) {
            for (uint32_t r = 0; r < blocks; ++r) {
                SampleShared *other = cluster.map_shared_rank(&sh, r);
                if (is_low) {
                    other->low_bin = bin;
                    other->low_before = (uint32_t)number_before;
                }
                if (is_high) {
                    other->high_bin = bin;
                    other->found_count = (uint32_t)number_before + number;
                }
            }
        }
        cluster.sync();
        const uint32_t low_bin = sh.low_bin, high_bin = sh.high_bin, down_to = sh.found_count, low_before = sh.low_before;
        sparse = down_to != 0 && down_to <= p.vocab / 3;
        if (down_to != 0 && down_to <= kListed) {
            // ---- few stay ----
            const float end = (float)(high_bin + 1);
            gather<false>(cluster, sh, slice, value_below(end),
                          [&](float x, uint32_t) { return place_of(x, high, to_bin, last_bin) < end; });
            if (rank == 0) finish_list(p, row, sh, weigh, k, share, everything, least, uniform);
            return;
        }
        // the first block puts its list in order and finds where the running weight reaches `wanted`
        auto rank_list = [&](uint64_t before) {
            if (rank == 0) {
                const uint32_t n = sh.listed;
                uint32_t size = 32;
                while (size < n) size *= 2;
                for (uint32_t i = n + threadIdx.x; i < size; i += blockDim.x) sh.list[i] = 0;
                __syncthreads();
                if (n <= blockDim.x) {
                    const uint64_t own = thread_sort(sh.list, size);
                    __syncthreads();
                    sh.list[threadIdx.x] = own;
                    __syncthreads();
                } else {
                    block_sort<false>(sh.list, n);
                }
                const uint32_t each = n <= blockDim.x ? 1 : kListed / blockDim.x, i0 = threadIdx.x * each;
                uint64_t sum = 0, running;
                for (uint32_t i = i0; i < min(n, i0 + each); ++i) sum += weigh.of(logit_of(sh.list[i]));
                block_scan(sum, sh.warp_values, running);
                running += before;
                for (uint32_t i = i0; i < min(n, i0 + each); ++i) {
                    const uint64_t w = weigh.of(logit_of(sh.list[i]));
                    if (running < wanted && running + w >= wanted) {
                        for (uint32_t r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->cut = sh.list[i];
                    }
                    running += w;
                }
            }
            cluster.sync();
            return sh.cut;
        };
        if (add && down_to != 0 && down_to - low_before <= kListed) {
            // ---- many stay, few lie in the bracket: those are put in order ----
            const float first = (float)low_bin, end = (float)(high_bin + 1);
            uint64_t above = 0, all_above;
            gather<true>(cluster, sh, slice, value_below(end), [&](float x, uint32_t) {
                const float v = place_of(x, high, to_bin, last_bin);
                if (v < first) above += weigh.of(x);
                return v >= first && v < end;
            });
            tell_parts(cluster, sh, 1, above);
            cluster.sync();
            sum_parts(cluster, sh, 1, all_above);
            cut = rank_list(all_above);
        } else if (add) {
            // ---- many stay: the bracket by exact weights ----
            for (uint32_t b = threadIdx.x; b < bins; b += blockDim.x) {
                sh.count[b] = 0;
                sh.mass[b] = 0;
            }
            __syncthreads();
            const float first = (float)low_bin, end = (float)(high_bin + 1), finer = (float)bins / (end - first);
            uint64_t above = 0;
            auto fine_bin = [&](float v) { return whole(fminf((v - first) * finer, last_bin)); };
            auto add_fine = [&](float x, uint32_t) {
                const float v = place_of(x, high, to_bin, last_bin);
                if (v >= end) return;
                const uint64_t w = weigh.of(x);
                if (v < first) {
                    above += w;
                } else {
                    const uint32_t b = fine_bin(v);
                    atomicAdd(&sh.count[b], 1u);
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)w);
                }
            };
            if (sparse) slice.each_above(value_below(end), sh.queue[warp], add_fine);
            else slice.each(add_fine);
            tell_parts(cluster, sh, 1, above);
            cluster.sync();
            const uint32_t fine_number = count_of(cluster, sh, bin);
            const uint64_t own = mass_of(cluster, sh, bin);
            uint64_t running = tell_parts(cluster, sh, 0, own), all_above;
            sum_parts(cluster, sh, 1, all_above);
            cluster.sync();  // the bins have been read everywhere: the list may take their place
            running += all_above + sum_parts(cluster, sh, 0, all_of);
            if (own != 0 && running < wanted && running + own >= wanted) {
                for (uint32_t r = 0; r < blocks; ++r) {
                    SampleShared *other = cluster.map_shared_rank(&sh, r);
                    other->fine_bin = bin;
                    other->fine_count = fine_number;
                    other->found_before = running;
                }
            }
            cluster.sync();
            const uint32_t border = sh.fine_bin, border_count = sh.fine_count;
            const uint64_t before = sh.found_before;
            if (border_count != 0 && border_count <= kListed) {
                gather<false>(cluster, sh, slice, value_below(end), [&](float x, uint32_t) {
                    const float v = place_of(x, high, to_bin, last_bin);
                    return v >= first && v < end && fine_bin(v) == border;
                });
                cut = rank_list(before);
            } else {
                cut = find_cut<true>(cluster, sh, slice, weigh, high, to_bin, bins, 0ull, wanted);
            }
        } else {
            cut = find_cut<false>(cluster, sh, slice, weigh, high, to_bin, bins, 0ull, wanted);
            if (share < 1.0f) {
                mine = 0;
                slice.each([&](float x, uint32_t i) {
                    if (composite(x, slice.begin + i) >= cut) mine += weigh.of(x);
                });
                mine = block_sum(mine, sh.warp_values);
                if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->total[rank] = mine;
                cluster.sync();
                for (uint32_t r = 0; r < blocks; ++r) everything += sh.total[r];
                cut = find_cut<true>(cluster, sh, slice, weigh, high, to_bin, bins, cut, reach_of(share, everything));
            }
        }
    }

    // ---- the token: sums per tile (the head is one of its own in front, the tail one behind) ----
    const bool all = cut == 0;
    const float cut_logit = all ? -INFINITY : logit_of(cut);
    auto kept = [&](float x, uint32_t i) -> uint64_t {
        if (!all && composite(x, slice.begin + i) < cut) return 0;
        const uint64_t w = weigh.of(x);
        return least != 0 && w < least ? 0ull : w;
    };
    const uint32_t word_tiles = slice.tiles(), tile_count = word_tiles + 2;
    for (uint32_t t = warp; t < tile_count; t += (blockDim.x / 32)) {
        uint64_t sum = 0;
        if (t == 0) {
            if (lane < slice.head) sum = kept(slice.at(lane), lane);
        } else if (t == tile_count - 1) {
            if (lane < slice.tail) sum = kept(slice.at(slice.size - slice.tail + lane), slice.size - slice.tail + lane);
        } else {
            if (all && least == 0) slice.tile(t - 1, [&](float x, uint32_t) { sum += weigh.of(x); });
            else if (all || !sparse) slice.tile(t - 1, [&](float x, uint32_t i) { sum += kept(x, i); });
            else slice.tile_above(t - 1, cut_logit, sh.queue[warp], [&](float x, uint32_t i) { sum += kept(x, i); });
        }
        sum = warp_sum(sum);
        if (lane == 0) tiles[t] = sum;
    }
    __syncthreads();
    uint64_t mine = 0;
    for (uint32_t t = threadIdx.x; t < tile_count; t += blockDim.x) mine += tiles[t];
    mine = block_sum(mine, sh.warp_values);
    // (the sums of the top-p passes have been read everywhere: a cluster barrier lies between)
    if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->total[rank] = mine;
    cluster.sync();  // the last look into another block's shared memory is behind this
    uint64_t total = 0, before = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
        if (r < rank) before += sh.total[r];
        total += sh.total[r];
    }
    const uint64_t target = target_of(uniform, total);
    if (target < before || target >= before + mine || warp != 0) return;
    // the tile, 32 at a time
    uint64_t running = before;
    uint32_t tile = 0;
    for (uint32_t t0 = 0; t0 < tile_count; t0 += 32) {
        const uint64_t own = t0 + lane < tile_count ? tiles[t0 + lane] : 0;
        const uint64_t inclusive = warp_inclusive(own);
        const uint32_t passed = __ballot_sync(0xffffffffu, running + inclusive > target);
        if (passed != 0) {
            const int first = __ffs(passed) - 1;
            tile = t0 + first;
            running += __shfl_sync(0xffffffffu, inclusive - own, first);
            break;
        }
        running += __shfl_sync(0xffffffffu, inclusive, 31);
    }
    // within it: rows of 32 words, a word per lane (or single values)
    const bool single = tile == 0 || tile == tile_count - 1;
    const uint32_t first = tile == 0 ? 0 : single ? slice.size - slice.tail : slice.head + (tile - 1) * kTileWords * Slice<T>::kWord;
    const uint32_t values = single ? 1 : Slice<T>::kWord, end = tile == 0 ? slice.head : single ? slice.size : slice.head + slice.words * Slice<T>::kWord;
    for (uint32_t r = 0; r < (single ? 1u : kTileRows4); ++r) {
        const uint32_t at = first + (r * 32 + lane) * values;
        uint64_t own[Slice<T>::kWord], sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < Slice<T>::kWord; ++j) {
            own[j] = j < values && at + j < end ? kept(slice.at(at + j), at + j) : 0;
            sum += own[j];
        }
        const uint64_t inclusive = warp_inclusive(sum);
        uint64_t here = running + inclusive - sum;
        if (here <= target && here + sum > target) {
#pragma unroll
            for (uint32_t j = 0; j < Slice<T>::kWord; ++j) {
                if (here <= target && here + own[j] > target) {
                    p.tokens[row] = slice.begin + at + j;
                    if (p.probabilities != nullptr) p.probabilities[row] = (float)((double)own[j] / (double)total);
                }
                here += own[j];
            }
        }
        running += __shfl_sync(0xffffffffu, inclusive, 31);
    }
}

template <typename T, bool ON_CHIP, int THREADS>
cudaError_t launch_sample_as(const SampleArgs &args, uint32_t blocks, uint32_t slice, size_t smem, cudaStream_t stream) {
    static bool configured[kMaxDevices] = {};
    const int slot = device_slot();
    if (slot < 0 || !configured[slot]) {
        const size_t most = sizeof(SampleShared) + ((1u << 20) / kMostBlocks * 4 / 16 / kTileWords + 3) * 8 + (ON_CHIP ? kSliceBytes : 0);
        cudaError_t status = cudaFuncSetAttribute(sample_kernel<T, ON_CHIP, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (status != cudaSuccess) return status;
        if (slot >= 0) configured[slot] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(args.rows * blocks);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = blocks;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, sample_kernel<T, ON_CHIP, THREADS>, args, slice);
}

template <typename T>
cudaError_t launch_sample_of(const SampleArgs &args, int sm_count, cudaStream_t stream) {
    // blocks per row: at least 4096 logits each, 8 at most
    uint32_t blocks = 1;
    while (blocks < kMostBlocks && args.vocab / (2 * blocks) >= 4096) blocks *= 2;
    const uint32_t slice = ceil_div(args.vocab, blocks);
    const size_t slice_bytes = (size_t)slice * sizeof(T) + 64;
    const size_t smem = sizeof(SampleShared) + ((size_t)slice * sizeof(T) / 16 / kTileWords + 3) * 8;
    if (slice_bytes <= kSliceBytes && (uint64_t)args.rows * blocks <= (uint64_t)sm_count)
        return launch_sample_as<T, true, 512>(args, blocks, slice, smem + slice_bytes, stream);
    // Two blocks of 512 threads per SM, or four of 256 whose short phases fill each other's waits: better for a whole
    // distribution in more than one wave (256 fp32 rows of 248,320: 196 us against 224 us), worse for the longer chain
    // of a top-p cut (64 fp16 rows: 195 us against 177 us).
    if (args.top_k == nullptr && args.top_p == nullptr && (uint64_t)args.rows * blocks > 2 * (uint64_t)sm_count)
        return launch_sample_as<T, false, 256>(args, blocks, slice, smem, stream);
    return launch_sample_as<T, false, 512>(args, blocks, slice, smem, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &args, int sm_count, cudaStream_t stream) {
    if (args.dtype == kF32) return launch_sample_of<float>(args, sm_count, stream);
    if (args.dtype == kBF16) return launch_sample_of<__nv_bfloat16>(args, sm_count, stream);
    return launch_sample_of<__half>(args, sm_count, stream);
}

}  // namespace q4b
