// One token per row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// All three cuts keep a prefix of the order (largest logit first, the lowest index first among equals), so each is ONE
// composite number c = (ordered bits of the logit, complement of the index): an element stays when its own composite is
// at least the cut.  The token is then the first index at which the running sum of the kept weights
// exp((logit - largest) / temperature) passes uniform x total.  No sort is needed.
//
// A row is spread over a cluster of 1 to 8 thread blocks that keep it in shared memory: it is read from HBM once,
// every further pass runs on chip.
//   load      the largest composite (greedy ends here) and the smallest finite logit
//   top-k     counts in 2048 bins, linear in the distance to the largest logit (linear bins spread a row of logits
//             evenly; bins of the float's own bits would put most of a row into a few and serialise the atomics); the
//             bin that holds the k-th element is gathered and ranked.  A bin too full for that is cut into 2048 again,
//             by composite, which differ in all elements, so equal logits end too
//   top-p     the same with weights in the bins
//   token     sums of kept weights per 256 indices, then within the 256 that the target falls into
// Weights are 64-bit integers in units of 2^-42 of the largest one's: sums are exact, in any order of the atomics, so
// equal inputs give equal tokens.  exp is taken in fp64: in fp32 the argument alone is off by 2^-24 x |logit - largest|,
// and over a flat distribution of 250,000 tokens such errors move the border between neighbours visibly.
#include "q4b_kernels.h"

#include <cooperative_groups.h>
#include <cmath>

namespace q4b {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kSampleThreads = 1024;
constexpr uint32_t kSampleWarps = kSampleThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMostBlocks = 8;        // thread blocks of a row
constexpr uint32_t kListed = 1024;         // elements of a bin that are ranked one against another
constexpr uint32_t kTile = 256;            // indices per partial sum of the last pass
constexpr uint32_t kSliceBytes = 160 * 1024;  // of a row that a thread block keeps in shared memory; longer ones are read again
constexpr uint32_t kMostTiles = (1u << 20) / kTile;
constexpr double kUnit = 4398046511104.0;  // 2^42

struct SampleShared {
    uint64_t high[kMostBlocks];          // largest composite of every block's slice
    float low[kMostBlocks];              // smallest finite logit
    uint64_t part_count[kMostBlocks], part_mass[kMostBlocks];  // of every 256 bins, over the whole row
    uint64_t before_count, before_mass;  // in front of the border bin
    uint32_t border, border_count;
    uint64_t span_low[kMostBlocks], span_high[kMostBlocks];    // composites of the border bin
    uint64_t cut;
    uint64_t total[kMostBlocks];
    uint64_t warp_values[kSampleWarps];
    float warp_low[kSampleWarps];
    uint32_t listed;
    uint64_t list[kListed];
    uint64_t list_weight[kListed];
    uint32_t count[kBins];
    uint64_t mass[kBins];
};

__device__ inline float as_float(float x) { return x; }
__device__ inline float as_float(__half x) { return __half2float(x); }
__device__ inline float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// NaN counts as -infinity, both zeros are one number
__device__ inline float tidy(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ inline uint64_t composite(float x, uint32_t index) {
    const uint32_t bits = __float_as_uint(x);
    const uint32_t ordered = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (uint64_t)ordered << 32 | (uint32_t)~index;
}
__device__ inline float logit_of(uint64_t c) {
    const uint32_t ordered = (uint32_t)(c >> 32);
    return __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
}
__device__ inline uint32_t index_of(uint64_t c) { return ~(uint32_t)c; }

template <typename V> __device__ inline V warp_sum(V x) {
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
// the same in every thread of the block; `scratch` is free again afterwards
__device__ inline uint64_t block_max(uint64_t x, uint64_t *scratch) {
    x = warp_max(x);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = warp_max(scratch[threadIdx.x & 31]);
    __syncthreads();
    return x;
}
__device__ inline uint64_t block_sum(uint64_t x, uint64_t *scratch) {
    x = warp_sum(x);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = warp_sum(scratch[threadIdx.x & 31]);
    __syncthreads();
    return x;
}
__device__ inline float block_min(float x, float *scratch) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fminf(x, __shfl_xor_sync(0xffffffffu, x, d));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = scratch[threadIdx.x & 31];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fminf(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();
    return x;
}

template <typename T>
struct Slice {
    const T *data;       // this block's part of the row, in shared memory or where it was
    uint32_t begin, size;
    __device__ inline float at(uint32_t i) const { return tidy(as_float(data[i])); }
};

struct Weigh {
    float high;
    double over;  // 1 / temperature
    __device__ inline double real(float x) const {
        const double distance = (double)x - (double)high;
        if (x == high) return 1.0;
        return distance == -INFINITY ? 0.0 : exp(distance * over);
    }
    static __device__ inline uint64_t units(double w) { return (uint64_t)(w * kUnit + 0.5); }
};

// Where the border lies: the composite of the last element that stays, over the whole cluster.  By count: the
// `wanted`-th element of those at or above `floor`.  By mass: the first at which the running weight reaches `wanted`.
template <bool MASS, typename T>
__device__ uint64_t find_cut(cg::cluster_group &cluster, SampleShared &sh, const Slice<T> &slice, const Weigh &weigh,
                             float low, uint64_t floor, uint64_t wanted) {
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t per_block = kBins / blocks;
    bool by_distance = true;
    const float to_bin = (float)(kBins - 1) / fmaxf(weigh.high - low, 1e-30f);
    uint64_t span_low = floor, span_high = ~0ull;  // composites still in question, and how they are cut into bins
    uint32_t shift = 0;
    uint64_t before = 0;                           // count or mass above the span
    auto bin_of = [&](float x, uint64_t c) -> uint32_t {
        if (by_distance) return x == weigh.high ? 0u : (uint32_t)fminf((weigh.high - x) * to_bin, (float)(kBins - 1));
        return (uint32_t)((span_high - c) >> shift);
    };
    for (;;) {
        for (uint32_t b = threadIdx.x; b < kBins; b += kSampleThreads) {
            sh.count[b] = 0;
            if (MASS) sh.mass[b] = 0;
        }
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < slice.size; i += kSampleThreads) {
            const float x = slice.at(i);
            const uint64_t c = composite(x, slice.begin + i);
            if (c < span_low || c > span_high) continue;
            const uint32_t b = bin_of(x, c);
            atomicAdd(&sh.count[b], 1u);
            if (MASS) {
                const uint64_t w = Weigh::units(weigh.real(x));
                if (w != 0) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)w);
            }
        }
        cluster.sync();
        // every block adds up its share of the bins over the cluster, tells the others the sum, ...
        uint64_t my_count = 0, my_mass = 0;
        if (threadIdx.x < per_block) {
            const uint32_t b = rank * per_block + threadIdx.x;
            for (uint32_t r = 0; r < blocks; ++r) {
                const SampleShared *other = cluster.map_shared_rank(&sh, r);
                my_count += other->count[b];
                if (MASS) my_mass += other->mass[b];
            }
        }
        if (blocks == 1) {  // 2048 bins, 1024 threads: two neighbours each
            my_count = my_mass = 0;
        }
        const uint32_t bins_each = per_block > kSampleThreads ? per_block / kSampleThreads : 1;
        const uint32_t bin0 = rank * per_block + threadIdx.x * bins_each;
        uint64_t each_count[2] = {my_count, 0}, each_mass[2] = {my_mass, 0};
        if (bins_each == 2) {
            for (uint32_t e = 0; e < 2; ++e) {
                each_count[e] = sh.count[bin0 + e];
                if (MASS) each_mass[e] = sh.mass[bin0 + e];
            }
            my_count = each_count[0] + each_count[1];
            my_mass = each_mass[0] + each_mass[1];
        }
        const uint64_t sum_count = block_sum(my_count, sh.warp_values);
        const uint64_t sum_mass = MASS ? block_sum(my_mass, sh.warp_values) : 0;
        if (threadIdx.x < blocks) {
            SampleShared *other = cluster.map_shared_rank(&sh, threadIdx.x);
            other->part_count[rank] = sum_count;
            other->part_mass[rank] = sum_mass;
        }
        cluster.sync();
        // ... and the one whose share holds the border finds its bin
        uint64_t parts_before = before;
        for (uint32_t r = 0; r < rank; ++r) parts_before += MASS ? sh.part_mass[r] : sh.part_count[r];
        uint32_t owner = blocks;
        {
            uint64_t sum = before;
            for (uint32_t r = 0; r < blocks; ++r) {
                sum += MASS ? sh.part_mass[r] : sh.part_count[r];
                if (owner == blocks && sum >= wanted) owner = r;
            }
        }
        if (owner == blocks) {  // fewer than wanted: everything stays
            cluster.sync();
            return floor;
        }
        if (owner == rank) {
            // exclusive running value of this thread's bins
            uint64_t inclusive = MASS ? my_mass : my_count;
            const uint64_t own = inclusive;
            const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, inclusive, d);
                if (lane >= (uint32_t)d) inclusive += y;
            }
            if (lane == 31) sh.warp_values[warp] = inclusive;
            __syncthreads();
            uint64_t exclusive = parts_before + inclusive - own;
            for (uint32_t w = 0; w < warp; ++w) exclusive += sh.warp_values[w];
            for (uint32_t e = 0; e < bins_each; ++e) {
                const uint64_t value = MASS ? each_mass[e] : each_count[e];
                if (value != 0 && exclusive < wanted && exclusive + value >= wanted) {
                    for (uint32_t r = 0; r < blocks; ++r) {
                        SampleShared *other = cluster.map_shared_rank(&sh, r);
                        other->border = bin0 + e;
                        other->border_count = (uint32_t)each_count[e];
                        other->before_mass = exclusive;
                    }
                }
                exclusive += value;
            }
        }
        cluster.sync();
        const uint32_t border = sh.border, border_count = sh.border_count;
        before = sh.before_mass;
        if (border_count <= kListed) {
            // gather the bin in the first block and rank it
            SampleShared *leader = cluster.map_shared_rank(&sh, 0);
            for (uint32_t i = threadIdx.x; i < slice.size; i += kSampleThreads) {
                const float x = slice.at(i);
                const uint64_t c = composite(x, slice.begin + i);
                if (c < span_low || c > span_high || bin_of(x, c) != border) continue;
                leader->list[atomicAdd(&leader->listed, 1u)] = c;
            }
            cluster.sync();
            if (rank == 0) {
                const uint32_t n = sh.listed;
                if (MASS) {
                    for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads)
                        sh.list_weight[i] = Weigh::units(weigh.real(logit_of(sh.list[i])));
                    __syncthreads();
                }
                for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads) {
                    const uint64_t c = sh.list[i];
                    uint64_t above = before;
                    for (uint32_t j = 0; j < n; ++j) {
                        if (sh.list[j] > c) above += MASS ? sh.list_weight[j] : 1u;
                    }
                    const uint64_t own = MASS ? sh.list_weight[i] : 1u;
                    if (above < wanted && above + own >= wanted) {
                        for (uint32_t r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->cut = c;
                    }
                }
            }
            cluster.sync();
            return sh.cut;
        }
        // too many for that: what span do they cover?
        uint64_t c_low = ~0ull, c_high = 0;
        for (uint32_t i = threadIdx.x; i < slice.size; i += kSampleThreads) {
            const float x = slice.at(i);
            const uint64_t c = composite(x, slice.begin + i);
            if (c < span_low || c > span_high || bin_of(x, c) != border) continue;
            c_low = c < c_low ? c : c_low;
            c_high = c > c_high ? c : c_high;
        }
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
        const uint32_t bits = 64 - __clzll((long long)(span_high - span_low));
        shift = bits > 11 ? bits - 11 : 0;  // bins 0 .. (span >> shift) < 2048
    }
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 1)
sample_kernel(const __grid_constant__ SampleArgs p, uint32_t slice_size, uint32_t kept_on_chip) {
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint8_t sample_smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(sample_smem);
    uint64_t *const tiles = reinterpret_cast<uint64_t *>(sample_smem + sizeof(SampleShared));
    uint8_t *const held = reinterpret_cast<uint8_t *>(tiles + ceil_div(slice_size, kTile));
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    const T *const logits = static_cast<const T *>(p.logits) + (size_t)row * p.ld;
    Slice<T> slice;
    slice.begin = min(rank * slice_size, p.vocab);
    slice.size = min(slice_size, p.vocab - slice.begin);
    slice.data = logits + slice.begin;

    // ---- load ----
    uint64_t best = 0;
    float low = INFINITY;
    auto look = [&](float raw, uint32_t i) {
        const float x = tidy(raw);
        const uint64_t c = composite(x, slice.begin + i);
        best = c > best ? c : best;
        if (x > -INFINITY) low = fminf(low, x);
    };
    if (kept_on_chip) {
        // the copy starts at the same place within 16 bytes as the original, so whole 16-byte words move
        const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(slice.data) & 15u);
        uint8_t *const place = held + ((16u - (uint32_t)(reinterpret_cast<uintptr_t>(held) & 15u)) & 15u) + skew;
        T *const copy = reinterpret_cast<T *>(place);
        constexpr uint32_t kWord = 16 / sizeof(T);
        const uint32_t head = min(slice.size, skew == 0 ? 0u : (16u - skew) / (uint32_t)sizeof(T));
        const uint32_t words = (slice.size - head) / kWord, tail = head + words * kWord;
        if (threadIdx.x < head) {
            copy[threadIdx.x] = slice.data[threadIdx.x];
            look(as_float(slice.data[threadIdx.x]), threadIdx.x);
        }
        const uint4 *from = reinterpret_cast<const uint4 *>(slice.data + head);
        uint4 *to = reinterpret_cast<uint4 *>(copy + head);
#pragma unroll 4
        for (uint32_t w = threadIdx.x; w < words; w += kSampleThreads) {
            const uint4 word = __ldcs(from + w);
            to[w] = word;
            const T *x = reinterpret_cast<const T *>(&word);
#pragma unroll
            for (uint32_t j = 0; j < kWord; ++j) look(as_float(x[j]), head + w * kWord + j);
        }
        if (tail + threadIdx.x < slice.size) {
            copy[tail + threadIdx.x] = slice.data[tail + threadIdx.x];
            look(as_float(slice.data[tail + threadIdx.x]), tail + threadIdx.x);
        }
        slice.data = copy;
    } else {
        for (uint32_t i = threadIdx.x; i < slice.size; i += kSampleThreads) look(as_float(slice.data[i]), i);
    }
    best = block_max(best, sh.warp_values);
    low = block_min(low, sh.warp_low);
    cluster.sync();  // every block of the cluster runs: its shared memory may be written
    if (threadIdx.x < blocks) {
        SampleShared *other = cluster.map_shared_rank(&sh, threadIdx.x);
        other->high[rank] = best;
        other->low[rank] = low;
    }
    cluster.sync();
    for (uint32_t r = 0; r < blocks; ++r) {
        best = sh.high[r] > best ? sh.high[r] : best;
        low = fminf(low, sh.low[r]);
    }
    Weigh weigh;
    weigh.high = logit_of(best);
    const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.0f;
    if (weigh.high == -INFINITY || !(temperature > 0.0f)) {
        if (rank == 0 && threadIdx.x == 0) {
            const bool none = weigh.high == -INFINITY;
            p.tokens[row] = none ? 0xffffffffu : index_of(best);
            if (p.probabilities != nullptr) p.probabilities[row] = none ? 0.0f : 1.0f;
        }
        return;  // the same decision in every block of the cluster, and nobody's shared memory is read any more
    }
    weigh.over = 1.0 / (double)temperature;

    // ---- the cuts ----
    uint64_t cut = 0;
    const uint32_t k = p.top_k != nullptr ? p.top_k[row] : 0;
    if (k != 0 && k < p.vocab) cut = find_cut<false>(cluster, sh, slice, weigh, low, 0ull, (uint64_t)k);
    const float share = p.top_p != nullptr ? p.top_p[row] : 1.0f;
    if (share < 1.0f) {
        uint64_t mine = 0;
        for (uint32_t i = threadIdx.x; i < slice.size; i += kSampleThreads) {
            const float x = slice.at(i);
            if (composite(x, slice.begin + i) >= cut) mine += Weigh::units(weigh.real(x));
        }
        mine = block_sum(mine, sh.warp_values);
        if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->total[rank] = mine;
        cluster.sync();
        uint64_t total = 0;
        for (uint32_t r = 0; r < blocks; ++r) total += sh.total[r];
        const double wanted = ceil((double)fmaxf(share, 0.0f) * (double)total);
        cut = find_cut<true>(cluster, sh, slice, weigh, low, cut, wanted < 1.0 ? 1ull : (uint64_t)wanted);
    }
    double least = p.min_p != nullptr ? (double)p.min_p[row] : 0.0;
    if (least > 1.0) least = 1.0;
    auto kept_units = [&](uint32_t i) -> uint64_t {
        const float x = slice.at(i);
        if (composite(x, slice.begin + i) < cut) return 0;
        const double w = weigh.real(x);
        return w < least ? 0ull : Weigh::units(w);
    };

    // ---- the token ----
    const uint32_t tile_count = ceil_div(slice.size, kTile);
    for (uint32_t tile = warp; tile < tile_count; tile += kSampleWarps) {
        uint64_t sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kTile / 32; ++j) {
            const uint32_t i = tile * kTile + j * 32 + lane;
            if (i < slice.size) sum += kept_units(i);
        }
        sum = warp_sum(sum);
        if (lane == 0) tiles[tile] = sum;
    }
    __syncthreads();
    uint64_t mine = 0;
    for (uint32_t tile = threadIdx.x; tile < tile_count; tile += kSampleThreads) mine += tiles[tile];
    mine = block_sum(mine, sh.warp_values);
    cluster.sync();  // sh.total of the top-p pass has been read everywhere
    if (threadIdx.x < blocks) cluster.map_shared_rank(&sh, threadIdx.x)->total[rank] = mine;
    cluster.sync();  // the last look into another block's shared memory is behind this
    uint64_t total = 0, before = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
        if (r < rank) before += sh.total[r];
        total += sh.total[r];
    }
    const float uniform = p.uniform[row];
    const double aim = uniform > 0.0f ? floor((double)uniform * (double)total) : 0.0;
    uint64_t target = aim < (double)total ? (uint64_t)aim : total - 1;
    if (target > total - 1) target = total - 1;
    if (target < before || target >= before + mine || warp != 0) return;
    // the tile, 32 at a time
    uint64_t running = before;
    uint32_t tile = 0;
    for (uint32_t t0 = 0; t0 < tile_count; t0 += 32) {
        const uint64_t own = t0 + lane < tile_count ? tiles[t0 + lane] : 0;
        uint64_t inclusive = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, inclusive, d);
            if (lane >= (uint32_t)d) inclusive += y;
        }
        const uint32_t passed = __ballot_sync(0xffffffffu, running + inclusive > target);
        if (passed != 0) {
            const int first = __ffs(passed) - 1;
            tile = t0 + first;
            running += __shfl_sync(0xffffffffu, inclusive - own, first);
            break;
        }
        running += __shfl_sync(0xffffffffu, inclusive, 31);
    }
    // eight neighbours per lane
    uint64_t own[kTile / 32], sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < kTile / 32; ++j) {
        const uint32_t i = tile * kTile + lane * (kTile / 32) + j;
        own[j] = i < slice.size ? kept_units(i) : 0;
        sum += own[j];
    }
    uint64_t inclusive = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= (uint32_t)d) inclusive += y;
    }
    running += inclusive - sum;
    if (running <= target && running + sum > target) {
#pragma unroll
        for (uint32_t j = 0; j < kTile / 32; ++j) {
            if (running <= target && running + own[j] > target) {
                p.tokens[row] = slice.begin + tile * kTile + lane * (kTile / 32) + j;
                if (p.probabilities != nullptr) p.probabilities[row] = (float)((double)own[j] / (double)total);
            }
            running += own[j];
        }
    }
}

template <typename T>
cudaError_t launch_sample_of(const SampleArgs &args, cudaStream_t stream) {
    // blocks per row: at least 4096 logits each, 8 at most
    uint32_t blocks = 1;
    while (blocks < kMostBlocks && args.vocab / (2 * blocks) >= 4096) blocks *= 2;
    const uint32_t slice = ceil_div(args.vocab, blocks);
    const size_t slice_bytes = (size_t)slice * sizeof(T) + 32;
    const bool on_chip = slice_bytes <= kSliceBytes;
    const size_t smem = sizeof(SampleShared) + (size_t)ceil_div(slice, kTile) * 8 + (on_chip ? slice_bytes : 0);
    static bool configured[kMaxDevices] = {};
    const int slot = device_slot();
    if (slot < 0 || !configured[slot]) {
        cudaError_t status = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  (int)(sizeof(SampleShared) + kMostTiles * 8 / kMostBlocks + kSliceBytes));
        if (status != cudaSuccess) return status;
        if (slot >= 0) configured[slot] = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(args.rows * blocks);
    config.blockDim = dim3(kSampleThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = blocks;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, sample_kernel<T>, args, slice, on_chip ? 1u : 0u);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &args, cudaStream_t stream) {
    if (args.dtype == kF32) return launch_sample_of<float>(args, stream);
    if (args.dtype == kBF16) return launch_sample_of<__nv_bfloat16>(args, stream);
    return launch_sample_of<__half>(args, stream);
}

}  // namespace q4b
