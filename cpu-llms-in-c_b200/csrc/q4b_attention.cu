// Attention of a few new tokens per sequence over the paged cache (decode, verify).
//
//   out(t, h) = sum_j w_j v(j) / sum_j w_j,   w_j = exp(scale q(t, h) . k(j) - m),   m the running maximum
//
// over the visible places j of the sequence: j <= p, and behind a window only j > p - window or j < sinks.
//
// Every cached value is read once and meets as few multiplications as there are rows (query heads of one key head x
// new tokens), so the kernel is bound by memory.  All query rows of a key head are taken together: 8 R of them, as
// columns of the tensor-core products
//     S^T [16 keys x 8 R rows] = K Q^T          (mma.sync m16n8k16, K from shared memory by ldmatrix)
//     O^T [D x 8 R rows]      += V^T P^T        (V by ldmatrix.trans, P^T by movmatrix from S^T's registers)
// in that orientation a row's maximum, sum and output column sit in the same lanes, eight rows cost no padding to
// sixteen, and a warp needs nothing from the others until its share of the keys is done.  An fp16 weight has no bits below
// 2^-24: with the largest at 1 a long context's many small ones would be lost together, so the largest is 2^15 there.
// A row's sum takes the weights as they meet the values, rounded to 16 bits: equal values come back as they are.  A second
// product with what the rounding leaves out would give the error of fp32 weights instead of 1.1 to 1.2 times it; it costs
// 1% of a step of 32 users with up to 8 rows each, but 10% with 16 rows, or with one user behind 16,000 tokens.
//
// Split: a unit is (sequence, key head, 8 R rows).  The units' groups of 16 keys form one list, cut into equal ranges,
// one per thread block, whatever the lengths are (they live in device memory; the host does not know them).  Within
// its range of a unit a thread block deals groups to its eight warps in turn; each warp streams its own keys and
// values through its own ring in shared memory with cp.async, so no barrier stands between a warp and its bytes.  At
// the end of a unit the warps' sums meet in shared memory.  A unit that is cut over thread blocks leaves fp32 sums in
// the workspace; whoever arrives last adds them up in block order, so results do not depend on timing.
//
// Matrix instructions cut a running sum off where they would have to round it, so a long chain of them comes out too small
// (by 8 x 10^-4 over the 8,192 products of a warp at a million keys).  A thread block's range of a unit is therefore taken in
// pieces of at most 8 x 512 groups (fp16; 8 x 4,096 in bf16), whose sums meet in the workspace by additions that round.
//
// One sequence has few units and waits mostly for sums to travel: there the thread blocks come in clusters of eight, each
// key head is cut into whole clusters of shares, and a cluster's sums meet in distributed shared memory; the workspace is
// left for units that take several clusters.
//
// Measured on B200 (24 query heads on 4 key heads of 256): single tokens of 32 users with 4,000 to 16,384 cached ones each,
// bf16, 218 us = 6.3 TB/s of 6.54; one token behind 1,024, 11 us, which is latency: lengths, page number, keys, exchange.
#include "q4b_cache.cuh"

#include <cooperative_groups.h>
#include <cmath>
#include <type_traits>

namespace q4b {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kWarps = 8;
constexpr uint32_t kThreads = kWarps * 32;
constexpr uint32_t kKeys = kGroupKeys;
constexpr uint32_t kMostRows = 16;      // rows of a unit, at most
constexpr uint32_t kMostHead = 256;
constexpr uint32_t kBlocksPerSm = 1;
// a unit's share of a thread block is at least this many groups (one per warp): fewer would leave warps idle while
// adding sums to join
constexpr uint32_t kLeastShare = 8;
// the largest weight, as a power of two
template <typename T> constexpr float kLift = std::is_same<T, __half>::value ? 15.0f : 0.0f;
constexpr uint32_t kCluster = 8;        // thread blocks of a cluster, where one sequence has the GPU to itself

template <int D> struct Ring {
    static constexpr uint32_t item = kKeys * D * 2;               // 16 keys or values
    static constexpr uint32_t items = D == 256 ? 3 : D == 128 ? 6 : 8;
};

__device__ inline uint32_t smem_u32(const void *pointer) { return (uint32_t)__cvta_generic_to_shared(pointer); }
__device__ inline float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes, zeros when `bytes` is 0
__device__ inline void copy16(uint32_t to, const void *from, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ inline void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ inline void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ inline void matrices4(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ inline void matrices4_transposed(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ inline uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T> __device__ inline void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ inline void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ inline void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ inline uint32_t pack(float low, float high);
template <> __device__ inline uint32_t pack<__half>(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ inline uint32_t pack<__nv_bfloat16>(float low, float high) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ inline float widen(__half x) { return __half2float(x); }
__device__ inline float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
// whether one of the two 16-bit values of a word is an infinity or a NaN
template <typename T> __device__ inline bool has_nonfinite(uint32_t word) {
    const uint32_t exponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return (word & exponent) == exponent || ((word >> 16) & exponent) == exponent;
}

// Walks the list of units from the one that holds a given group.
struct UnitWalk {
    uint32_t sequence, head, chunk, chunks, chunk_rows;
    SequenceRows rows;
    Groups groups;
};
__device__ inline void unit_groups(const AttentionArgs &p, UnitWalk &u) {
    const uint32_t row0 = u.chunk * u.chunk_rows, row1 = min(row0 + u.chunk_rows, u.rows.count * p.group) - 1;
    u.groups = groups_of(u.rows, row0 / p.group, row1 / p.group, p.window, p.sinks);
}
__device__ inline uint64_t sequence_groups(const AttentionArgs &p, const SequenceRows &rows, uint32_t chunk_rows) {
    const uint32_t all = rows.count * p.group;
    uint64_t sum = 0;
    for (uint32_t row0 = 0; row0 < all; row0 += chunk_rows) {
        const uint32_t row1 = min(row0 + chunk_rows, all) - 1;
        sum += groups_of(rows, row0 / p.group, row1 / p.group, p.window, p.sinks).count();
    }
    return sum * p.cache.kv_heads;
}
// sum over the thread block; every thread gets it, and the sum before it
__device__ inline uint64_t block_scan(uint64_t value, uint64_t *scratch, uint64_t &before) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t inclusive = value;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t other = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= (uint32_t)d) inclusive += other;
    }
    if (lane == 31) scratch[warp] = inclusive;
    __syncthreads();
    uint64_t total = 0, warps_before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) warps_before += scratch[w];
        total += scratch[w];
    }
    __syncthreads();
    before = warps_before + inclusive - value;
    return total;
}

// CLUSTER: launched in clusters of kCluster, for one sequence
template <typename T, int D, int R, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
attend_kernel(const __grid_constant__ AttentionArgs p) {
    constexpr uint32_t kRows = 8 * R;
    constexpr uint32_t kChunks = D / 8;          // 16-byte pieces of a row
    constexpr uint32_t kItem = Ring<D>::item, kItems = Ring<D>::items;
    constexpr uint32_t kFold = std::is_same<T, __half>::value ? kFoldStepsF16 : kFoldStepsBF16;
    extern __shared__ __align__(128) uint8_t smem[];
    // [query rows][rings of the warps]; the rings' place is also where the warps' sums meet
    T *const query = reinterpret_cast<T *>(smem);
    uint8_t *const rings = smem + kRows * D * 2;
    // [warps][kRows][D], rows four floats further apart: a warp's stores then fall into 32 different banks
    constexpr uint32_t kSumRow = D + 4;
    float *const sums = reinterpret_cast<float *>(rings);
    __shared__ float top_of[kWarps][kRows], total_of[kWarps][kRows];
    __shared__ uint64_t scan[kWarps];
    __shared__ uint64_t found_before;
    __shared__ uint32_t found_sequence, last_to_arrive;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(rings) + warp * kItem * kItems;

    // ---- this thread block's range of the list of groups ----
    UnitWalk u;
    u.chunk_rows = kRows;
    u.head = 0;
    u.chunk = 0;
    uint64_t begin, end, share, unit_begin;  // in groups; a thread block has [begin, end), `share` of them at most
    uint64_t unit_stride = 0;                // not 0: units begin this far apart, each cut into whole clusters of shares
    uint32_t unit_clusters = 0;              // clusters that share a unit
    if constexpr (CLUSTER) {
        // One sequence: its key heads are equally long.  Each is cut into equally many shares, a whole number of clusters,
        // so the shares' sums meet in distributed shared memory and few or none go through the workspace.
        u.sequence = 0;
        u.rows = sequence_rows(p.batch, p.cache.page_tokens, 0, p.status);
        u.chunks = ceil_div(u.rows.count * p.group, kRows);
        const uint32_t clusters = gridDim.x / kCluster;
        if (u.chunks == 1 && p.cache.kv_heads <= clusters) {
            unit_groups(p, u);
            const uint32_t count = u.groups.count();
            unit_clusters = min(clusters / p.cache.kv_heads, ceil_div(count, kCluster * kLeastShare));
            const uint32_t parts = unit_clusters * kCluster;
            share = ceil_div(count, parts);
            unit_stride = share * parts;
            u.head = blockIdx.x / parts;
            if (u.head >= p.cache.kv_heads) return;
            unit_begin = u.head * unit_stride;
            begin = unit_begin + min(blockIdx.x % parts * (uint32_t)share, count);  // the last shares may be empty
            end = min(begin + share, unit_begin + count);
        }
    }
    if (unit_stride == 0) {
        uint64_t all = 0, before, mine = 0;
        for (uint32_t s0 = 0; s0 < p.batch.sequences; s0 += kThreads) {
            const uint32_t s = s0 + threadIdx.x;
            mine = s < p.batch.sequences ? sequence_groups(p, sequence_rows(p.batch, p.cache.page_tokens, s, p.status), kRows) : 0;
            all += block_scan(mine, scan, before);
        }
        share = max((all + gridDim.x - 1) / gridDim.x, (uint64_t)kLeastShare);
        begin = (uint64_t)blockIdx.x * share;
        end = min(begin + share, all);
        if (begin >= end) return;
        for (uint64_t s0 = 0, sum = 0; sum <= begin; s0 += kThreads) {
            const uint32_t s = (uint32_t)s0 + threadIdx.x;
            uint64_t total = all;  // a batch of one round has its numbers at hand
            if (p.batch.sequences > kThreads) {
                mine = s < p.batch.sequences ? sequence_groups(p, sequence_rows(p.batch, p.cache.page_tokens, s, p.status), kRows) : 0;
                total = block_scan(mine, scan, before);
            }
            if (sum + before <= begin && begin < sum + before + mine) {
                found_sequence = s;
                found_before = sum + before;
            }
            sum += total;
        }
        __syncthreads();
        u.sequence = found_sequence;
        u.rows = sequence_rows(p.batch, p.cache.page_tokens, u.sequence, p.status);
        u.chunks = ceil_div(u.rows.count * p.group, kRows);
        unit_begin = found_before;
        unit_groups(p, u);
        // the unit within the sequence: heads outside, chunks of rows inside
        while (unit_begin + u.groups.count() <= begin) {
            unit_begin += u.groups.count();
            if (++u.chunk == u.chunks) {
                u.chunk = 0;
                ++u.head;
            }
            unit_groups(p, u);
        }
    }

    const float scale = p.scale * 1.44269504088896341f;
    uint64_t position = begin;
    do {
        const uint32_t unit_count = u.groups.count();
        const uint64_t unit_end = unit_begin + unit_count;
        // A long range is taken in pieces, so that no warp's chain of products gets longer than the sums bear: all but the last
        // leave theirs in the workspace.
        const uint32_t g0 = (uint32_t)(position - unit_begin);
        const uint32_t g1 = min((uint32_t)(min(unit_end, end) - unit_begin), g0 + kWarps * kFold);
        const bool last_piece = unit_begin + g1 == min(unit_end, end);
        const uint32_t unit_row0 = u.chunk * kRows, unit_rows = min(kRows, u.rows.count * p.group - unit_row0);
        const int64_t place0 = (int64_t)u.rows.length - u.rows.count;  // of the sequence's first new token
        const uint32_t keys_end = u.groups.end == 0 ? 0 : u.rows.length;
        const uint32_t *table = p.batch.table + (size_t)u.sequence * p.batch.table_stride;

        __syncthreads();  // the last unit's sums have been read: the rings are free
        // the places of this lane's rows 8 r + 2 t and 8 r + 2 t + 1 (negative: a row that sees nothing)
        int64_t place[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t row = 8 * r + 2 * t + i;
                place[r][i] = row < unit_rows ? place0 + (unit_row0 + row) / p.group : -1;
            }
        }
        // between these places every row of the unit sees everything: no mask, no look at the values
        const int64_t least = place0 + unit_row0 / p.group, most = place0 + (unit_row0 + unit_rows - 1) / p.group;

        float out[R][D / 16][4], top[R][2], total[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            top[r][0] = top[r][1] = -INFINITY;
            total[r][0] = total[r][1] = 0.0f;
#pragma unroll
            for (int m = 0; m < D / 16; ++m) out[r][m][0] = out[r][m][1] = out[r][m][2] = out[r][m][3] = 0.0f;
        }

        // ---- the stream: items K, V, K, V, ... of this warp's groups g0 + warp, g0 + warp + 8, ... ----
        const uint32_t my_groups = g0 + warp < g1 ? (g1 - g0 - warp + kWarps - 1) / kWarps : 0;
        const uint32_t my_items = 2 * my_groups;
        // The page of the group that is fetched next is looked up one group ahead.
        auto page_of = [&](uint32_t index) -> uint32_t {
            if (index >= my_groups || keys_end == 0) return 0xffffffffu;
            const uint32_t key0 = u.groups.at(g0 + warp + index * kWarps) * kKeys;
            return __ldg(table + (key0 >> p.cache.page_shift));
        };
        uint32_t page = page_of(0), next_page = page_of(1);
        auto fetch = [&](uint32_t item) {
            if (item < my_items) {
                const uint32_t index = item >> 1;
                const uint32_t key0 = u.groups.at(g0 + warp + index * kWarps) * kKeys;
                const bool held = page < p.cache.pages;
                if (!held && lane == 0 && keys_end != 0) report(p.status, kBadPage);
                const T *pool = static_cast<const T *>(item & 1 ? p.cache.values : p.cache.keys);
                const T *from = pool + (((size_t)(held ? page : 0) * p.cache.kv_heads + u.head) * p.cache.page_tokens +
                                        (key0 & (p.cache.page_tokens - 1))) * D;
                const uint32_t to = ring + (item % kItems) * kItem;
#pragma unroll
                for (uint32_t i = 0; i < kKeys * kChunks / 32; ++i) {
                    const uint32_t cell = i * 32 + lane, key = cell / kChunks, piece = cell % kChunks;
                    // keys behind the sequence's end are zeros, not what the page happens to hold
                    copy16(to + (key * kChunks + (piece ^ (key & 7))) * 16, from + cell * 8,
                           held && key0 + key < keys_end ? 16 : 0);
                }
                if (item & 1) {
                    page = next_page;
                    next_page = page_of(index + 2);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (uint32_t i = 0; i + 1 < kItems; ++i) fetch(i);

        // ---- query rows, pieces of a row turned by the row (no bank conflicts for ldmatrix) ----
        for (uint32_t i = threadIdx.x; i < kRows * kChunks; i += kThreads) {
            const uint32_t row = i / kChunks, piece = i % kChunks;
            uint4 value = make_uint4(0, 0, 0, 0);
            if (row < unit_rows) {
                const uint32_t flat = unit_row0 + row;
                const T *from = static_cast<const T *>(p.q) + (size_t)(u.rows.begin + flat / p.group) * p.ldq +
                                (size_t)(u.head * p.group + flat % p.group) * D + piece * 8;
                value = *reinterpret_cast<const uint4 *>(from);
            }
            *reinterpret_cast<uint4 *>(query + row * D + ((piece ^ (row & 7)) * 8)) = value;
        }
        __syncthreads();

        const uint32_t q_base = smem_u32(query);
        for (uint32_t index = 0; index < my_groups; ++index) {
            const uint32_t key0 = u.groups.at(g0 + warp + index * kWarps) * kKeys;
            // -- S^T = K Q^T --
            copy_wait<kItems - 2>();
            __syncwarp();
            fetch(2 * index + kItems - 1);
            const uint32_t k_base = ring + ((2 * index) % kItems) * kItem;
            float score[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r) score[r][0] = score[r][1] = score[r][2] = score[r][3] = 0.0f;
            {
                const uint32_t key = lane & 15, half = lane >> 4;        // K: keys 0-7, 8-15, then the next 8 columns
                const uint32_t q_row = lane & 7, q_piece = lane >> 3;    // Q: four 8-column pieces of eight rows
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t ka[4], kb[4];
                    matrices4(ka, k_base + (key * kChunks + ((4 * c + half) ^ (key & 7))) * 16);
                    matrices4(kb, k_base + (key * kChunks + ((4 * c + 2 + half) ^ (key & 7))) * 16);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        uint32_t q[4];
                        matrices4(q, q_base + ((8 * r + q_row) * kChunks + ((4 * c + q_piece) ^ q_row)) * 16);
                        mma<T>(score[r], ka, q[0], q[1]);
                        mma<T>(score[r], kb, q[2], q[3]);
                    }
                }
            }
            // -- mask, running maximum, weights --
            const bool clear = (int64_t)key0 + kKeys - 1 <= least &&
                               (p.window == 0 || (int64_t)key0 > most - (int64_t)p.window || key0 + kKeys <= p.sinks);
            uint32_t weight[R][2];
            float keep[R][2];
            bool seen[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float s[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t key = key0 + gid + 8 * (i >> 1);
                    const int64_t at = place[r][i & 1];
                    seen[r][i] = clear || ((int64_t)key <= at && (p.window == 0 || (int64_t)key > at - (int64_t)p.window ||
                                                                  key < p.sinks));
                    s[i] = seen[r][i] ? score[r][i] * scale : -INFINITY;
                }
                float high[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], d));
                    const float grown = fmaxf(top[r][i], high[i] - kLift<T>);
                    const float base = grown == -INFINITY ? 0.0f : grown;  // nothing visible so far
                    keep[r][i] = exp2_fast(top[r][i] - base);
                    top[r][i] = grown;
                    s[i] = exp2_fast(s[i] - base);
                    s[i + 2] = exp2_fast(s[i + 2] - base);
                }
                const uint32_t first = pack<T>(s[0], s[1]), second = pack<T>(s[2], s[3]);
#pragma unroll
                for (int i = 0; i < 2; ++i)  // as they meet the values
                    total[r][i] = total[r][i] * keep[r][i] +
                                  (widen(reinterpret_cast<const T *>(&first)[i]) + widen(reinterpret_cast<const T *>(&second)[i]));
                // keys gid (and gid + 8) of rows 2t, 2t+1 -> rows gid of keys 2t, 2t+1
                weight[r][0] = transposed(first);
                weight[r][1] = transposed(second);
#pragma unroll
                for (int m = 0; m < D / 16; ++m) {
                    out[r][m][0] *= keep[r][0];
                    out[r][m][1] *= keep[r][1];
                    out[r][m][2] *= keep[r][0];
                    out[r][m][3] *= keep[r][1];
                }
            }
            // -- O^T += V^T P^T --
            copy_wait<kItems - 2>();
            __syncwarp();
            fetch(2 * index + kItems);
            const uint32_t v_base = ring + ((2 * index + 1) % kItems) * kItem;
            bool poisoned = false;
            if (!clear) {
                // 0 x infinity is NaN: values that some row must not see are looked at before they are multiplied
                for (uint32_t i = 0; i < kKeys * kChunks / 32; ++i) {
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(v_base + (i * 32 + lane) * 16) : "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j) poisoned = poisoned || has_nonfinite<T>(w[j]);
                }
                poisoned = __any_sync(0xffffffffu, poisoned);
            }
            if (!poisoned) {
                const uint32_t key = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
                for (int m = 0; m < D / 16; ++m) {
                    uint32_t v[4];
                    matrices4_transposed(v, v_base + (key * kChunks + ((2 * m + half) ^ (key & 7))) * 16);
#pragma unroll
                    for (int r = 0; r < R; ++r) mma<T>(out[r][m], v, weight[r][0], weight[r][1]);
                }
            } else {
                // the same sums in plain fp32, each row over the keys that it sees
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t back[2] = {transposed(weight[r][0]), transposed(weight[r][1])};
                    for (uint32_t key = 0; key < kKeys; ++key) {
                        const uint32_t word = __shfl_sync(0xffffffffu, back[key >> 3], (key & 7) * 4 + t);
                        const uint32_t mask = __shfl_sync(0xffffffffu,
                            (uint32_t)(key < 8 ? seen[r][0] : seen[r][2]) | (uint32_t)(key < 8 ? seen[r][1] : seen[r][3]) << 1,
                            (key & 7) * 4 + t);
                        const T *pair = reinterpret_cast<const T *>(&word);
                        const float w[2] = {widen(pair[0]), widen(pair[1])};
#pragma unroll
                        for (int m = 0; m < D / 16; ++m) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t column = 16 * m + gid + 8 * (i >> 1);
                                uint16_t raw;
                                asm volatile("ld.shared.u16 %0, [%1];"
                                             : "=h"(raw)
                                             : "r"(v_base + (key * kChunks + ((column >> 3) ^ (key & 7))) * 16 + (column & 7) * 2)
                                             : "memory");
                                if ((mask >> (i & 1)) & 1u)
                                    out[r][m][i] += w[i & 1] * widen(*reinterpret_cast<const T *>(&raw));
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }
        copy_wait<0>();

        // ---- the warps' sums meet ----
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) total[r][i] += __shfl_xor_sync(0xffffffffu, total[r][i], d);
                if (gid == 0) {
                    top_of[warp][8 * r + 2 * t + i] = top[r][i];
                    total_of[warp][8 * r + 2 * t + i] = total[r][i];
                }
            }
        }
        __syncthreads();  // every ring is drained and every maximum is there
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t row = 8 * r + 2 * t + i;
                float high = top_of[0][row];
#pragma unroll
                for (uint32_t w = 1; w < kWarps; ++w) high = fmaxf(high, top_of[w][row]);
                const float factor = top[r][i] == -INFINITY ? 0.0f : exp2_fast(top[r][i] - high);
                // a warp that saw nothing has sums of zero (and NaN only from rows that see a NaN)
                float *to = sums + (warp * kRows + row) * kSumRow + gid;
#pragma unroll
                for (int m = 0; m < D / 16; ++m) {
                    to[16 * m] = out[r][m][i] * factor;
                    to[16 * m + 8] = out[r][m][2 + i] * factor;
                }
            }
        }
        __syncthreads();
        const bool whole = unit_begin >= begin && unit_end <= end;
        const bool first_piece = position == max(begin, unit_begin);
        // four outputs over the warps and the pieces in front of this one; false: they wait for the next piece
        float *const folds = p.folds + (size_t)blockIdx.x * kFoldFloats;  // every thread reads what it wrote
        auto gather = [&](uint32_t i, uint32_t row, uint32_t column, float4 &sum, float &high, float &mass) {
            sum = make_float4(0, 0, 0, 0);
            high = -INFINITY;
            mass = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) high = fmaxf(high, top_of[w][row]);
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float4 part = *reinterpret_cast<const float4 *>(sums + (w * kRows + row) * kSumRow + column);
                sum.x += part.x; sum.y += part.y; sum.z += part.z; sum.w += part.w;
                mass += top_of[w][row] == -INFINITY ? total_of[w][row] : total_of[w][row] * exp2_fast(top_of[w][row] - high);
            }
            if (first_piece && last_piece) return true;
            float4 *const fold = reinterpret_cast<float4 *>(folds) + i;
            float2 *const told = reinterpret_cast<float2 *>(folds + kMostRows * kMostHead) + i;  // (top, total)
            if (!first_piece) {
                const float4 before = *fold;
                const float grown = fmaxf(high, told->x);
                const float keep = told->x == -INFINITY ? 1.0f : exp2_fast(told->x - grown);  // sums of nothing are zeros, or NaN
                const float scaled = high == -INFINITY ? 1.0f : exp2_fast(high - grown);
                sum.x = sum.x * scaled + before.x * keep;
                sum.y = sum.y * scaled + before.y * keep;
                sum.z = sum.z * scaled + before.z * keep;
                sum.w = sum.w * scaled + before.w * keep;
                mass = mass * scaled + told->y * keep;
                high = grown;
            }
            if (!last_piece) {
                *fold = sum;
                *told = make_float2(high, mass);
            }
            return last_piece;
        };
        if (CLUSTER && unit_stride != 0) {
            cg::cluster_group cluster = cg::this_cluster();
            const uint32_t rank = cluster.block_rank(), items = unit_rows * (D / 4);
            float *const own_sum = sums + kWarps * kRows * kSumRow, *const own_top = own_sum + kRows * D,
                        *const own_total = own_top + kRows;
            for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
                const uint32_t row = i / (D / 4), column = (i % (D / 4)) * 4;
                float4 sum;
                float high, mass;
                if (!gather(i, row, column, sum, high, mass)) continue;
                *reinterpret_cast<float4 *>(own_sum + row * D + column) = sum;
                if (column == 0) {
                    own_top[row] = high;
                    own_total[row] = mass;
                }
            }
            if (!last_piece) {
                position = unit_begin + g1;
                continue;
            }
            cluster.sync();
            // every block adds an eighth of the outputs up over the cluster
            const uint32_t each = (items + kCluster - 1) / kCluster, i = rank * each + threadIdx.x;
            const bool mine = threadIdx.x < each && i < items;
            const uint32_t row = mine ? i / (D / 4) : 0, column = (i % (D / 4)) * 4;
            float4 sum = make_float4(0, 0, 0, 0);
            float high = -INFINITY, mass = 0.0f;
            if (mine) {
                float top_r[kCluster], total_r[kCluster];
                float4 sum_r[kCluster];
#pragma unroll
                for (uint32_t r = 0; r < kCluster; ++r) {
                    top_r[r] = cluster.map_shared_rank(own_top, r)[row];
                    total_r[r] = cluster.map_shared_rank(own_total, r)[row];
                    sum_r[r] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(own_sum, r) + row * D + column);
                    high = fmaxf(high, top_r[r]);
                }
#pragma unroll
                for (uint32_t r = 0; r < kCluster; ++r) {
                    const float factor = top_r[r] == -INFINITY ? 1.0f : exp2_fast(top_r[r] - high);
                    sum.x += sum_r[r].x * factor; sum.y += sum_r[r].y * factor;
                    sum.z += sum_r[r].z * factor; sum.w += sum_r[r].w * factor;
                    mass += total_r[r] * factor;
                }
            }
            auto answer = [&](const float4 &value, float total) {
                const uint32_t flat = unit_row0 + row;
                T *to = static_cast<T *>(p.out) + (size_t)(u.rows.begin + flat / p.group) * p.ldo +
                        (size_t)(u.head * p.group + flat % p.group) * D + column;
                const float over = total == 0.0f ? 0.0f : 1.0f / total;
                *reinterpret_cast<uint2 *>(to) = make_uint2(pack<T>(value.x * over, value.y * over), pack<T>(value.z * over, value.w * over));
            };
            auto arrived = cluster.barrier_arrive();  // this block has read the others' sums
            if (unit_clusters == 1) {
                if (mine) answer(sum, mass);
            } else {
                // blocks of equal rank in the unit's clusters have the same outputs: the last of them adds up in cluster order
                constexpr uint32_t kItems4 = kMostRows * kMostHead / 4, kSlot = kItems4 * 6;  // sums, then (top, total) pairs
                float *const unit_slots = p.partials + (size_t)(u.head * unit_clusters) * kSlot;
                const uint32_t slot = blockIdx.x / kCluster % unit_clusters;
                if (mine) {
                    reinterpret_cast<float4 *>(unit_slots + (size_t)slot * kSlot)[i] = sum;
                    reinterpret_cast<float2 *>(unit_slots + (size_t)slot * kSlot + 4 * kItems4)[i] = make_float2(high, mass);
                }
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) {
                    uint32_t *const counter = p.arrivals + u.head * kCluster + rank;
                    last_to_arrive = atomicAdd(counter, 1u) == unit_clusters - 1 ? 1u : 0u;
                    if (last_to_arrive) *counter = 0;
                }
                __syncthreads();
                if (last_to_arrive && mine) {
                    __threadfence();
                    high = -INFINITY;
                    mass = 0.0f;
                    sum = make_float4(0, 0, 0, 0);
                    for (uint32_t c0 = 0; c0 < unit_clusters; c0 += 8) {
                        float4 piece[8];
                        float2 told[8];
                        float grown = high;
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) {
                            told[e] = make_float2(-INFINITY, 0.0f);
                            piece[e] = make_float4(0, 0, 0, 0);
                            if (c0 + e < unit_clusters) {
                                const float *const from = unit_slots + (size_t)(c0 + e) * kSlot;
                                piece[e] = __ldcg(reinterpret_cast<const float4 *>(from) + i);
                                told[e] = __ldcg(reinterpret_cast<const float2 *>(from + 4 * kItems4) + i);
                            }
                        }
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) grown = fmaxf(grown, told[e].x);
                        const float keep = high == -INFINITY ? 1.0f : exp2_fast(high - grown);
                        sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
                        mass *= keep;
                        high = grown;
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) {
                            const float factor = told[e].x == -INFINITY ? 1.0f : exp2_fast(told[e].x - high);
                            sum.x += piece[e].x * factor; sum.y += piece[e].y * factor;
                            sum.z += piece[e].z * factor; sum.w += piece[e].w * factor;
                            mass += told[e].y * factor;
                        }
                    }
                    answer(sum, mass);
                }
            }
            cluster.barrier_wait(static_cast<cg::cluster_group::arrival_token &&>(arrived));
            return;
        }
        // the unit's first thread block has its counter; a thread block leaves two sums at most: of the unit that it
        // begins in the middle of, and of the one that it does not finish
        const uint32_t first_block = whole ? 0 : (uint32_t)(unit_begin / share);
        const uint32_t last_block = whole ? 0 : (uint32_t)((unit_end - 1) / share);
        const uint32_t slot = 2 * blockIdx.x + (unit_begin < begin ? 0u : 1u);
        constexpr uint32_t kSlotFloats = kMostRows * (kMostHead + 2);
        float *const partial = p.partials + (size_t)slot * kSlotFloats;  // [rows][D], then maxima, then totals
        for (uint32_t i = threadIdx.x; i < unit_rows * (D / 4); i += kThreads) {
            const uint32_t row = i / (D / 4), column = (i % (D / 4)) * 4;
            float4 sum;
            float high, mass;
            if (!gather(i, row, column, sum, high, mass)) continue;
            if (whole) {
                const uint32_t flat = unit_row0 + row;
                T *to = static_cast<T *>(p.out) + (size_t)(u.rows.begin + flat / p.group) * p.ldo +
                        (size_t)(u.head * p.group + flat % p.group) * D + column;
                const float over = mass == 0.0f ? 0.0f : 1.0f / mass;
                *reinterpret_cast<uint2 *>(to) = make_uint2(pack<T>(sum.x * over, sum.y * over), pack<T>(sum.z * over, sum.w * over));
            } else {
                *reinterpret_cast<float4 *>(partial + row * D + column) = sum;
                if (column == 0) {
                    partial[kMostRows * kMostHead + row] = high;
                    partial[kMostRows * (kMostHead + 1) + row] = mass;
                }
            }
        }
        if (!last_piece) {
            position = unit_begin + g1;
            continue;
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t arrived = atomicAdd(p.arrivals + first_block, 1u);
                last_to_arrive = arrived == last_block - first_block ? 1u : 0u;
                if (last_to_arrive) p.arrivals[first_block] = 0;
            }
            __syncthreads();
            if (last_to_arrive) {
                __threadfence();
                // the first block's sum is of the unit that it does not finish, the others' of the one they begin in
                const uint32_t parts = last_block - first_block + 1;
                const float *const from = p.partials + (size_t)(2 * first_block) * kSlotFloats;
                auto slot_of = [&](uint32_t part) { return from + (size_t)(2 * part + (part == 0 ? 1u : 0u)) * kSlotFloats; };
                float *const factor_of = sums;                          // [parts][kRows], in the rings' place
                float *const mass_of = sums + (size_t)gridDim.x * kRows;
                for (uint32_t i = threadIdx.x; i < parts * unit_rows; i += kThreads) {
                    const uint32_t part = i / unit_rows, row = i % unit_rows;
                    factor_of[part * kRows + row] = __ldcg(slot_of(part) + kMostRows * kMostHead + row);
                    mass_of[part * kRows + row] = __ldcg(slot_of(part) + kMostRows * (kMostHead + 1) + row);
                }
                __syncthreads();
                for (uint32_t row = warp; row < unit_rows; row += kWarps) {
                    float high = -INFINITY, mass = 0.0f;
                    for (uint32_t part = lane; part < parts; part += 32) high = fmaxf(high, factor_of[part * kRows + row]);
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
                    for (uint32_t part = lane; part < parts; part += 32) {
                        const float own = factor_of[part * kRows + row];
                        const float factor = own == -INFINITY ? 1.0f : exp2_fast(own - high);
                        factor_of[part * kRows + row] = factor;
                        mass += mass_of[part * kRows + row] * factor;
                    }
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, d);
                    if (lane == 0) total_of[0][row] = mass;
                }
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < unit_rows * (D / 4); i += kThreads) {
                    const uint32_t row = i / (D / 4), column = (i % (D / 4)) * 4;
                    float4 sum = make_float4(0, 0, 0, 0);
                    // sixteen loads on their way per thread: one thread block takes in 60 bytes per clock like that
                    for (uint32_t part0 = 0; part0 < parts; part0 += 16) {
                        float4 piece[16];
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e)
                            if (part0 + e < parts)
                                piece[e] = __ldcg(reinterpret_cast<const float4 *>(slot_of(part0 + e) + row * D + column));
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) {
                            if (part0 + e < parts) {
                                const float factor = factor_of[(part0 + e) * kRows + row];
                                sum.x += piece[e].x * factor; sum.y += piece[e].y * factor;
                                sum.z += piece[e].z * factor; sum.w += piece[e].w * factor;
                            }
                        }
                    }
                    const float mass = total_of[0][row];
                    const uint32_t flat = unit_row0 + row;
                    T *to = static_cast<T *>(p.out) + (size_t)(u.rows.begin + flat / p.group) * p.ldo +
                            (size_t)(u.head * p.group + flat % p.group) * D + column;
                    const float over = mass == 0.0f ? 0.0f : 1.0f / mass;
                    *reinterpret_cast<uint2 *>(to) = make_uint2(pack<T>(sum.x * over, sum.y * over), pack<T>(sum.z * over, sum.w * over));
                }
            }
        }

        // ---- the next unit ----
        position = min(unit_end, end);
        if (position < end) {
            unit_begin = unit_end;
            if (++u.chunk == u.chunks) {
                u.chunk = 0;
                if (++u.head == p.cache.kv_heads) {
                    u.head = 0;
                    do {  // sequences without new tokens have no units
                        ++u.sequence;
                        u.rows = sequence_rows(p.batch, p.cache.page_tokens, u.sequence, p.status);
                    } while (u.rows.count == 0 && u.sequence + 1 < p.batch.sequences);
                    u.chunks = ceil_div(u.rows.count * p.group, kRows);
                }
            }
            unit_groups(p, u);
        }
    } while (position < end);
}

template <typename T, int D, int R, bool CLUSTER>
cudaError_t launch_instance(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    constexpr size_t stream_bytes = (size_t)kWarps * Ring<D>::item * Ring<D>::items;
    constexpr size_t sum_bytes = (size_t)kWarps * 8 * R * (D + 4) * 4 + (size_t)8 * R * (D + 2) * 4;
    constexpr size_t smem = (size_t)8 * R * D * 2 + (stream_bytes > sum_bytes ? stream_bytes : sum_bytes);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)sm_count * kBlocksPerSm / (CLUSTER ? kCluster : 1) * (CLUSTER ? kCluster : 1));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = kCluster;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = CLUSTER ? 1 : 0;
    static int room[kMaxDevices] = {};  // clusters that a device holds at once; 1 where there are none
    const int slot = device_slot();
    int clusters = slot >= 0 ? room[slot] : 0;
    if (clusters == 0) {
        cudaError_t status = cudaFuncSetAttribute(attend_kernel<T, D, R, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (status != cudaSuccess) return status;
        clusters = 1;
        if (CLUSTER) {
            status = cudaOccupancyMaxActiveClusters(&clusters, attend_kernel<T, D, R, CLUSTER>, &config);
            if (status != cudaSuccess) return status;
            if (clusters < 1) clusters = 1;
            if (clusters > sm_count / (int)kCluster) clusters = sm_count / (int)kCluster;
        }
        if (slot >= 0) room[slot] = clusters;
    }
    if (CLUSTER) config.gridDim = dim3((unsigned)clusters * kCluster);
    return cudaLaunchKernelEx(&config, attend_kernel<T, D, R, CLUSTER>, args);
}

template <typename T, int D>
cudaError_t launch_rows(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)(args.most_tokens != 0 ? args.most_tokens : args.batch.tokens) * args.group;
    if (args.batch.sequences == 1)
        return rows <= 8 ? launch_instance<T, D, 1, true>(args, sm_count, stream) : launch_instance<T, D, 2, true>(args, sm_count, stream);
    return rows <= 8 ? launch_instance<T, D, 1, false>(args, sm_count, stream) : launch_instance<T, D, 2, false>(args, sm_count, stream);
}

template <typename T>
cudaError_t launch_head(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    switch (args.cache.head_size) {
        case 64: return launch_rows<T, 64>(args, sm_count, stream);
        case 128: return launch_rows<T, 128>(args, sm_count, stream);
        case 256: return launch_rows<T, 256>(args, sm_count, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

size_t attention_partial_bytes(int sm_count) {
    return (size_t)sm_count * kBlocksPerSm * 2 * kMostRows * (kMostHead + 2) * sizeof(float);
}
size_t attention_fold_bytes(int sm_count) { return (size_t)sm_count * kBlocksPerSm * kFoldFloats * sizeof(float); }
// a counter per thread block, and behind them the owners of the folded sums (a prompt's thread blocks are more than SMs)
size_t attention_arrival_bytes(int sm_count) { return (size_t)sm_count * kBlocksPerSm * 2 * sizeof(uint32_t); }

cudaError_t launch_attention(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)(args.most_tokens != 0 ? args.most_tokens : args.batch.tokens) * args.group;
    if (rows > kMostRows && prompt_serves(args)) return launch_prompt(args, sm_count, stream);
    return args.cache.dtype == kBF16 ? launch_head<__nv_bfloat16>(args, sm_count, stream)
                                     : launch_head<__half>(args, sm_count, stream);
}

}  // namespace q4b
