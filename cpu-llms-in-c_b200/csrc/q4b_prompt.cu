// Attention of many new tokens per sequence over the paged cache (prompts, pieces of prompts, wide verify steps).
//
//   out(t, h) = sum_j w_j v(j) / sum_j w_j,   w_j = exp(scale q(t, h) . k(j) - m)
//
// The tensor cores' share is 4 D multiplications per visible (query head, key) pair, so the kernel is bound by them and
// by what feeds them.  A unit is 128 query rows of one key head -- (token, query head of the group) pairs, tokens
// outside -- so a key head's keys and values are read once for all its query heads.  Per tile of 128 keys:
//   S[128 x 128] = Q K^T   tcgen05.mma, both operands in shared memory (128-byte swizzle), S in TMEM, two buffers
//   P = exp2(S c - m)      eight warps, two threads per row of 64 columns each; 16-bit P goes back over S in TMEM
//   O[128 x D] += P V      tcgen05.mma, P from TMEM, V as it lies in the cache (rows of keys: the MN-major form)
// TMEM: O takes D columns, S 2 x 128: 512 at D = 256.  The order on the tensor pipe is S(0) S(1) | O(0) S(2) | O(1) S(3)
// ...: while the warps turn S(j+1) into P(j+1), the pipe does O(j) and S(j+2).
//
// The running maximum is moved only when a row's grows by more than 2^8: weights then stay below that (sums are fp32), and
// O in TMEM is rescaled a few times per unit instead of once per tile.  An fp16 weight has no bits below 2^-24: with the
// largest at 1 a long context's many small ones would be lost together, so the maximum is set to 2^7, which with the 2^8
// stays within fp16's 65,504 (moving it at 2^4 and setting it to 2^11 costs 2.6% of 8,192 tokens' 764 us).
// Weights meet the values in 16 bits, as the tensor cores take them, and a row's sum takes them so too: what the rounding
// does to a weight it then does to numerator and denominator alike, and equal values come back as they are.  Summed as they
// were before it, a row that one key dominates is off by a rounding more: behind the first tile that key's weight is any
// number.  The sum by the mixed addition cost 0.6% of 8,192 tokens' time (1.6% with the weights widened first), 2% of a
// verify step's.  A second product with what the rounding leaves out would bring the error down from 1.2 to 1.4 times that
// of fp32 weights, for 1,024 more of a tile's 2,048 clocks of products.
//
// Keys and values come by TMA straight from their pages, through a ring and a producer warp of their own each: a slot of
// 16 KB is 128 keys x 64 columns, or the values of 8192 / D keys.  A copy costs its warp about 60 clocks however small it
// is, and a slot's barriers as much again; one warp for both was the bound of the whole kernel (3,700 clocks per tile).
// Tiles on the edge of what the rows see are masked, and their values are looked at first by a warp of its own: what no
// row sees becomes zero, and an infinity or a NaN that some rows see and others do not (0 x infinity is NaN) sends the
// unit through a plain fp32 loop at the end.
//
// The tensor cores cut a running sum off where they would have to round it: after the 65,536 products of a million keys O
// was too small by 0.7%.  So every 64 tiles (fp16; 512 in bf16) the softmax's warps fold O into fp32 sums in the workspace,
// by additions that round, and O starts again; at the end what was folded comes back.  The place for that, 128 KB, is lent to
// the thread block.  The loop over tiles is in two levels for it: with the fold inside, tiles took 2 to 6% longer.
//
// When there are fewer units than SMs the keys of a unit are split over a cluster of 2 to 8 thread blocks, whose sums meet
// in distributed shared memory.
//
// What bounds it: keys and values from L2, 512 D bytes per tile and SM.  At D = 256 the ring holds 1.25 tiles and 42 bytes
// per clock and SM arrive (more than 10 TB/s over the chip); a tile takes some 3,000 clocks, 2,048 of them products.
// Measured on B200 (fp16 and bf16 alike), in bursts of 20 calls: a prompt of 8,192 tokens, 24 query heads on 4 key heads of
// 256, 751 us = 1,098 TFLOP/s of 1,677; four prompts of up to 4,001 tokens behind a window of 1,024, 434 us; 511 tokens behind
// 30,001, 16 heads on 4 of 128, 162 us = 782 TFLOP/s; four tokens of six users behind a window of 4,096, 32 us.  Called for
// seconds, under the power cap, the first takes 858 us and the third 169.
#include "q4b_cache.cuh"
#include "q4b_tc.cuh"

#include <cooperative_groups.h>
#include <cmath>
#include <type_traits>

namespace q4b {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kPromptThreads = 384;   // keys, MMA, values, one that looks at values, eight of the softmax
constexpr uint32_t kTileRowsQ = 128, kTileKeys = 128;
constexpr uint32_t kMostSplits = 8;
constexpr float kRescaleAt = 8.0f;         // powers of two
template <typename T> constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;

constexpr uint32_t kSlotBytes = 16384;
template <int D> struct Shape {
    static constexpr uint32_t parts = D / 64;                       // ring slots of a tile of keys, or of values
    static constexpr uint32_t slots = D == 256 ? 5 : 6;             // of either ring
    static constexpr uint32_t v_rows = kTileKeys / parts;           // a slot is 128 keys x 64 columns, or v_rows values x D
    static constexpr uint32_t query = kTileRowsQ * D * 2;
};
constexpr uint32_t kMiscBytes = 2048;

struct PromptParams {
    CUtensorMap k_map, v_map;   // [D / 64][pages x kv_heads x page_tokens][64]
    AttentionArgs a;
    uint32_t units, splits, k_shift, v_shift;  // boxes of 1 << k_shift, 1 << v_shift tokens
    uint32_t sms;
};

// A place for folded sums: one per SM, and a thread block that needs one has an SM to itself, so one of them is free --
// most likely that of this SM's number.  kNoPlace when none is.
constexpr uint32_t kNoPlace = 0xffffffffu;
__device__ inline uint32_t take_place(uint32_t *owners, uint32_t places) {
    uint32_t sm;
    asm volatile("mov.u32 %0, %%smid;" : "=r"(sm));
    for (uint32_t i = 0; i < 4 * places; ++i) {
        const uint32_t at = (sm + i) % places;
        if (atomicCAS(owners + at, 0u, 1u) == 0) {
            __threadfence();
            return at;
        }
    }
    return kNoPlace;
}

__device__ inline float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ inline uint32_t pack2(float low, float high);
template <> __device__ inline uint32_t pack2<__half>(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ inline uint32_t pack2<__nv_bfloat16>(float low, float high) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ inline float wide(__half x) { return __half2float(x); }
__device__ inline float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ inline float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two floats of neighbouring registers, for the instructions that take both
__device__ inline uint64_t two(float low, float high) {
    uint64_t both;
    asm("mov.b64 %0, {%1, %2};" : "=l"(both) : "f"(low), "f"(high));
    return both;
}
__device__ inline float2 apart(uint64_t both) {
    float2 x;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x.x), "=f"(x.y) : "l"(both));
    return x;
}
__device__ inline uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// a sum and a 16-bit weight, by one instruction
__device__ inline float plus_weight(float sum, __half weight) {
    float all;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(all) : "h"(__half_as_ushort(weight)), "f"(sum));
    return all;
}
__device__ inline float plus_weight(float sum, __nv_bfloat16 weight) {
    float all;
    asm("add.rn.f32.bf16 %0, %1, %2;" : "=f"(all) : "h"(__bfloat16_as_ushort(weight)), "f"(sum));
    return all;
}
// the halves of a word, each to a sum of its own
template <typename T> __device__ inline void plus_weights(float &low_sum, float &high_sum, uint32_t word) {
    const T *const pair = reinterpret_cast<const T *>(&word);
    low_sum = plus_weight(low_sum, pair[0]);
    high_sum = plus_weight(high_sum, pair[1]);
}
__device__ inline void pair_barrier(uint32_t id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// (token, query head of the group) of every `step`th row, without a division for each
struct RowWalk {
    uint32_t token, member, group, step_tokens, step_members;
    __device__ inline RowWalk(uint32_t flat, uint32_t of, uint32_t step)
        : token(flat / of), member(flat % of), group(of), step_tokens(step / of), step_members(step % of) {}
    __device__ inline void next() {
        token += step_tokens;
        member += step_members;
        if (member >= group) {
            member -= group;
            ++token;
        }
    }
};

// What a thread block works on.
struct Unit {
    SequenceRows rows;
    uint32_t sequence, head, row0, count;  // query rows [row0, row0 + count) of the sequence's count x group
    Groups tiles;                          // of 128 keys
    uint32_t first, size;                  // this thread block's share of them
    int64_t least, most, place0;           // places of the first and the last row; of the sequence's first new token
    __device__ inline uint32_t key(uint32_t j) const { return tiles.at(first + j) * kTileKeys; }
    __device__ inline bool clear(const AttentionArgs &a, uint32_t key0) const { return every(a, key0, kTileKeys); }
    // does any row see one of the keys [key, key + count), do all rows see all of them?
    __device__ inline bool any(const AttentionArgs &a, uint32_t key, uint32_t count) const {
        return (int64_t)key <= most && (a.window == 0 || key < a.sinks || (int64_t)key + count - 1 > least - (int64_t)a.window);
    }
    __device__ inline bool every(const AttentionArgs &a, uint32_t key, uint32_t count) const {
        return (int64_t)key + count - 1 <= least &&
               (a.window == 0 || (int64_t)key > most - (int64_t)a.window || (uint64_t)key + count <= a.sinks);
    }
};

// A row's sums in TMEM and, times the factor, what was folded of them before (nothing the first time): into the folded ones,
// or back into TMEM.  Not inlined: it is rare.
__device__ __noinline__ void fold_columns(uint32_t columns, uint32_t count, float *folded, float factor, bool first, bool back) {
#pragma unroll 1
    for (uint32_t column = 0; column < count; column += 32) {
        uint32_t o[32];
        float *const at = folded + (size_t)column * kTileRowsQ;
        tc_load_32(columns + column, o);
        tc_wait_loaded(o);
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!first) o[i] = __float_as_uint(fmaf(__ldcg(at + i * kTileRowsQ), factor, __uint_as_float(o[i])));
        if (back) {
            tc_store_32(columns + column, o);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) __stcg(at + i * kTileRowsQ, __uint_as_float(o[i]));
        }
    }
    if (back) tc_wait_store();
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
prompt_kernel(const __grid_constant__ PromptParams p) {
    using S = Shape<D>;
    extern __shared__ __align__(1024) uint8_t prompt_smem[];
    uint8_t *const base = prompt_smem + ((1024u - (tc_smem_u32(prompt_smem) & 1023u)) & 1023u);
    uint8_t *const query = base, *const ring = base + S::query;
    uint8_t *const misc = ring + 2 * S::slots * kSlotBytes;
    float *const exchange = reinterpret_cast<float *>(misc);                    // [2][128]
    uint64_t *const bars = reinterpret_cast<uint64_t *>(misc + 1024);
    uint32_t *const words = reinterpret_cast<uint32_t *>(bars + 4 * S::slots + 8);  // TMEM address, poison flag, place of folds
    const uint32_t k_full0 = tc_smem_u32(bars), k_empty0 = k_full0 + 8 * S::slots, v_full0 = k_empty0 + 8 * S::slots,
                   v_empty0 = v_full0 + 8 * S::slots;
    const uint32_t k_ring = tc_smem_u32(ring), v_ring = k_ring + S::slots * kSlotBytes;
    const uint32_t q_full = v_empty0 + 8 * S::slots, s_full0 = q_full + 8, p_full0 = s_full0 + 16, o_done = p_full0 + 16,
                   v_look = o_done + 8, v_ready = v_look + 8;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttentionArgs &a = p.a;
    const uint32_t rank = blockIdx.x % p.splits;

    // ---- which rows ---- (the last tiles of a sequence see most: they go first)
    Unit u;
    {
        const uint32_t index = p.units - 1 - blockIdx.x / p.splits;
        u.head = index % a.cache.kv_heads;
        const uint32_t tile = index / a.cache.kv_heads;
        uint32_t before = 0;
        bool found = false;
        // the first block looks at the sequences behind its own too: somebody has to tell of each one's mistakes
        for (uint32_t s0 = 0; s0 < a.batch.sequences && (!found || blockIdx.x == 0); s0 += 32) {
            uint32_t own = 0;
            if (s0 + lane < a.batch.sequences)
                own = ceil_div(sequence_rows(a.batch, a.cache.page_tokens, s0 + lane, a.status).count * a.group, kTileRowsQ);
            uint32_t inclusive = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, inclusive, d);
                if (lane >= (uint32_t)d) inclusive += y;
            }
            const uint32_t passed = __ballot_sync(0xffffffffu, before + inclusive > tile);
            if (passed != 0 && !found) {
                const int at = __ffs(passed) - 1;
                u.sequence = s0 + at;
                u.row0 = (tile - before - __shfl_sync(0xffffffffu, inclusive - own, at)) * kTileRowsQ;
                found = true;
            }
            before += __shfl_sync(0xffffffffu, inclusive, 31);
        }
        if (!found) return;  // the grid is made for the most tiles that the host's numbers allow; the whole cluster leaves
        u.rows = sequence_rows(a.batch, a.cache.page_tokens, u.sequence, a.status);
        u.count = min(kTileRowsQ, u.rows.count * a.group - u.row0);
        const uint32_t token0 = u.row0 / a.group, token1 = (u.row0 + u.count - 1) / a.group;
        u.tiles = groups_of<kTileKeys>(u.rows, token0, token1, a.window, a.sinks);
        u.place0 = (int64_t)u.rows.length - u.rows.count;
        u.least = u.place0 + token0;
        u.most = u.place0 + token1;
        const uint32_t all = u.tiles.sink + (u.tiles.end - u.tiles.first);
        u.first = (uint32_t)((uint64_t)all * rank / p.splits);
        u.size = (uint32_t)((uint64_t)all * (rank + 1) / p.splits) - u.first;
    }
    const uint32_t n = u.size;
    constexpr uint32_t kFold = (std::is_same<T, __half>::value ? kFoldStepsF16 : kFoldStepsBF16) * 16 / kTileKeys;  // tiles
    const bool folds = n > kFold;
    const uint32_t *const table = a.batch.table + (size_t)u.sequence * a.batch.table_stride;

    uint32_t own_place = kNoPlace;  // the first thread's to give back
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < 4 * S::slots; ++s) tc_mbar_init(k_full0 + 8 * s, 1);  // full and empty of both rings
        tc_mbar_init(q_full, kPromptThreads - 96);
        for (uint32_t b = 0; b < 2; ++b) {
            tc_mbar_init(s_full0 + 8 * b, 1);
            tc_mbar_init(p_full0 + 8 * b, 8);
        }
        tc_mbar_init(o_done, 1);
        tc_mbar_init(v_look, 1);
        tc_mbar_init(v_ready, 32);
        words[1] = 0;
        if (folds) {
            own_place = take_place(a.arrivals + p.sms, p.sms);
            if (own_place == kNoPlace) atomicExch(a.status, 0x86u);  // cannot be; the results are then not to be used
            words[2] = own_place == kNoPlace ? 0 : own_place;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(tc_smem_u32(words)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[0], tmem_o = tmem, tmem_s = tmem + 256;
    bool ok = true;

    if (warp == 0 || warp == 2) {
        // ---- producers: warp 0 the keys, warp 2 the values ----
        // A box ends with its page.  Page numbers are fetched, one box per lane, a whole tile ahead of their use.
        const bool keys = warp == 0;
        const uint32_t keys_end = u.rows.length, shift = keys ? p.k_shift : p.v_shift;
        const uint32_t rows = keys ? kTileKeys : S::v_rows, box_bytes = (keys ? 128u : 128u * S::parts) << shift;
        const uint32_t full0 = keys ? k_full0 : v_full0, empty0 = keys ? k_empty0 : v_empty0, to0 = keys ? k_ring : v_ring;
        const CUtensorMap *const map = keys ? &p.k_map : &p.v_map;
        const uint32_t my_token = min(lane << shift, kTileKeys - 1);
        // the token of this lane's box; one behind the sequence's end counts as the last one (its box is not fetched)
        auto token_of = [&](uint32_t j) { return min(u.key(j) + my_token, keys_end - 1); };
        auto page_of = [&](uint32_t token) { return __ldg(table + (token >> a.cache.page_shift)); };
        const bool leader = tc_leader();
        uint32_t item = 0, slot = 0, lap = 0;
        uint32_t token = n > 0 ? token_of(0) : 0, page = n > 0 ? page_of(token) : 0;
        for (uint32_t j = 0; j < n && ok; ++j) {
            // the boxes that hold something which some row sees, a bit each: on the edges of a window most do not
            const uint32_t wanted = __ballot_sync(0xffffffffu, (lane << shift) < kTileKeys && u.key(j) + my_token < keys_end &&
                                                                   u.any(a, u.key(j) + my_token, 1u << shift));
            if (page >= a.cache.pages) {  // never followed: the pool's first page stands in for it
                // the entry of a box that is not fetched may be anything: pages behind a window are dealt anew
                if (wanted >> lane & 1u) report(a.status, kBadPage);
                page = 0;
            }
            const int line = (int)((page * a.cache.kv_heads + u.head) * a.cache.page_tokens + (token & (a.cache.page_tokens - 1)));
            if (j + 1 < n) {
                token = token_of(j + 1);
                page = page_of(token);
            }
#pragma unroll
            for (uint32_t part = 0; part < S::parts; ++part) {
                if (lap > 0 && !tc_warp_wait(empty0 + 8 * slot, (lap - 1) & 1)) {
                    ok = false;
                    break;
                }
                const uint32_t first = keys ? 0 : part * S::v_rows >> shift, boxes = rows >> shift;
                const uint32_t here = wanted >> first & ((1u << boxes) - 1);
                const uint32_t bar = full0 + 8 * slot;
                uint32_t to = to0 + slot * kSlotBytes;
                if (leader) tc_mbar_expect_tx(bar, __popc(here) * box_bytes);
                __syncwarp();
                for (uint32_t box = 0; box < boxes; ++box, to += box_bytes) {
                    const int y = __shfl_sync(0xffffffffu, line, first + box);
                    if (here >> box & 1u) tc_tensor_copy_3d_by(leader, to, map, 0, y, keys ? (int)part : 0, bar);
                }
                ++item;
                if (++slot == S::slots) {
                    slot = 0;
                    ++lap;
                }
            }
        }
        if (!ok) {
            if (leader) atomicExch(a.status, keys ? 0x81u : 0x85u);
            // copies already issued land before the shared memory is released
            for (uint32_t back = 0; back < S::slots && back < item; ++back) {
                const uint32_t i = item - 1 - back;
                tc_wait(full0 + 8 * (i % S::slots), (i / S::slots) & 1);
            }
        }
    } else if (warp == 1) {
        // ---- MMA issuer ----
        if (n > 0) {
            constexpr uint32_t format = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t s_idesc = (1u << 4) | format | ((kTileKeys >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t o_idesc = (1u << 4) | format | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
            // rows of 128 bytes, eight of them 1024 bytes (stride field), swizzled; for V the 64-column chunks of a box
            // follow one another at the leading field's distance
            constexpr uint64_t k_desc = ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
            const uint64_t v_desc = ((uint64_t)((128u << p.v_shift) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
                                    ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
            // a descriptor takes the low 18 bits of an address: in a cluster those above name the thread block
            auto at = [](uint32_t address) { return (uint64_t)((address & 0x3ffffu) >> 4); };
            const bool leader = tc_leader();
            const uint32_t to_s = __shfl_sync(0xffffffffu, tmem_s, 0), to_o = __shfl_sync(0xffffffffu, tmem_o, 0);
            const uint64_t rows0 = k_desc + at(tc_smem_u32(query));
            uint32_t v_step[S::v_rows / 16];  // where a slot's steps of 16 values lie, in units of 16 bytes as descriptors count
#pragma unroll
            for (uint32_t k = 0; k < S::v_rows / 16; ++k)
                v_step[k] = ((k * 16 >> p.v_shift << p.v_shift) * S::parts + (k * 16 & ((1u << p.v_shift) - 1))) * 8;
            uint32_t k_slot = 0, k_lap = 0, v_slot = 0, v_lap = 0, looked = 0, begun = 0;
            auto advance = [](uint32_t &slot, uint32_t &lap) {
                if (++slot == S::slots) {
                    slot = 0;
                    ++lap;
                }
            };
            auto scores = [&](uint32_t j) {
#pragma unroll
                for (uint32_t part = 0; part < S::parts; ++part) {
                    if (!tc_warp_wait(k_full0 + 8 * k_slot, k_lap & 1)) return false;
                    tc_fence_after();
                    const uint64_t keys = k_desc + at(k_ring + k_slot * kSlotBytes), rows = rows0 + part * (kTileRowsQ * 128 >> 4);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        tc_mma_shared_by(leader, to_s + (j & 1) * 128, rows + k * 2, keys + k * 2, s_idesc,
                                         part > 0 || k > 0 ? 1u : 0u);
                    tc_commit_by(leader, k_empty0 + 8 * k_slot);
                    advance(k_slot, k_lap);
                }
                tc_commit_by(leader, s_full0 + 8 * (j & 1));
                return true;
            };
            ok = tc_warp_wait(q_full, 0);
            tc_fence_after();
            if (ok) ok = scores(0);
            if (ok && n > 1) ok = scores(1);
            for (uint32_t j = 0; j < n && ok; ++j) {
                // the values came long ago: their waits (100 clocks each) are over before the weights are there
                uint32_t slot = v_slot, lap = v_lap;
                if (j % kFold == 0) begun = 0;  // what O holds has been folded before these weights were handed over
#pragma unroll
                for (uint32_t part = 0; part < S::parts; ++part) {
                    if (ok) ok = tc_warp_wait(v_full0 + 8 * slot, lap & 1);
                    advance(slot, lap);
                }
                if (!ok) break;
                // a masked tile's values are handed to the warp that looks at them and handed back: a strict exchange,
                // so neither side can miss a round of a barrier that the other is already past
                const bool edge = !u.clear(a, u.key(j));
                uint32_t steps = 0xffu;  // of 16 keys that some row sees
                if (edge) {
                    steps = __ballot_sync(0xffffffffu, lane < kTileKeys / 16 && u.any(a, u.key(j) + lane * 16, 16));
                    if (leader) tc_mbar_arrive(v_look);
                }
                ok = tc_warp_wait(p_full0 + 8 * (j & 1), (j >> 1) & 1);
                if (edge && ok) {
                    ok = tc_warp_wait(v_ready, looked & 1);
                    ++looked;
                }
                if (!ok) break;
                tc_fence_after();
                const uint32_t weights = to_s + (j & 1) * 128;
#pragma unroll
                for (uint32_t part = 0; part < S::parts; ++part) {
                    constexpr uint32_t kSteps = S::v_rows / 16;
                    const uint64_t values = v_desc + at(v_ring + v_slot * kSlotBytes);
                    if (steps == 0xffu) {
#pragma unroll
                        for (uint32_t k = 0; k < kSteps; ++k)
                            tc_mma_by(leader, to_o, weights + (part * kSteps + k) * 8, values + v_step[k], o_idesc,
                                      part > 0 || k > 0 ? 1u : begun);
                    } else {
#pragma unroll
                        for (uint32_t k = 0; k < kSteps; ++k) {
                            // keys that no row sees are left out, with whatever their place in the slot holds
                            if (!(steps >> (part * kSteps + k) & 1u)) continue;
                            tc_mma_by(leader, to_o, weights + (part * kSteps + k) * 8, values + v_step[k], o_idesc, begun);
                            begun = 1;
                        }
                    }
                    tc_commit_by(leader, v_empty0 + 8 * v_slot);
                    advance(v_slot, v_lap);
                }
                begun = 1;
                tc_commit_by(leader, o_done);
                if (j + 2 < n) ok = scores(j + 2);
            }
            if (!ok && leader) atomicExch(a.status, 0x82u);
        }
    } else {
        // ---- query rows into shared memory, swizzled; a negative scale turns their sign, scale 0 makes them zero ----
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, hold = a.scale == 0.0f ? 0u : 0xffffffffu;
        constexpr uint32_t kLoaders = kPromptThreads - 96, kAtOnce = 8;  // pieces of 16 bytes on their way per thread
        constexpr uint32_t kStep = kLoaders / (D / 8);                   // rows between a thread's pieces, all in one column
        static_assert(kLoaders % (D / 8) == 0, "whole rows per round");
        uint32_t row = (threadIdx.x - 96) / (D / 8);
        const uint32_t piece = (threadIdx.x - 96) % (D / 8);
        RowWalk at(u.row0 + row, a.group, kStep);
        const T *const from = static_cast<const T *>(a.q) + (size_t)u.rows.begin * a.ldq + (size_t)u.head * a.group * D + piece * 8;
#pragma unroll 1
        for (; row < kTileRowsQ; row += kStep * kAtOnce) {
            uint4 value[kAtOnce];
#pragma unroll
            for (uint32_t e = 0; e < kAtOnce; ++e, at.next()) {
                value[e] = make_uint4(0, 0, 0, 0);
                if (row + e * kStep < u.count)
                    value[e] = *reinterpret_cast<const uint4 *>(from + (size_t)at.token * a.ldq + at.member * D);
            }
#pragma unroll
            for (uint32_t e = 0; e < kAtOnce; ++e) {
                const uint32_t r = row + e * kStep;
                if (r < kTileRowsQ)
                    *reinterpret_cast<uint4 *>(query + (piece >> 3) * (kTileRowsQ * 128) + r * 128 + (((piece & 7) ^ (r & 7)) * 16)) =
                        make_uint4((value[e].x ^ flip) & hold, (value[e].y ^ flip) & hold, (value[e].z ^ flip) & hold,
                                   (value[e].w ^ flip) & hold);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_mbar_arrive(q_full);

        if (warp == 3) {
            // ---- the values of masked tiles, in the steps of 16 keys that some rows see and others do not: zeros where no
            // row sees them, no infinity where only some do ----
            constexpr uint32_t exponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            constexpr uint32_t both = exponent | exponent << 16, low = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
            uint32_t looked = 0, passed = 0;
            for (uint32_t j = 0; j < n && ok; ++j) {
                const uint32_t key0 = u.key(j);
                if (u.clear(a, key0)) {
                    ++passed;
                    continue;
                }
                // a bit per key: nobody sees it, some do and some do not; four words of 32 keys
                uint32_t nobody[4], some[4];
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    const bool any = u.any(a, key0 + 32 * w + lane, 1), every = u.every(a, key0 + 32 * w + lane, 1);
                    nobody[w] = __ballot_sync(0xffffffffu, !any);
                    some[w] = __ballot_sync(0xffffffffu, any && !every);
                }
                // the tiles in between may take longer than one wait bears: 2^15 tiles of up to 120,000 clocks for each
                for (uint32_t patience = passed >> 15;; --patience) {
                    ok = tc_warp_wait(v_look, looked & 1);
                    if (ok || patience == 0) break;
                }
                if (!ok) break;
                passed = 0;
                ++looked;
                uint32_t strange = 0;
#pragma unroll
                for (uint32_t g = 0; g < kTileKeys / 16; ++g) {
                    const uint32_t part = g * 16 / S::v_rows, k = g - part * (S::v_rows / 16);
                    const uint32_t item = j * S::parts + part, slot = item % S::slots;
                    const uint32_t none = nobody[g >> 1] >> (g & 1) * 16 & 0xffffu, mixed = some[g >> 1] >> (g & 1) * 16 & 0xffffu;
                    if (none == 0xffffu || (none | mixed) == 0) continue;  // not multiplied, or seen by all
                    ok = ok && tc_warp_wait(v_full0 + 8 * slot, (item / S::slots) & 1);  // it is: acquires
                    // [box][chunk][token of the box][8 cells]
                    uint4 *const cells = reinterpret_cast<uint4 *>(ring + (S::slots + slot) * kSlotBytes) +
                                         ((k * 16 >> p.v_shift << p.v_shift) * S::parts + (k * 16 & ((1u << p.v_shift) - 1))) * 8 + lane;
                    // four tokens of a chunk at a time, all on their way at once
                    uint4 cell[4 * S::parts];
#pragma unroll
                    for (uint32_t i = 0; i < 4 * S::parts; ++i) cell[i] = cells[(i >> 2 << p.v_shift) * 8 + (i & 3) * 32];
                    uint32_t found[4] = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t i = 0; i < 4 * S::parts; ++i) {
                        // an exponent of all ones carries into the bit above it
                        const uint4 &c = cell[i];
                        found[i & 3] |= ((c.x & both) + low) | ((c.y & both) + low) | ((c.z & both) + low) | ((c.w & both) + low);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t token = i * 4 + (lane >> 3);
                        strange |= mixed >> token & 1u ? found[i] & 0x80008000u : 0;
                        if (none >> token & 1u) {
#pragma unroll
                            for (uint32_t chunk = 0; chunk < S::parts; ++chunk)
                                cells[(chunk << p.v_shift) * 8 + i * 32] = make_uint4(0, 0, 0, 0);
                        }
                    }
                }
                if (strange != 0) words[1] = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_mbar_arrive(v_ready);
            }
            if (!ok && lane == 0) atomicExch(a.status, 0x83u);
        } else {
            // ---- softmax ----
            const uint32_t quad = warp & 3, half = (warp - 4) >> 2, row = quad * 32 + lane;
            const uint32_t lanes = (quad * 32) << 16;
            const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896341f;
            const bool active = quad * 32 < u.count;  // otherwise none of the warp's rows is asked for
            const int64_t place = row < u.count ? u.place0 + (u.row0 + row) / a.group : -1;
            float top = -INFINITY, total = 0.0f;
            float folded_top = -INFINITY, folded_total = 0.0f;
            auto fold = [&](uint32_t next, bool back) {  // O holds the sums of the tiles before `next`
                if (ok && !tc_wait(o_done, (next - 1) & 1)) ok = false;
                if (!ok || !active) return;
                // [columns][128 rows]: every thread reads what it wrote
                float *const folded = a.folds + (size_t)words[2] * kFoldFloats + (size_t)half * (D / 2) * kTileRowsQ + row;
                const float factor = folded_top == -INFINITY ? 0.0f : exp2_of(folded_top - top);
                tc_fence_after();
                fold_columns(tmem_o + lanes + half * (D / 2), D / 2, folded, factor, next == kFold, back);
                folded_total = fmaf(folded_total, factor, total);
                folded_top = top;
                total = 0.0f;
            };
            for (uint32_t j = 0, stop = min(n, kFold);;) {
                for (; j < stop; ++j) {
                    // found out while S(j) is on its way: are there columns to hide, and which
                    const uint32_t key0 = u.key(j);
                    const bool edge = !u.clear(a, key0);
                    if (ok && !tc_wait(s_full0 + 8 * (j & 1), (j >> 1) & 1)) ok = false;
                    tc_fence_after();
                    const uint32_t s_columns = tmem_s + (j & 1) * 128 + lanes;
                    if (active) {
                        uint32_t raw[2][32];
                        tc_load_32(s_columns + half * 64, raw[0]);
                        tc_load_32(s_columns + half * 64 + 32, raw[1]);
                        tc_wait_loaded(raw[0]);
                        tc_wait_loaded(raw[1]);
                        if (edge) {
                            // visible columns: below `behind`, and from `from` on or below `sink`
                            const int64_t first = (int64_t)key0 + half * 64;
                            const int32_t behind = (int32_t)max((int64_t)0, min((int64_t)64, place + 1 - first));
                            const int32_t from = a.window == 0 ? 0 : (int32_t)max((int64_t)0, min((int64_t)64, place - (int64_t)a.window + 1 - first));
                            const int32_t sink = (int32_t)max((int64_t)0, min((int64_t)64, (int64_t)a.sinks - first));
#pragma unroll
                            for (int i = 0; i < 64; ++i) {
                                if (!(i < behind && (i >= from || i < sink))) raw[i >> 5][i & 31] = 0xff800000u;  // -infinity
                            }
                        }
                        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 64; i += 2)
                            most[i >> 1 & 3] = max3(most[i >> 1 & 3], __uint_as_float(raw[i >> 5][i & 31]), __uint_as_float(raw[i >> 5][i + 1 & 31]));
                        float high = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                        pair_barrier(5 + quad);  // the other half has read what it was told last time
                        exchange[half * 128 + row] = high;
                        pair_barrier(1 + quad);
                        high = fmaxf(high, exchange[(half ^ 1) * 128 + row]) * c - kLift<T>;
                        const bool grow = high > top + kRescaleAt || (top == -INFINITY && high > -INFINITY);
                        bool waited = j == 0;
                        if (__any_sync(0xffffffffu, grow)) {
                            const float factor = grow ? exp2_of(top - high) : 1.0f;
                            if (grow) top = high;
                            total *= factor;
                            if (j > 0) {
                                if (ok && !tc_wait(o_done, (j - 1) & 1)) ok = false;
                                waited = true;
                                tc_fence_after();
#pragma unroll 1
                                for (uint32_t column = half * (D / 2); column < (half + 1) * (D / 2); column += 32) {
                                    uint32_t o[32];
                                    tc_load_32(tmem_o + lanes + column, o);
                                    tc_wait_loaded(o);
#pragma unroll
                                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                                    tc_store_32(tmem_o + lanes + column, o);
                                }
                            }
                        }
                        const float minus = top == -INFINITY ? 0.0f : -top;
                        uint32_t weights[32];
                        const uint64_t factors = two(c, c), offsets = two(minus, minus);
                        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float2 x = apart(fma2(two(__uint_as_float(raw[i >> 4][(2 * i) & 31]), __uint_as_float(raw[i >> 4][(2 * i + 1) & 31])),
                                                  factors, offsets));
                            weights[i] = pack2<T>(exp2_of(x.x), exp2_of(x.y));
                            plus_weights<T>(sum[2 * (i & 1)], sum[2 * (i & 1) + 1], weights[i]);
                        }
                        tc_store_32(s_columns + half * 32, weights);
                        tc_wait_store();
                        // O(j - 1) is complete long before P(j) is needed; every warp sees every round of its barrier
                        if (!waited && ok && !tc_wait(o_done, (j - 1) & 1)) ok = false;
                        total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    } else if (j > 0 && ok && !tc_wait(o_done, (j - 1) & 1)) {
                        ok = false;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc_mbar_arrive(p_full0 + 8 * (j & 1));
                }
                if (j == n) break;
                fold(j, false);
                stop = min(n, j + kFold);
            }
            if (n > 0 && ok && !tc_wait(o_done, (n - 1) & 1)) ok = false;
            if (!ok && lane == 0) atomicExch(a.status, 0x84u);
            tc_fence_after();
            if (folds) {  // what was folded comes back into O
                fold(n, true);
                total = folded_total;
            }
            if (active) {
                pair_barrier(5 + quad);
                exchange[half * 128 + row] = total;
                pair_barrier(1 + quad);
                total = exchange[row] + exchange[128 + row];
            }
            // ---- output, or sums for the cluster ----
            if (p.splits == 1) {
                // through shared memory (the ring is done with): a row leaves in whole lines, not 64 bytes at a time per thread
                const float over = total == 0.0f ? 0.0f : 1.0f / total;
                if (active) {
                    uint4 *const staged = reinterpret_cast<uint4 *>(ring);  // [128][D / 8], pieces turned by the row
#pragma unroll 1
                    for (uint32_t column = half * (D / 2); column < (half + 1) * (D / 2); column += 32) {
                        uint32_t o[32];
                        if (n > 0) {
                            tc_load_32(tmem_o + lanes + column, o);
                            tc_wait_loaded(o);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint4 packed;
                            uint32_t *const w = reinterpret_cast<uint32_t *>(&packed);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                w[k] = pack2<T>(__uint_as_float(o[i + 2 * k]) * over, __uint_as_float(o[i + 2 * k + 1]) * over);
                            staged[row * (D / 8) + (((column + i) >> 3) ^ (row & 7))] = packed;
                        }
                    }
                    pair_barrier(1 + quad);
                    // the pair's 32 rows, 64 lanes over their pieces
                    constexpr uint32_t kRowsAtOnce = 64 / (D / 8);
                    const uint32_t lane64 = half * 32 + lane, out_piece = lane64 % (D / 8), out_row0 = quad * 32 + lane64 / (D / 8);
                    RowWalk out_at(u.row0 + out_row0, a.group, kRowsAtOnce);
                    T *const to = static_cast<T *>(a.out) + (size_t)u.rows.begin * a.ldo + (size_t)u.head * a.group * D + out_piece * 8;
#pragma unroll 4
                    for (uint32_t r = 0; r < 32 / kRowsAtOnce; ++r, out_at.next()) {
                        const uint32_t out_row = out_row0 + r * kRowsAtOnce;
                        if (out_row < u.count)
                            *reinterpret_cast<uint4 *>(to + (size_t)out_at.token * a.ldo + out_at.member * D) =
                                staged[out_row * (D / 8) + (out_piece ^ (out_row & 7))];
                    }
                }
            } else if (active) {
                float *const sums = reinterpret_cast<float *>(ring);  // [128][D], pieces of four turned by the row
#pragma unroll 1
                for (uint32_t column = half * (D / 2); column < (half + 1) * (D / 2); column += 32) {
                    uint32_t o[32];
                    if (n > 0) {
                        tc_load_32(tmem_o + lanes + column, o);
                        tc_wait_loaded(o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        *reinterpret_cast<uint4 *>(sums + row * D + (((column + i) / 4) ^ (row & 7)) * 4) =
                            make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                pair_barrier(5 + quad);  // both have read the totals
                if (half == 0) {
                    exchange[row] = top;
                    exchange[128 + row] = total;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (own_place != kNoPlace) {
        __threadfence();
        atomicExch(a.arrivals + p.sms + own_place, 0u);
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }

    // ---- a unit whose edge tiles hold infinities or NaN: again, row by row in fp32, over what each row sees ----
    if (words[1] != 0) {
        float *const sums = reinterpret_cast<float *>(ring);
        for (uint32_t row = warp; row < u.count; row += kPromptThreads / 32) {
            const uint32_t flat = u.row0 + row;
            const int64_t place = u.place0 + flat / a.group;
            const T *const q = static_cast<const T *>(a.q) + (size_t)(u.rows.begin + flat / a.group) * a.ldq +
                               (size_t)(u.head * a.group + flat % a.group) * D;
            float mine[D / 32], sum[D / 32], top = -INFINITY, total = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                mine[i] = wide(q[i * 32 + lane]) * a.scale * 1.44269504088896341f;
                sum[i] = 0.0f;
            }
            for (uint32_t j = 0; j < n; ++j) {
                float tile_sum[D / 32], tile_top = -INFINITY, tile_total = 0.0f;  // no long chain of additions
#pragma unroll
                for (int i = 0; i < D / 32; ++i) tile_sum[i] = 0.0f;
                for (uint32_t key = u.key(j); key < u.key(j) + kTileKeys; ++key) {
                    if ((int64_t)key > place || !(a.window == 0 || (int64_t)key > place - (int64_t)a.window || key < a.sinks)) continue;
                    const uint32_t page = __ldg(table + (key >> a.cache.page_shift));
                    if (page >= a.cache.pages) continue;
                    const size_t line = (((size_t)page * a.cache.kv_heads + u.head) * a.cache.page_tokens +
                                         (key & (a.cache.page_tokens - 1))) * D;
                    float score = 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) score += mine[i] * wide(static_cast<const T *>(a.cache.keys)[line + i * 32 + lane]);
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) score += __shfl_xor_sync(0xffffffffu, score, d);
                    const float high = fmaxf(tile_top, score);
                    const float minus = high == -INFINITY ? 0.0f : high;
                    const float keep = exp2_of(tile_top - minus), weight = exp2_of(score - minus);
                    tile_top = high;
                    tile_total = tile_total * keep + weight;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
                        tile_sum[i] = tile_sum[i] * keep + weight * wide(static_cast<const T *>(a.cache.values)[line + i * 32 + lane]);
                }
                const float high = fmaxf(top, tile_top);
                const float minus = high == -INFINITY ? 0.0f : high;
                // what saw nothing has sums of zero (or NaN)
                const float keep = top == -INFINITY ? 1.0f : exp2_of(top - minus), scale = tile_top == -INFINITY ? 1.0f : exp2_of(tile_top - minus);
                top = high;
                total = total * keep + tile_total * scale;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) sum[i] = sum[i] * keep + tile_sum[i] * scale;
            }
            if (p.splits == 1) {
                T *const to = static_cast<T *>(a.out) + (size_t)(u.rows.begin + flat / a.group) * a.ldo +
                              (size_t)(u.head * a.group + flat % a.group) * D;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint32_t word = pack2<T>(total == 0.0f ? 0.0f : sum[i] / total, 0.0f);
                    to[i * 32 + lane] = *reinterpret_cast<const T *>(&word);
                }
            } else {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint32_t column = i * 32 + lane;
                    sums[row * D + ((column / 4) ^ (row & 7)) * 4 + (column & 3)] = sum[i];
                }
                if (lane == 0) {
                    exchange[row] = top;
                    exchange[128 + row] = total;
                }
            }
        }
    }
    if (p.splits > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        // the rows are dealt to the cluster's warps; sums are added in the order of the split
        for (uint32_t row = rank + p.splits * warp; row < u.count; row += p.splits * (kPromptThreads / 32)) {
            float high = -INFINITY;
            for (uint32_t r = 0; r < p.splits; ++r) high = fmaxf(high, cluster.map_shared_rank(exchange, r)[row]);
            float total = 0.0f;
            float4 sum[D > 128 ? D / 128 : 1];
#pragma unroll
            for (int i = 0; i < (D > 128 ? D / 128 : 1); ++i) sum[i] = make_float4(0, 0, 0, 0);
            for (uint32_t r = 0; r < p.splits; ++r) {
                const float *const told = cluster.map_shared_rank(exchange, r);
                const float factor = told[row] == -INFINITY ? 1.0f : exp2_of(told[row] - high);
                total += told[128 + row] * factor;
                const float *const sums = reinterpret_cast<const float *>(cluster.map_shared_rank(ring, r)) + row * D;
#pragma unroll
                for (int i = 0; i < (D > 128 ? D / 128 : 1); ++i) {
                    if (D >= 128 || lane < D / 4) {
                        const float4 part = *reinterpret_cast<const float4 *>(sums + ((i * 32 + lane) ^ (row & 7)) * 4);
                        sum[i].x += part.x * factor; sum[i].y += part.y * factor;
                        sum[i].z += part.z * factor; sum[i].w += part.w * factor;
                    }
                }
            }
            const float over = total == 0.0f ? 0.0f : 1.0f / total;
            const uint32_t flat = u.row0 + row;
            T *const to = static_cast<T *>(a.out) + (size_t)(u.rows.begin + flat / a.group) * a.ldo +
                          (size_t)(u.head * a.group + flat % a.group) * D;
#pragma unroll
            for (int i = 0; i < (D > 128 ? D / 128 : 1); ++i) {
                if (D >= 128 || lane < D / 4)
                    *reinterpret_cast<uint2 *>(to + (i * 32 + lane) * 4) =
                        make_uint2(pack2<T>(sum[i].x * over, sum[i].y * over), pack2<T>(sum[i].z * over, sum[i].w * over));
            }
        }
        cluster.sync();  // the sums stay until everybody has read them
    }
}

template <typename T, int D>
cudaError_t launch_prompt_of(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    using S = Shape<D>;
    EncodeTiledFn encode = encode_tiled();
    if (encode == nullptr) return cudaErrorNotSupported;
    PromptParams p;
    p.a = args;
    // a box ends with its page or its slot; K's hold one chunk of 64 columns, V's all of them
    const uint32_t page = args.cache.page_tokens, v_rows = S::v_rows;
    const uint32_t k_tokens = page < kTileKeys ? page : kTileKeys, v_tokens = page < v_rows ? page : v_rows;
    p.k_shift = p.v_shift = 4;
    while ((1u << p.k_shift) < k_tokens) ++p.k_shift;
    while ((1u << p.v_shift) < v_tokens) ++p.v_shift;
    const cuuint64_t dims[3] = {64, (cuuint64_t)args.cache.pages * args.cache.kv_heads * page, (cuuint64_t)S::parts};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, 128};
    const cuuint32_t element_strides[3] = {1, 1, 1};
    const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int which = 0; which < 2; ++which) {
        const cuuint32_t k_box[3] = {64, k_tokens, 1};
        const cuuint32_t v_box[3] = {64, v_tokens, S::parts};
        if (encode(which == 0 ? &p.k_map : &p.v_map, type, 3, which == 0 ? args.cache.keys : args.cache.values, dims, strides,
                   which == 0 ? k_box : v_box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    // As many tiles of rows as the host's numbers allow.  A sequence of n tokens has 1 + floor((n G - 1) / 128): the sum over
    // s sequences of N tokens is at most s + floor((N G - s) / 128), and, as a further tile takes floor(128 / G) further
    // tokens, at most s + floor((N - s) / floor(128 / G)).
    const uint64_t tokens = args.batch.tokens, group = args.group;
    const uint64_t sequences = args.batch.sequences < tokens ? args.batch.sequences : tokens;
    uint64_t tiles = sequences + (tokens * group - sequences) / kTileRowsQ;
    if (group <= kTileRowsQ && (tokens - sequences) / (kTileRowsQ / group) < (tokens * group - sequences) / kTileRowsQ)
        tiles = sequences + (tokens - sequences) / (kTileRowsQ / group);
    const uint64_t units = tiles * args.cache.kv_heads;
    const size_t smem = S::query + (size_t)2 * S::slots * kSlotBytes + kMiscBytes + 1024;
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(kPromptThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = 1;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    // clusters of 2 .. 8 that a device holds at once: fewer than its SMs divided, a cluster stays within a part of the chip
    static int room[kMaxDevices][kMostSplits + 1] = {};
    int here[kMostSplits + 1] = {};
    const int slot = device_slot();
    if (slot >= 0 && room[slot][1] != 0) {
        for (uint32_t k = 1; k <= kMostSplits; ++k) here[k] = room[slot][k];
    } else {
        cudaError_t status = cudaFuncSetAttribute(prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (status != cudaSuccess) return status;
        here[1] = sm_count;
        for (uint32_t k = 2; k <= kMostSplits; ++k) {
            attribute[0].val.clusterDim.x = k;
            config.gridDim = dim3((unsigned)sm_count / k * k);
            status = cudaOccupancyMaxActiveClusters(&here[k], prompt_kernel<T, D>, &config);
            if (status != cudaSuccess) return status;
        }
        if (slot >= 0)
            for (uint32_t k = kMostSplits; k >= 1; --k) room[slot][k] = here[k];
    }
    p.splits = 1;
    for (uint32_t k = 2; k <= kMostSplits; ++k)
        if (units <= (uint64_t)here[k]) p.splits = k;
    if (units * p.splits > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    p.units = (uint32_t)units;
    p.sms = (uint32_t)sm_count;
    config.gridDim = dim3((unsigned)(units * p.splits));
    attribute[0].val.clusterDim.x = p.splits;
    return cudaLaunchKernelEx(&config, prompt_kernel<T, D>, p);
}

template <typename T>
cudaError_t launch_prompt_head(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    switch (args.cache.head_size) {
        case 64: return launch_prompt_of<T, 64>(args, sm_count, stream);
        case 128: return launch_prompt_of<T, 128>(args, sm_count, stream);
        case 256: return launch_prompt_of<T, 256>(args, sm_count, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

bool prompt_serves(const AttentionArgs &args) {
    // TMA counts the pools' rows in 31 bits.  No B200 holds such a pool (256 GiB at 64 values a row); a cache that declares
    // more pages than it uses may count as one, and is served as before, by the other kernel
    return (uint64_t)args.cache.pages * args.cache.kv_heads * args.cache.page_tokens <= 0x7fffffffull;
}

cudaError_t launch_prompt(const AttentionArgs &args, int sm_count, cudaStream_t stream) {
    return args.cache.dtype == kBF16 ? launch_prompt_head<__nv_bfloat16>(args, sm_count, stream)
                                     : launch_prompt_head<__half>(args, sm_count, stream);
}

}  // namespace q4b
