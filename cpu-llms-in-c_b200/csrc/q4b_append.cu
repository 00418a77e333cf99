// New tokens' keys and values into the paged cache, keys and queries turned by their positions on the way.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * frequency(i)
//
// for the pairs of the first rotary_size values of every query and key head; everything else is copied.  One pass:
// every value is read once and written once, so the kernel is bound by memory for many tokens and by the latency of
// launch -> sequence -> length -> page number -> store for few.
//
// A position of a million radians has two digits left in fp32, and sincosf of it is slow as well.  Positions are
// therefore counted in full turns: position * (frequency / 2 pi) in fp64, less its nearest whole number, is the
// angle to 2^-22 of a turn over the whole range of int32 positions and far better at ordinary ones; sincospif takes
// the rest, half a turn at most.  One thread does that per (token, pair); the heads share it through shared memory.
//
// Work unit: 16 values of one head -- 8 + 8 that are partners in the HALVES form, 16 neighbours otherwise -- so a
// thread reads both partners before it writes either and q may be turned in place.  Two units per thread at once took
// longer (57 us against 52 us for 8,192 tokens).
//
// Measured on B200 (24 query heads and 4 key heads of 256, 16-bit in and out): 8,192 tokens in 52 us = 5.2 TB/s of 6.54, one
// token in 4.1 us on the device, 6.4 us with the host's call.
#include "q4b_cache.cuh"

namespace q4b {

namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kAppendTokens = 4;  // tokens a thread block takes: their tables are made together

template <typename T> __device__ inline void load8(const T *from, float (&x)[8]);
template <> __device__ inline void load8<float>(const float *from, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(from)[0], b = reinterpret_cast<const float4 *>(from)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ inline void load8<__half>(const __half *from, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(from);
    const __half2 *h = reinterpret_cast<const __half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <> __device__ inline void load8<__nv_bfloat16>(const __nv_bfloat16 *from, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(from);
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ inline void store8(__half *to, const float (&x)[8]) {
    uint4 raw;
    __half2 *h = reinterpret_cast<__half2 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(to) = raw;
}
__device__ inline void store8(__nv_bfloat16 *to, const float (&x)[8]) {
    uint4 raw;
    __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(to) = raw;
}

template <typename In, typename Out>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(const __grid_constant__ AppendArgs p) {
    __shared__ float2 turn[kAppendTokens][128];  // cos, sin
    __shared__ int32_t place[kAppendTokens];     // in its sequence; negative: nothing to do
    __shared__ uint32_t slot_page[kAppendTokens];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row0 = blockIdx.x * kAppendTokens;
    const uint32_t rows = min(kAppendTokens, p.batch.tokens - row0);
    const uint32_t D = p.cache.head_size, pairs = p.rotary_size / 2;
    if (warp < rows) {
        const uint32_t row = row0 + warp;
        const uint32_t s = sequence_of_row(p.batch, row, lane);
        int32_t at = -1;
        uint32_t page = 0;
        if (s < p.batch.sequences) {
            const SequenceRows mine = sequence_rows(p.batch, p.cache.page_tokens, s, p.status);
            if (row >= mine.begin && row < mine.begin + mine.count) {
                const int64_t where = (int64_t)mine.length - mine.count + (row - mine.begin);
                if (where >= 0) {
                    at = (int32_t)where;
                    page = p.batch.table[(size_t)s * p.batch.table_stride + ((uint32_t)at >> p.cache.page_shift)];
                    if (page >= p.cache.pages) {
                        report(p.status, kBadPage);
                        at = -1;
                    }
                }
            }
        }
        if (lane == 0) {
            place[warp] = at;
            slot_page[warp] = page;
        }
        const double position = p.positions != nullptr ? (double)p.positions[row] : (double)at;
        for (uint32_t i = lane; i < pairs; i += 32) {
            const double turns = position * p.turns[i];
            float sine, cosine;
            sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
            turn[warp][i] = make_float2(cosine, sine);
        }
    } else if (warp >= kAppendTokens) {
        // the warps without a token look at all sequences: rows that a wrong begin leaves to nobody are told as well
        // (in 64 bits: the grid's threads are more than 2^32 from 2^27 rows on)
        constexpr uint32_t kLookers = kAppendThreads - 32 * kAppendTokens;
        for (uint64_t s = (uint64_t)blockIdx.x * kLookers + threadIdx.x - 32 * kAppendTokens; s < p.batch.sequences;
             s += (uint64_t)gridDim.x * kLookers)
            sequence_rows(p.batch, p.cache.page_tokens, (uint32_t)s, p.status);
    }
    __syncthreads();
    const uint32_t per_head = D / 16, heads = p.q_heads + 2 * p.cache.kv_heads;
    const uint32_t units = rows * heads * per_head;
    const bool halves = p.pairing == 0;
    for (uint32_t unit = threadIdx.x; unit < units; unit += kAppendThreads) {
        const uint32_t u = unit % per_head, rest = unit / per_head;
        const uint32_t head = rest % heads, local = rest / heads;
        const int32_t at = place[local];
        if (at < 0) continue;
        const uint32_t row = row0 + local;
        const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + p.cache.kv_heads;
        const uint32_t kv = is_v ? head - p.q_heads - p.cache.kv_heads : head - p.q_heads;
        const In *from;
        Out *to;
        if (is_q) {
            from = static_cast<const In *>(p.q) + (size_t)row * p.ldq + (size_t)head * p.q_head_stride;
            to = static_cast<Out *>(p.q_out) + (size_t)row * p.ldq_out + (size_t)head * D;
        } else {
            from = (is_v ? static_cast<const In *>(p.v) + (size_t)row * p.ldv
                         : static_cast<const In *>(p.k) + (size_t)row * p.ldk) + (size_t)kv * D;
            const size_t line = ((size_t)slot_page[local] * p.cache.kv_heads + kv) * p.cache.page_tokens +
                                ((uint32_t)at & (p.cache.page_tokens - 1));
            to = static_cast<Out *>(is_v ? p.cache.values : p.cache.keys) + line * D;
        }
        const bool turned = !is_v && u * 8 < pairs;
        const uint32_t lower = turned && halves ? 8 * u : 16 * u;
        const uint32_t upper = turned && halves ? pairs + 8 * u : 16 * u + 8;
        float a[8], b[8];
        load8(from + lower, a);
        load8(from + upper, b);
        if (turned) {
            const float2 *t = &turn[local][8 * u];
            if (halves) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = a[i], y = b[i];
                    a[i] = x * t[i].x - y * t[i].y;
                    b[i] = y * t[i].x + x * t[i].y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float x = a[i], y = a[i + 1], z = b[i], w = b[i + 1];
                    a[i] = x * t[i / 2].x - y * t[i / 2].y;
                    a[i + 1] = y * t[i / 2].x + x * t[i / 2].y;
                    b[i] = z * t[4 + i / 2].x - w * t[4 + i / 2].y;
                    b[i + 1] = w * t[4 + i / 2].x + z * t[4 + i / 2].y;
                }
            }
        }
        store8(to + lower, a);
        store8(to + upper, b);
    }
}

template <typename In>
cudaError_t launch_append_from(const AppendArgs &args, cudaStream_t stream) {
    const uint32_t blocks = ceil_div(args.batch.tokens, kAppendTokens);
    if (args.cache.dtype == kBF16) append_kernel<In, __nv_bfloat16><<<blocks, kAppendThreads, 0, stream>>>(args);
    else append_kernel<In, __half><<<blocks, kAppendThreads, 0, stream>>>(args);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append(const AppendArgs &args, cudaStream_t stream) {
    if (args.dtype == kF32) return launch_append_from<float>(args, stream);
    if (args.dtype == kBF16) return launch_append_from<__nv_bfloat16>(args, stream);
    return launch_append_from<__half>(args, stream);
}

}  // namespace q4b
