// The index arithmetic of the paged-cache kernels on the host: reads descriptors from stdin, prints what the kernels
// would make of them.  Needs no GPU.
//   input:  tokens sequences table_stride page_tokens window sinks group chunk_rows, begin[sequences + 1], lengths[sequences]
//   output: per sequence "rows begin count length status", then per chunk of rows "groups i0 i1 ..." (16-key groups)
#include "../../cpu-llms-in-c_b200/csrc/q4b_cache.cuh"

#include <cstdio>
#include <vector>

using namespace q4b;

int main() {
    unsigned tokens, sequences, stride, page_tokens, window, sinks, group, chunk;
    if (scanf("%u %u %u %u %u %u %u %u", &tokens, &sequences, &stride, &page_tokens, &window, &sinks, &group, &chunk) != 8) return 1;
    std::vector<uint32_t> begin(sequences + 1), lengths(sequences);
    for (auto &x : begin) if (scanf("%u", &x) != 1) return 1;
    for (auto &x : lengths) if (scanf("%u", &x) != 1) return 1;
    const BatchView batch = {begin.data(), lengths.data(), nullptr, sequences, tokens, stride};
    for (uint32_t s = 0; s < sequences; ++s) {
        uint32_t status = 0;
        const SequenceRows rows = sequence_rows(batch, page_tokens, s, &status);
        printf("rows %u %u %u %u\n", rows.begin, rows.count, rows.length, status);
        for (uint32_t row0 = 0; row0 < rows.count * group; row0 += chunk) {
            const uint32_t row1 = (row0 + chunk < rows.count * group ? row0 + chunk : rows.count * group) - 1;
            const Groups g = groups_of(rows, row0 / group, row1 / group, window, sinks);
            printf("groups");
            for (uint32_t i = 0; i < g.count(); ++i) printf(" %u", g.end == 0 ? 0xffffffffu : g.at(i));
            printf("\n");
        }
    }
    return 0;
}
