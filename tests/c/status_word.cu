// What a descriptor that does not hold together leaves in the status word, on the host.  Needs no GPU.
//   input:  the word before, tokens page_tokens table_stride begin0 begin1 length;  output: the word behind
#include "../../cpu-llms-in-c_b200/csrc/q4b_cache.cuh"

#include <cstdio>

int main() {
    uint32_t status, tokens, page_tokens, stride, begin[2], length;
    if (scanf("%u %u %u %u %u %u %u", &status, &tokens, &page_tokens, &stride, &begin[0], &begin[1], &length) != 7) return 1;
    const q4b::BatchView batch = {begin, &length, nullptr, 1, tokens, stride};
    q4b::sequence_rows(batch, page_tokens, 0, &status);
    printf("%u\n", status);
    return 0;
}
