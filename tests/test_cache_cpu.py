"""The paged-cache operators without a GPU: refusals that need none, and the kernels' index arithmetic, compiled for the
host (tests/c/cache_indices.cu) and compared with the definition -- descriptors that do not hold together among it."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_missing_contexts_are_refused(q4b):
    lib = q4b.library()
    err = ctypes.create_string_buffer(256)
    cache, batch, rope = q4b.KVCache(), q4b.TokenBatch(), q4b.Rope()
    assert lib.q4b_rope_append(None, cache, batch, rope, None, 0, 0, None, 0, None, 0, 0, 0, None, 0, err, 256) == 1
    assert lib.q4b_attention(None, cache, batch, None, 0, 1, 1.0, 0, 0, None, 0, err, 256) == 1
    assert lib.q4b_sample(None, None, 0, 1, 1, 1, None, None, None, None, err, 256) == 1
    assert b"NULL" in err.value


@pytest.fixture(scope="module")
def indices(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    program = str(tmp_path_factory.mktemp("indices") / "cache_indices")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-o", program,
                    os.path.join(ROOT, "tests", "c", "cache_indices.cu")], check=True, capture_output=True)

    def ask(tokens, begin, lengths, stride, page_tokens, window, sinks, group, chunk):
        text = " ".join(str(int(x)) for x in [tokens, len(lengths), stride, page_tokens, window, sinks, group, chunk, *begin, *lengths])
        out = subprocess.run([program], input=text, capture_output=True, text=True, check=True, timeout=60).stdout
        sequences = []
        for line in out.splitlines():
            name, *numbers = line.split()
            if name == "rows":
                sequences.append((tuple(int(x) for x in numbers), []))
            else:
                sequences[-1][1].append([int(x) for x in numbers])
        return sequences
    return ask


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (5, 4), (16, 17), (33, 64), (40, 1000), (1000, 4)])
@pytest.mark.parametrize("group,chunk", [(1, 8), (6, 16), (6, 128), (8, 8), (3, 16)])
def test_groups_cover_what_the_rows_see(indices, window, sinks, group, chunk):
    counts, lengths = [1, 4, 0, 37, 3, 9], [1, 100, 7, 37, 300, 5]    # the last one: rows in front of the sequence's start
    begin = np.concatenate([[0], np.cumsum(counts)])
    for s, ((first, count, length, status), chunks) in enumerate(
            indices(int(begin[-1]), begin, lengths, 20, 16, window, sinks, group, chunk)):
        assert (first, count, length, status) == (begin[s], counts[s], lengths[s], 0)
        assert len(chunks) == -(-counts[s] * group // chunk)
        for c, groups in enumerate(chunks):
            seen = set()
            for row in range(c * chunk, min((c + 1) * chunk, counts[s] * group)):
                at = lengths[s] - counts[s] + row // group
                seen |= {j // 16 for j in range(at + 1) if window == 0 or j > at - window or j < sinks}
            if seen:
                assert len(groups) == len(set(groups)) and seen <= set(groups)
                assert max(groups) <= (lengths[s] - 1) // 16
                if window and chunk == 8 and group == 8:     # one token: no group for nothing
                    assert set(groups) == seen
            else:
                assert groups == [0xffffffff]


def test_descriptors_that_do_not_hold_together_stay_inside(indices):
    def check(tokens, begin, lengths, stride, page, statuses):
        found = indices(tokens, begin, lengths, stride, page, 7, 2, 2, 8)
        assert [f[0][3] for f in found] == statuses
        for (first, count, length, _), chunks in found:
            assert first + count <= tokens and length <= stride * page
            for groups in chunks:
                assert all(g == 0xffffffff or g * 16 < stride * page for g in groups)
    bad_length, bad_begin = 0x1002, 0x1003
    check(10, [0, 4, 10], [4, 64], 4, 16, [0, 0])
    check(10, [0, 4, 10], [4, 65], 4, 16, [0, bad_length])                       # a table too short
    check(10, [0, 4, 10], [0xffffffff, 0x80000000], 4, 16, [bad_length] * 2)
    check(10, [0, 6, 5], [8, 8], 4, 16, [0, bad_begin])                          # falls
    check(10, [0, 4, 11], [8, 8], 4, 16, [0, bad_begin])                         # passes the rows
    check(10, [0xfffffff0, 0xffffffff, 3], [8, 8], 4, 16, [bad_begin] * 2)
