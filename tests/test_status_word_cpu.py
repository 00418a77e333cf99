"""The status word that queued work leaves its first mistake in (tests/c/status_word.cu): a descriptor's code takes the place
of nothing, so the code of an expired wait reaches q4b_sync, which clears the counters that such work leaves behind."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD_LENGTH, BAD_BEGIN = 0x1002, 0x1003


@pytest.fixture(scope="module")
def word(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    program = str(tmp_path_factory.mktemp("word") / "status_word")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-o", program,
                    os.path.join(ROOT, "tests", "c", "status_word.cu")], check=True, capture_output=True)

    def behind(before, begin, length, tokens=8, page_tokens=16, stride=2):
        text = " ".join(str(x) for x in (before, tokens, page_tokens, stride, *begin, length))
        return int(subprocess.run([program], input=text, capture_output=True, text=True, check=True, timeout=60).stdout)
    return behind


def test_a_mistake_is_noted(word):
    assert word(0, [0, 8], 32) == 0
    assert word(0, [0, 9], 32) == BAD_BEGIN and word(0, [5, 4], 32) == BAD_BEGIN
    assert word(0, [0, 8], 33) == BAD_LENGTH


@pytest.mark.parametrize("expired", [0x81, 0x82, 0x84, 0x11])
def test_the_code_of_an_expired_wait_stays(word, expired):
    assert word(expired, [0, 9], 32) == expired
    assert word(expired, [0, 8], 33) == expired


def test_the_first_mistake_stays(word):
    assert word(BAD_LENGTH, [0, 9], 32) == BAD_LENGTH
    assert word(0, [0, 9], 33) == BAD_BEGIN
