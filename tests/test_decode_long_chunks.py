"""Chunk lengths set by the caller up to the largest (kvc_config.decode_chunk_blocks,
"never split"): the split rules on the CPU, without an overflow, and on the GPU
the results of one chunk per sequence."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NQ, say

CSRC = Path(__file__).resolve().parents[1] / "qwen3.5-9b-bfp8b-1xn300_amd" / "csrc"
CXX = shutil.which("g++")
MAX = 2 ** 31 - 1

# stdin: "chunk_blocks nb n8 nb n8 ..."; stdout: the caller's chunk as taken,
# then both chunk lengths and each sequence's first chunk
PROGRAM = r"""
#include <cstdio>
#include <iostream>
#include <memory>
#include <sstream>
#include <string>
#include "kvc_decode_q8_split.h"
using namespace kvc;
int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        auto a = std::make_unique<DecodeQ8Args>();
        int chunk, nb[kMaxBatch], n = 0;
        in >> chunk;
        for (int x, y; in >> x >> y; n++) nb[n] = x, a->n8[n] = y;
        decode_q8_split(nb, n, chunk, *a);
        std::printf("%d %d %d", caller_chunk_blocks(chunk), a->cb8, a->cbf);
        for (int j = 0; j <= n; j++) std::printf(" %d", a->chunk_begin[j]);
        std::printf("\n");
    }
}
"""


@pytest.mark.skipif(CXX is None, reason="needs g++")
def test_split_of_long_chunks(tmp_path):
    (tmp_path / "split.cpp").write_text(PROGRAM)
    subprocess.run([CXX, "-O1", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{CSRC}", str(tmp_path / "split.cpp"), "-o", str(tmp_path / "split")], check=True)
    most = 2 ** 26  # the blocks of 2^31 tokens
    cases = [(c, seqs) for c in (MAX, MAX - 1, MAX - 39, 2 ** 30, most + 1, most, 41, 40)
             for seqs in ([(41, 40)], [(40, 40)], [(1, 0)], [(5, 0), (41, 40), (33, 33), (64, 1)])]
    text = "\n".join(" ".join(map(str, (c, *(x for p in seqs for x in p)))) for c, seqs in cases)
    out = subprocess.run([str(tmp_path / "split")], input=text, capture_output=True, text=True, check=True).stdout
    for (c, seqs), line in zip(cases, out.splitlines()):
        taken, cb8, cbf, *begin = map(int, line.split())
        assert taken == cb8 == cbf == min(c, most)
        want = [0]
        for nb, n8 in seqs:
            want.append(want[-1] - (-n8 // taken) - (-(nb - n8) // taken))
        assert begin == want, (c, seqs)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [0, 3000])
def test_decode_in_one_chunk(keep):
    """with 8-bit blocks and without: the bits of a chunk that is just longer
    than the sequences"""
    say(f"decode, chunks of {MAX} blocks, keep {keep}")
    lens = [1300, 64, 33, 1]
    got = []
    for chunk in (64, MAX):
        with Q.Filled(lens, seed=501, decode_chunk_blocks=chunk) as f:
            q = O.normal_bf16(len(lens) * NQ * D, 502).reshape(len(lens), NQ, D)
            f.ctx.kv_quantize(f.seqs, keep)
            calls = [f.ctx.decode_attn, f.ctx.decode_attn_static] if keep else [f.ctx.decode_attn]
            got.append([f.run(lambda a, o: call(0, f.seqs, a, o, out_dtype=dt), q.shape, bits, q)
                        for call in calls for dt, bits in ((kvc.DTYPE_F32, np.uint32), (kvc.DTYPE_BF16, np.uint16))])
    assert all(np.array_equal(a, b) and a.any() for a, b in zip(*got))
