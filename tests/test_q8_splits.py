"""The rules for the work split of decode and prefill launches over sequences
with 8-bit blocks (csrc/kvc_decode_q8_split.h, csrc/kvc_prefill_q8_split.h), on
the CPU: every block is taken once, in the order that the kernels assume, and
the picks are the measured ones."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen3.5-9b-bfp8b-1xn300_amd" / "csrc"
CXX = shutil.which("g++")
pytestmark = pytest.mark.skipif(CXX is None, reason="needs g++")

# stdin: "d chunk_blocks nb n8 nb n8 ..." (decode) or "p n_q prefix prefix ..."
# stdout: the split's numbers, a launch a line
PROGRAM = r"""
#include <cstdio>
#include <iostream>
#include <memory>
#include <sstream>
#include <string>
#include "kvc_decode_q8_split.h"
#include "kvc_prefill_q8_split.h"
using namespace kvc;
int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        char kind;
        in >> kind;
        if (kind == 'd') {
            auto a = std::make_unique<DecodeQ8Args>();
            int chunk, nb[kMaxBatch], n = 0;
            in >> chunk;
            for (int x, y; in >> x >> y; n++) nb[n] = x, a->n8[n] = y;
            decode_q8_split(nb, n, chunk, *a);
            std::printf("%d %d %d %d %d %d", a->cb8, a->cbf, a->total_chunks, a->n_items, a->per_xcd, (int)kMaxChunks);
            for (int j = 0; j <= n; j++) std::printf(" %d", a->chunk_begin[j]);
        } else {
            auto a = std::make_unique<PrefillQ8Args>();
            PrefillArgs few{};
            in >> a->n_q;
            few.n_q = a->n_q;
            for (int p; in >> p;) few.q_pos0[few.n_seqs++] = a->q_pos0[a->n_seqs++] = p;
            const bool ok = prefill_q8_fits(few);
            if (ok) prefill_q8_split(*a);
            std::printf("%d %d %d %d", (int)prefill_q8_few(few), (int)ok, a->n_wgs, a->per_xcd);
            for (int j = 0; ok && j <= a->n_seqs; j++) std::printf(" %d", a->begin[j]);
            for (int w = 0; ok && w <= a->n_wgs; w++) std::printf(" %d", a->cut[w]);
            for (int w = 0; ok && w < a->n_wgs; w++) std::printf(" %d", a->seq_at[w]);
        }
        std::printf("\n");
    }
}
"""


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    d = tmp_path_factory.mktemp("q8_split")
    (d / "split.cpp").write_text(PROGRAM)
    subprocess.run([CXX, "-O2", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{CSRC}", str(d / "split.cpp"), "-o", str(d / "split")], check=True)

    def run(lines):
        text = "\n".join(" ".join(map(str, x)) for x in lines)
        out = subprocess.run([str(d / "split")], input=text, capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]

    return run


def up(a, b):
    return -(-a // b)


def test_decode_chunks_cover_every_block(split):
    rng = random.Random(1)
    cases = []
    for i in range(400):
        n = rng.randint(1, 64)
        top = rng.choice([3, 40, 600, 4000])
        nb = [rng.randint(1, top) for _ in range(n)]
        n8 = [rng.randint(0, x) if rng.random() < 0.8 else rng.choice([0, x]) for x in nb]
        cases.append((rng.choice([0, 0, 0, 1, 5, 300]), nb, n8))
    cases.append((1, [30000] * 64, [29999] * 64))  # more chunks than a launch holds: longer ones
    got = split([("d", c, *(x for p in zip(nb, n8) for x in p)) for c, nb, n8 in cases])
    for (chunk, nb, n8), (cb8, cbf, total, items, per_xcd, most, *begin) in zip(cases, got):
        assert cb8 >= 1 and cbf >= 1 and total <= most and items == 4 * total and per_xcd == up(items, 8)
        assert begin[0] == 0 and begin[-1] == total
        for j in range(len(nb)):
            assert begin[j + 1] - begin[j] == up(n8[j], cb8) + up(nb[j] - n8[j], cbf)
        if chunk and sum(up(x, chunk) + up(y - x, chunk) for x, y in zip(n8, nb)) <= most:
            assert (cb8, cbf) == (chunk, chunk)


def test_decode_picks(split):
    """blocks per chunk where the sweep over chunk lengths showed a best or
    nearly best one"""
    launches = [([128], 4), ([47], 4), ([500], 8), ([10] * 64, 10), ([160] * 40, 20)]
    got = split([("d", 0, *(x for n in nb for x in (n, n))) for nb, _ in launches])
    assert [x[0] for x in got][:2] == [4, 4] and got[2][0] in (4, 8)
    assert got[3][0] >= 10  # short sequences are not cut
    assert 16 <= got[4][0] <= 32


def blocks_of(n_q, prefix):
    return [up(prefix + min(r + 64, n_q), 32) for r in range(0, n_q, 64)]


def test_prefill_runs_cover_every_block(split):
    rng = random.Random(2)
    cases = [(1, [0]), (1, [40000]), (33, [0]), (512, [16384]), (4096, [16000] * 64), (64, [0] * 64), (700, [5] * 24)]
    for i in range(400):
        n = rng.randint(1, 64)
        top = rng.choice([5, 300, 6000, 16384])
        cases.append((rng.choice([1, 2, 31, 32, 33, 64, 65, 127, 128, 300, 1000]), [rng.randint(0, top) for _ in range(n)]))
    for (n_q, prefix), (few, ok, wgs, per_xcd, *rest) in zip(cases, split([("p", q, *p) for q, p in cases])):
        n = len(prefix)
        begin, cut, seq_at = rest[:n + 1], rest[n + 1:n + 2 + wgs], rest[n + 2 + wgs:]
        items = [[x for _ in range(4) for x in blocks_of(n_q, p)] for p in prefix]
        assert ok and 1 <= wgs <= 256 and per_xcd == up(wgs, 8) and len(seq_at) == wgs
        assert begin == [sum(map(sum, items[:j])) for j in range(n + 1)]
        assert cut[0] == 0 and cut[-1] == begin[-1]
        cost = []
        starts, at = set(), 0
        for x in sum(items, []):
            starts.add(at)
            at += x
        for w in range(wgs):
            assert cut[w] < cut[w + 1]
            assert begin[seq_at[w]] <= cut[w] < begin[seq_at[w] + 1]
            taken = sum(1 for s in starts if cut[w] < s < cut[w + 1]) + 1
            cost.append(cut[w + 1] - cut[w] + 7 * taken) if begin[-1] < 20000 else None
        total = begin[-1]
        if cost and total >= 2000:  # no run is much longer than the mean
            assert max(cost) <= 1.5 * (total + 7 * len(starts)) / 256 + 12, (n_q, prefix)
        assert few == (n_q <= 32 or total <= 2000)


def test_prefill_too_large_is_refused(split):
    for n_q, prefix in ((1 << 20, [1 << 20]), (1 << 15, [1 << 20] * 64), (2 ** 31 - 64, [0])):
        (few, ok, *_), = split([("p", n_q, *prefix)])
        assert not few and not ok
