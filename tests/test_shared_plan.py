"""How a decode launch over shared blocks is cut into work
(csrc/kvc_shared_plan.h), on the CPU: every key block of every sequence is
attended once, in order, shared ones once for all their members; every
(chunk, kv head, group of members) is one workgroup's, as the kernel reads its
item number; partial rows do not overlap and fit the workspace."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen3.5-9b-bfp8b-1xn300_amd" / "csrc"
CXX = shutil.which("g++")
pytestmark = pytest.mark.skipif(CXX is None, reason="needs g++")
BT, HEADS = 32, 4
KEYS, ALL_HEADS, ONE = 0, 1, 2  # kinds

# stdin: launches as "n chunk share", then per sequence "keys nblk id id ..."; stdout: the plan
PROGRAM = r"""
#include <cstdio>
#include <iostream>
#include <vector>
#include "kvc_shared_plan.h"
int main() {
    int n, chunk, share;
    while (std::cin >> n >> chunk >> share) {
        std::vector<std::vector<int32_t>> t(n);
        std::vector<int32_t> keys(n);
        std::vector<const int32_t*> tab(n);
        for (int i = 0; i < n; i++) {
            int nb;
            std::cin >> keys[i] >> nb;
            t[i].resize(nb);
            for (auto& x : t[i]) std::cin >> x;
            tab[i] = t[i].data();
        }
        kvc::SharedPlan p;
        kvc::shared_plan(tab.data(), keys.data(), n, chunk, p);
        std::printf("%d %d %d %d %lld %lld %d %d\n", p.n_nodes, p.n_items, p.parts, p.path, (long long)p.blocks,
                    (long long)p.blocks_apart, (int)kvc::shared_pays(p, n, share), p.group);
        for (int k = 0; k < p.n_nodes; k++) {
            std::printf("%d %d %d %d %d %d", p.first[k], p.len[k], p.item_begin[k], p.chunk[k], p.kind[k], p.item_begin[k + 1]);
            for (int i = p.member_begin[k]; i < p.member_begin[k] + p.members[k]; i++)
                std::printf(" %d %d", p.member[i], p.seq_row[p.member[i]] + p.part[i]);
            std::printf("\n");
        }
    }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("shared_plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([CXX, "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)

    def run(launches, share=True):
        """launches: (chunk, [(keys, table), ...]); share: over shared blocks wherever there are any"""
        text = "\n".join("\n".join([f"{len(seqs)} {chunk} {int(share)}"] + [" ".join(map(str, (k, len(t), *t))) for k, t in seqs])
                         for chunk, seqs in launches)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        lines = iter(out.splitlines())
        got = []
        for _ in launches:
            head = dict(zip(("n_nodes", "n_items", "parts", "path", "blocks", "apart", "pays", "group"), map(int, next(lines).split())))
            nodes = []
            for _ in range(head["n_nodes"]):
                x = list(map(int, next(lines).split()))
                nodes.append(dict(zip(("first", "len", "item", "chunk", "kind", "end"), x[:6]), members=x[6::2], rows=x[7::2]))
            got.append((head, nodes))
        return got

    return run


def tree(rng, n, depth_blocks, ids):
    """A random trie of n tables, [(keys, table)]."""
    def grow(k, prefix):
        prefix = prefix + [next(ids) for _ in range(rng.choice([0, 1, 2, 7, rng.randint(0, depth_blocks)]))]
        if k == 1:
            return [prefix]
        out = []
        while k:
            take = rng.randint(1, k) if k < 3 or rng.random() < 0.8 else k
            if take == k and len(out) == 0:
                take = rng.randint(1, k - 1)
            out += grow(take, prefix)
            k -= take
        return out

    seqs = []
    for t in grow(n, []):
        t = t or [next(ids)]
        keys = max(1, len(t) * BT - rng.choice([0, 0, 1, 31, rng.randint(0, 200)]))
        keys = rng.choice([keys, keys, 0]) if rng.random() < 0.1 else keys
        seqs.append((keys, t))
    rng.shuffle(seqs)
    return seqs


def check(head, nodes, seqs):
    path = {i: [] for i in range(len(seqs))}
    used = set()  # partials
    for x in nodes:
        assert x["len"] > 0 and len(set(x["members"])) == len(x["members"])
        chunks = -(-x["len"] // x["chunk"])
        units = chunks * (1 if x["kind"] == ALL_HEADS else HEADS)
        # the kernel's reading of its item number
        seen = set()
        groups = -(-len(x["members"]) // head["group"])
        begin = 0 if x is nodes[0] else nodes[nodes.index(x) - 1]["end"]
        for item in range(begin, x["end"]):
            j, grp = item - begin, 0
            if groups > 1:
                j = item - (begin + 7) // 8 * 8
                if j < 0:
                    continue
                grp, j = (j >> 3) % groups, (j >> 3) // groups * 8 + (j & 7)
            if j >= units:
                continue
            assert (j, grp) not in seen
            seen.add((j, grp))
        assert len(seen) == units * groups
        assert x["chunk"] <= {KEYS: 2 * 64, ALL_HEADS: 32, ONE: 1023}[x["kind"]]  # ids that a wave holds
        assert (x["kind"] == ONE) == (len(x["members"]) == 1)
        for m, row in zip(x["members"], x["rows"]):
            keys, t = seqs[m]
            path[m].append((x["first"], x["len"], chunks))
            if head["pays"]:
                rows = set(range(row, row + chunks))
                assert not rows & used
                used |= rows
            first = seqs[x["members"][0]][1]
            assert t[x["first"]:x["first"] + x["len"]] == first[x["first"]:x["first"] + x["len"]]
            if len(x["members"]) > 1:  # whole blocks only
                assert (x["first"] + x["len"]) * BT <= keys
    assert head["n_items"] == (nodes[-1]["end"] if nodes else 0) and head["group"] in (4, 8)
    for i, (keys, t) in enumerate(seqs):
        at = 0
        for first, n, _ in sorted(path[i]):  # once each
            assert first == at
            at += n
        assert at == -(-keys // BT)
    parts = [sum(c for _, _, c in p) for p in path.values()]
    assert head["path"] == max(parts, default=0) and head["parts"] == sum(parts)
    assert head["blocks"] == sum(x["len"] for x in nodes)
    assert head["apart"] == sum(-(-k // BT) for k, _ in seqs)
    if head["pays"]:
        assert used == set(range(head["parts"]))
        assert head["path"] <= 512 and head["parts"] * 16 * 258 * 4 <= 8192 * 4 * 1056 * 4


@pytest.mark.parametrize("seed", range(8))
def test_random_tries(plans, seed):
    rng = random.Random(seed)
    launches = []
    for _ in range(60):
        ids = iter(rng.sample(range(100000), 20000))
        launches.append((rng.choice([0, 0, 0, 1, 3, 40, 1 << 20]), tree(rng, rng.randint(1, 64), rng.choice([3, 20, 150]), ids)))
    for (head, nodes), (_, seqs) in zip(plans(launches), launches):
        check(head, nodes, seqs)


def common(n, prefix_blocks, tail_blocks):
    ids = iter(range(10 ** 6))
    prefix = [next(ids) for _ in range(prefix_blocks)]
    return [((prefix_blocks + tail_blocks) * BT, prefix + [next(ids) for _ in range(tail_blocks)]) for _ in range(n)]


def test_a_common_prefix_is_read_once(plans):
    for n in (2, 4, 5, 16, 17, 64):
        (head, nodes), = plans([(0, common(n, 128, 3))])
        check(head, nodes, common(n, 128, 3))
        assert head["blocks"] == 128 + 3 * n and head["pays"]
        assert nodes[0]["members"] == list(range(n)) and nodes[0]["kind"] == KEYS


def test_nothing_in_common(plans):
    seqs = [(100, [4 * i, 4 * i + 1, 4 * i + 2, 4 * i + 3]) for i in range(10)]
    (head, nodes), = plans([(0, seqs)])
    check(head, nodes, seqs)
    assert head["blocks"] == head["apart"] == 40 and not head["pays"]


def test_ladders_and_long_prefixes(plans):
    """Each sequence leaves one block after the one before it: more memberships
    than the argument block holds are not made.  A prefix of 2^18 tokens."""
    ids = list(range(2000))
    ladder = [((8 * i + 9) * BT, ids[:8 * i + 8] + [5000 + i]) for i in range(64)]
    long = common(64, 8192, 1)
    for (head, nodes), seqs in zip(plans([(0, ladder), (0, long), (1, long)]), (ladder, long, long)):
        check(head, nodes, seqs)
        assert sum(-(-len(x["members"]) // 8) * 8 for x in nodes if len(x["members"]) > 1) <= 512 and head["n_nodes"] <= 128


def test_only_new_tokens(plans):
    (head, nodes), = plans([(0, [(0, [1]), (0, [2])])])
    assert head["n_nodes"] == 0 and head["n_items"] == 0 and not head["pays"]


def test_same_sequence_many_times_over_ends_in_a_shared_block(plans):
    """Forks that have not been written to: the last block is not full, so each
    attends it alone."""
    t = list(range(20))
    seqs = [(20 * BT - 5, t) for _ in range(9)]
    (head, nodes), = plans([(0, seqs)])
    check(head, nodes, seqs)
    assert nodes[0]["len"] == 19 and head["blocks"] == 19 + 9


@pytest.mark.parametrize("n,prefix,tail,shares", [(4, 9, 1, False), (8, 31, 1, False), (2, 128, 1, False),
                                                  (8, 128, 1, True), (16, 62, 2, True), (64, 31, 1, True),
                                                  (64, 3, 30, False), (64, 256, 24, True), (4, 500, 1, True),
                                                  (4, 128, 1, True), (8, 62, 1, False), (16, 31, 1, False)])
def test_where_it_is_worth_it(plans, n, prefix, tail, shares):
    """the measured side (us per layer in the rule's comment)"""
    (head, _), = plans([(0, common(n, prefix, tail))], share=False)
    assert bool(head["pays"]) == shares
