"""Plans of long decode launches over shared blocks (CPU): partials of a sequence past
64 and past 256, chunks of one member past 64 blocks.  test_gpu_shared_long.py runs
launches of these trees."""
import pytest

from test_shared_plan import BT, CXX, ONE, check, plans  # noqa: F401

pytestmark = pytest.mark.skipif(CXX is None, reason="needs g++")


def launch(prefix, tails):
    """[(keys, table)] of sequences behind a common prefix, in tokens"""
    full = prefix // BT
    ids = iter(range(10 ** 6))
    head = [next(ids) for _ in range(full)]
    return [(prefix + t, head + [next(ids) for _ in range(-(-(prefix + t) // BT) - full)]) for t in tails]


@pytest.mark.parametrize("prefix,tails,chunk,low,high", [
    (3000, (1, 40, 1000), 1, 65, 256), (600, (9000, 3, 100), 1, 257, 512),
    (4000, (7900, 8000), 1, 257, 512), (65536, (1, 5, 40, 100), 0, 65, 256), (8192, (5,) * 30 + (30000,), 0, 65, 256),
])
def test_many_partials(plans, prefix, tails, chunk, low, high):  # noqa: F811
    seqs = launch(prefix, tails)
    (head, nodes), = plans([(chunk, seqs)], share=chunk > 0)
    check(head, nodes, seqs)
    assert head["pays"] and low <= head["path"] <= high


@pytest.mark.parametrize("prefix,tails,chunk", [(1000, (2500, 4500, 30), 1000), (500, (2080, 1, 64 * 32), 1000)])
def test_long_chunks_of_one_member(plans, prefix, tails, chunk):  # noqa: F811
    seqs = launch(prefix, tails)
    (head, nodes), = plans([(chunk, seqs)])
    check(head, nodes, seqs)
    assert head["pays"] and max(min(x["len"], x["chunk"]) for x in nodes if x["kind"] == ONE) > 64
