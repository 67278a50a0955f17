"""Pages of sequences that decode with draft trees: a step's nodes need pages in front of the step, the context moves on by the
accepted path alone."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def paged():
    from wukong_b200 import build
    build.build()
    from wukong_b200 import paged
    return paged


def test_contexts_and_pages_follow_the_accepted_paths(paged):
    rng = np.random.default_rng(3)
    page, slots, mbps = 16, 5, 12
    m = paged.BlockManager(40, page, slots, mbps)
    ctx = rng.integers(0, 40, slots)
    for s in range(slots):
        m.reserve(s, int(ctx[s]))
    tables = m.flat_block_table()
    for _ in range(12):
        nodes = rng.integers(1, 25, slots)
        for s in range(slots):
            m.ensure_capacity(s, int(nodes[s]))
            assert m.context_len(s) == ctx[s]
            for i in range(int(nodes[s])):
                m.locate(s, int(ctx[s]) + i)                     # every node has its place
        now = m.flat_block_table()
        for s in range(slots):
            held = -(-int(ctx[s]) // page)
            assert (now[s, :held] == tables[s, :held]).all()     # what is committed stays where it is
        tables = now
        for s in range(slots):
            n_path = int(rng.integers(1, min(4, nodes[s]) + 1))
            assert m.reserve(s, n_path) == ctx[s]                # inside the pages that are there
            ctx[s] += n_path
        assert m.ctx_lens().tolist() == ctx.tolist()
        assert (m.flat_block_table() == tables).all()
        assert m.used_blocks() <= sum(-(-int(c + 24) // page) for c in ctx)


def test_capacity_that_is_not_there(paged):
    m = paged.BlockManager(4, 2, 2, 3)
    m.reserve(0, 3)
    before = m.flat_block_table()
    with pytest.raises(paged.OutOfBlocks):
        m.ensure_capacity(0, 4)                                  # past the table row
    m.reserve(1, 3)
    with pytest.raises(paged.OutOfBlocks):
        m.ensure_capacity(0, 2)                                  # no page left
    assert (m.flat_block_table()[0] == before[0]).all() and m.context_len(0) == 3 and m.free_blocks() == 0
    m.ensure_capacity(0, 1)
    m.ensure_capacity(0, 0)
    assert m.context_len(0) == 3
