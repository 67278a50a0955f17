"""Host side of the speculative-decoding operators: the tree helper, and every refusal of the C entries.  A refused call
returns before it touches the device, so these run without a GPU."""
import numpy as np
import pytest

BAD, MISALIGNED = 1, 716      # cudaErrorInvalidValue, cudaErrorMisalignedAddress


@pytest.fixture(scope="module")
def L():
    from wukong_b200 import build
    build.build()
    import wukong_b200
    return wukong_b200.lib()


def test_tree_layout_masks_and_depths():
    from wukong_b200.device import tree_layout
    rng = np.random.default_rng(0)
    counts = [1, 0, 5, 70, 33]
    row0 = np.concatenate([[0], np.cumsum(counts)])
    parent = np.full(row0[-1], -1)
    for t, k in enumerate(counts):
        for i in range(1, k):
            parent[row0[t] + i] = rng.integers(0, i)
    mask, depth = tree_layout(parent, row0)
    assert mask.dtype == np.int32 and mask.shape == (row0[-1], 3)
    for t, k in enumerate(counts):
        for i in range(k):
            line, j = {i}, i
            while j:
                j = int(parent[row0[t] + j])
                line.add(j)
            bits = {b for b in range(96) if (int(mask[row0[t] + i].view(np.uint32)[b // 32]) >> (b % 32)) & 1}
            assert bits == line and depth[row0[t] + i] == len(line) - 1
    m, dep = tree_layout(np.zeros(0), [0])
    assert m.shape == (0, 1) and dep.shape == (0,)


@pytest.mark.parametrize("parent,row0", [([-1, 1], [0, 2]), ([-1, -1], [0, 2]), ([-1, 2, 0], [0, 3]), ([-1], [0, 2]), ([-1, 0], [1, 2]), ([-1, 0], [0, 2, 1])])
def test_tree_layout_refusals(parent, row0):
    from wukong_b200.device import tree_layout
    with pytest.raises(ValueError):
        tree_layout(parent, row0)


P = 1 << 20          # a 16-byte aligned address that nothing reads


def attn(L, **over):
    a = dict(q=P, qd=0, qs=512, k=P, v=P, pages=10, bt=P, slot=P, ctx=P, row0=P, mask=P, words=2, out=P, od=1, os=512, rows=4, n=1, nodes=64, qh=4, kvh=2, hd=128,
             page=16, mbps=4, scale=1.0, scratch=P, size=1 << 40)
    a.update(over)
    return L.wkb_paged_attn_tree(*a.values(), None)


@pytest.mark.parametrize("over,code", [
    (dict(qh=3), BAD), (dict(qh=12), BAD), (dict(qh=32, kvh=2), BAD), (dict(kvh=0), BAD), (dict(hd=96), BAD), (dict(hd=256), BAD), (dict(page=2), BAD), (dict(page=24), BAD), (dict(page=0), BAD),
    (dict(nodes=0), BAD), (dict(nodes=257, words=9), BAD), (dict(nodes=65), BAD), (dict(n=4097), BAD), (dict(mbps=0), BAD), (dict(pages=0), BAD), (dict(qd=2), BAD), (dict(od=3), BAD),
    (dict(pages=1 << 30), BAD), (dict(mbps=1 << 28), BAD), (dict(scratch=None), BAD), (dict(size=0), BAD), (dict(rows=1 << 40), BAD), (dict(qs=-8), BAD), (dict(os=504), BAD), (dict(os=-512, rows=1), BAD),
    (dict(n=4096, kvh=8, qh=64, nodes=256, words=8, mbps=1 << 20), BAD),
    (dict(qs=516), MISALIGNED), (dict(os=516), MISALIGNED), (dict(q=P + 4), MISALIGNED), (dict(k=P + 8), MISALIGNED), (dict(v=P + 2), MISALIGNED), (dict(out=P + 8), MISALIGNED),
    (dict(scratch=P + 4), MISALIGNED)])
def test_attention_refusals(L, over, code):
    assert attn(L, **over) == code


def test_nothing_to_do_is_fine(L):
    assert attn(L, rows=0) == 0 and attn(L, n=0) == 0
    assert L.wkb_token_probs(P, 0, 10, None, P, 10, 0, 10, None) == 0
    assert L.wkb_tree_verify(P, 8, None, 0, P, P, P, 0, 0, 4, 8, P, P, P, P, P, 4, None) == 0
    assert L.wkb_paged_kv_commit(P, P, 1, 0, 1, P, P, P, P, P, 1, 0, 1, 64, 16, 1, None, None) == 0


@pytest.mark.parametrize("dtype,ld,ld_out,rows,cols", [(2, 10, 10, 1, 10), (0, 9, 10, 1, 10), (0, 10, 9, 1, 10), (0, 1 << 40, 1 << 40, 1, 1 << 35), (0, 1 << 31, 1 << 31, 1, (1 << 30) + 1), (0, 10, 10, 1 << 40, 10)])
def test_probs_refusals(L, dtype, ld, ld_out, rows, cols):
    assert L.wkb_token_probs(P, dtype, ld, None, P, ld_out, rows, cols, None) == BAD


@pytest.mark.parametrize("over", [dict(rows=-1), dict(rows=1 << 40), dict(n=1 << 40), dict(nodes=0), dict(nodes=257), dict(cols=0), dict(ld=7), dict(ldq=7), dict(max_path=0), dict(max_path=5)])
def test_verify_refusals(L, over):
    a = dict(rows=4, n=1, nodes=4, cols=8, ld=8, ldq=8, max_path=4)
    a.update(over)
    assert L.wkb_tree_verify(P, a["ld"], P, a["ldq"], P, P, P, a["rows"], a["n"], a["nodes"], a["cols"], P, P, P, P, P, a["max_path"], None) == BAD


@pytest.mark.parametrize("over,code", [(dict(n=65536), BAD), (dict(max_path=0), BAD), (dict(kvh=0), BAD), (dict(hd=4), BAD), (dict(hd=12), BAD), (dict(page=0), BAD), (dict(mbps=0), BAD),
                                       (dict(pages=0), BAD), (dict(stride=1000), BAD), (dict(pages=1 << 40, stride=1 << 56), BAD), (dict(new_ctx=P + 64), BAD), (dict(k=P + 8), MISALIGNED), (dict(stride=(1 << 20) + 4), MISALIGNED)])
def test_commit_refusals(L, over, code):
    a = dict(k=P, layers=2, stride=1 << 20, pages=4, max_path=4, n=1, kvh=2, hd=64, page=16, mbps=4, new_ctx=None)
    a.update(over)
    assert L.wkb_paged_kv_commit(a["k"], P, a["layers"], a["stride"], a["pages"], P, P, P + 64, P, P, a["max_path"], a["n"], a["kvh"], a["hd"], a["page"], a["mbps"],
                                 a["new_ctx"], None) == code


def test_wrappers_refuse_host_tensors():
    import torch
    from wukong_b200 import device as dev
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)
    f = torch.float32
    kv = dev.PagedKV(1, 2, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        dev.token_probs(z(2, 8, dt=f))
    with pytest.raises(ValueError):
        dev.tree_verify(z(4, 8, dt=f), None, z(4), z(4), z(2), z(4, dt=f), z(1, dt=f), 4, 4)
    with pytest.raises(ValueError):
        dev.paged_kv_commit(kv, z(1, 2), z(1), z(1), z(1, 3), z(1), 2)
    with pytest.raises(ValueError):
        dev.paged_attn_tree(z(1, 64, dt=f), 64, kv, 0, z(1, 2), z(1), z(1), z(2), z(1, 1), z(1, 64, dt=f), 1, 2, 1, 1.0, z(8, dt=torch.uint8))
