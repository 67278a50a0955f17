"""Calls of the speculative-decoding entries that have to be refused, none of which reaches the device: these run without a
GPU.  Addresses are numbers that nothing reads; one of each call is not aligned, so that a call which passes the check in
question ends with that (716) and not on a device."""
import pytest

BAD, MISALIGNED = 1, 716      # cudaErrorInvalidValue, cudaErrorMisalignedAddress
P = 1 << 20


@pytest.fixture(scope="module")
def L():
    from wukong_b200 import build
    build.build()
    import wukong_b200
    return wukong_b200.lib()


def attn(L, **over):
    a = dict(q=P, qd=0, qs=512, k=P, v=P, pages=10, bt=P, slot=P, ctx=P, row0=P, mask=P, words=2, out=P, od=1, os=512, rows=4, n=1, nodes=64, qh=4, kvh=2, hd=128,
             page=16, mbps=4, scale=1.0, scratch=P + 4, size=1 << 40)
    a.update(over)
    return L.wkb_paged_attn_tree(*a.values(), None)


def commit(L, **over):
    a = dict(k=P + 8, v=P, layers=2, stride=1 << 20, pages=4, bt=P, slot=P, ctx=P + 64, path=P + 128, n_path=P + 192, max_path=4, n=1, kvh=2, hd=64, page=16, mbps=4, new_ctx=None)
    a.update(over)
    return L.wkb_paged_kv_commit(*a.values(), None)


# extents whose products wrap around in 64 bits
@pytest.mark.parametrize("over", [dict(qh=1 << 62, kvh=1 << 62, page=65536), dict(qh=1 << 62, kvh=1 << 60), dict(mbps=1 << 60), dict(mbps=(1 << 60) + 4),
                                  dict(words=1 << 58), dict(words=(1 << 32) + 2), dict(qs=1 << 61), dict(os=1 << 61)])
def test_attention_extents_that_wrap_around(L, over):
    assert attn(L, **over) == BAD


@pytest.mark.parametrize("over", [dict(mbps=1 << 60), dict(page=1 << 60, mbps=16), dict(layers=1 << 62), dict(layers=1 << 61, kvh=1 << 20, hd=1 << 10), dict(kvh=1 << 62)])
def test_commit_extents_that_wrap_around(L, over):
    assert commit(L, **over) == BAD


def test_the_calls_are_right_otherwise(L):
    assert attn(L) == MISALIGNED and commit(L) == MISALIGNED


def test_scratch_of_extents_that_wrap_around(L):
    assert L.wkb_paged_attn_tree_scratch_bytes(1 << 62, 4, 2, 128) == 0
    assert L.wkb_paged_attn_tree_scratch_bytes(4, 1 << 62, 1, 128) == 0
    assert L.wkb_paged_attn_tree_scratch_bytes(4, 4, 2, 1 << 60) == 0
    assert L.wkb_paged_attn_tree_scratch_bytes(4, 4, 2, 128) > 0


@pytest.mark.parametrize("new_ctx", [P + 4 * 7, P + 64 + 4, P + 64 - 4, P + 128, P + 128 + 4 * 31, P + 128 - 4 * 7, P + 512 + 4, P + 512 - 4 * 7])
def test_commit_into_an_array_that_it_reads(L, new_ctx):
    """Eight trees: slots at P, contexts at P + 64, paths of four entries at P + 128 .. P + 256, lengths at P + 512; the next
    contexts may share no element with any of them, since other blocks of the kernel still read it."""
    at = dict(n=8, slot=P, ctx=P + 64, path=P + 128, n_path=P + 512)
    assert commit(L, new_ctx=new_ctx, **at) == BAD
    for apart in (P - 32, P + 32, P + 96, P + 256, P + 480, P + 544):
        assert commit(L, new_ctx=apart, **at) == MISALIGNED


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38, -3e38])
def test_attention_scale_that_is_not_a_number_of_use(L, scale):
    """NaN would have been taken for the smallest scale there is, and infinite products with zeros are NaN everywhere."""
    assert attn(L, scale=scale) == BAD
    assert attn(L, scale=-1e30) == MISALIGNED and attn(L, scale=0.0) == MISALIGNED
