"""GPU tests of the speculative-decoding operators where they are easily wrong: values that are not finite in long contexts,
accuracy in the mean, refused calls."""
import math

import numpy as np
import pytest

from test_gpu_tree_decode import Case, dev, i32  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


# ---- V that is not finite -------------------------------------------------------------------------------------------

def plant(c, cache, t, pos, head, dim, what):
    cache[0, int(c.table[t, pos // c.page]), head, pos % c.page, dim] = what


@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("hd,kvh,nodes", [(64, 2, 5), (64, 1, 30), (128, 2, 9), (128, 1, 16)])
def test_not_finite_values_in_long_contexts(dev, hd, kvh, nodes, types):
    """Whatever the length: a column's NaN or infinities in the context reach every row, those of nodes the rows that see them."""
    import torch
    tq, to = ({"f32": torch.float32, "bf16": torch.bfloat16}[t] for t in types.split("-"))
    c = Case(dev, [(20011, nodes), (700, 3), (0, nodes), (4096, nodes)], 2 * kvh, kvh, hd, seed=nodes, q_dtype=tq)
    for t, pos, dim, what in [(0, 0, 3, math.inf), (0, 9000, 3, math.inf), (0, 12345, 7, math.nan), (0, 17, 20, -math.inf), (0, 19999, 21, math.inf),
                              (0, 20005, 22, -math.inf), (0, 20011 + 2, 23, math.inf), (0, 20011 + 3, 21, -math.inf), (1, 701, 5, math.nan),
                              (2, nodes - 1, 9, math.inf), (3, 4095, 11, -math.inf), (3, 4096 + nodes - 1, 12, math.nan)]:
        plant(c, c.kv.v, t, pos, kvh - 1, dim, what)
    out = torch.zeros((c.rows, 2 * kvh * hd), dtype=to, device="cuda")
    c.run(dev, out)
    c.check(out)
    assert dev.gemm_status() == 0


@pytest.mark.parametrize("hd,ctx", [(64, 150000), (128, 150000)])
def test_not_finite_values_in_long_pieces(dev, hd, ctx):
    """One block of the kernel works on 150 000 keys in one piece, and its other warps' waits do not run out while the results
    are mended.  All trees' tables repeat the same pages.  Expected: softmax over the pages' keys, each as often as it
    occurs; the tolerance is that of the other attention tests."""
    import torch
    n, pool, page = 148 * (2 if hd == 64 else 1), 512, 16
    g = torch.Generator(device="cuda").manual_seed(hd)
    kv = dev.PagedKV(1, pool, 1, hd, page)
    kv.k.normal_(generator=g); kv.v.normal_(generator=g)
    kv.v[0, 37, 0, 5, 3] = math.inf
    kv.v[0, 400, 0, 0, 60] = math.nan
    kv.v[0, 401, 0, 0, 61], kv.v[0, 401, 0, 1, 61] = -math.inf, math.inf
    mbps = -(-(ctx + 1) // page)
    table = torch.arange(mbps, dtype=torch.int32, device="cuda").remainder(pool).repeat(n, 1)
    q = torch.randn((n, hd), generator=g, device="cuda")
    out, scale = torch.zeros((n, hd), device="cuda"), 1.0 / math.sqrt(hd)
    dev.paged_attn_tree(q, hd, kv, 0, table, i32(np.arange(n)), i32(np.full(n, ctx)), i32(np.arange(n + 1)), i32(np.ones((n, 1))), out, 1, mbps, 1, scale,
                        dev.paged_attn_tree_scratch(1, 1, 1, hd))
    assert dev.gemm_status() == 0
    k, v = (x[0, :, 0].reshape(-1, hd).double() for x in (kv.k, kv.v))
    at = torch.arange(pool * page, device="cuda")
    count = ((ctx + 1 - at + pool * page - 1) // (pool * page)).double()
    s = q.double() @ k.T * scale
    p = torch.exp(s - s.amax(1, keepdim=True)) * count
    p /= p.sum(1, keepdim=True)
    fine = torch.isfinite(v)
    want, mag = p @ torch.where(fine, v, 0.0), p @ torch.where(fine, v, 0.0).abs()
    most = float((q.double().abs() @ k.abs().T).max()) * scale
    tol = 2.0 ** -14 * most + 2.0 ** -15 + (ctx + 1) * 2.0 ** -22
    ok = fine.all(0)
    assert bool(((out.double() - want).abs() <= tol * mag)[:, ok].all())
    assert bool((out[:, 3] == math.inf).all()) and bool(out[:, 60:62].isnan().all())


@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("gain", [1.0, 40.0])
@pytest.mark.parametrize("hd,group,page,trees", [(64, 1, 16, [(300, 100), (40, 70)]), (128, 1, 16, [(300, 100), (40, 70)]), (64, 4, 16, [(9000, 140), (2000, 3)]),
                                                 (128, 4, 16, [(9000, 140), (2000, 3)]), (128, 8, 16, [(30011, 40)]), (64, 2, 4, [(300, 20), (9, 9)])])
def test_infinities_in_the_context_whatever_the_tree_and_the_weights(dev, hd, group, page, trees, gain, types):
    """An infinity in a column gives that infinity in every row, for wide trees as for narrow ones, in a joined result as in one
    piece, and where the key's weight is below what f32 holds (gain 40: exp(-300))."""
    import torch
    tq, to = ({"f32": torch.float32, "bf16": torch.bfloat16}[t] for t in types.split("-"))
    c = Case(dev, trees, group, 1, hd, page, seed=hd + group, q_dtype=tq, q_gain=gain)
    for t, (ctx, nodes) in enumerate(trees):
        for dim, pos in enumerate([0, 3, 8, ctx // 3, ctx // 2, ctx - 1]):
            plant(c, c.kv.v, t, pos, 0, dim, math.inf if dim % 2 else -math.inf)
        plant(c, c.kv.v, t, 1, 0, 40, math.inf)
        plant(c, c.kv.v, t, ctx - 2, 0, 40, -math.inf)
        plant(c, c.kv.v, t, 2, 0, 41, math.nan)
        plant(c, c.kv.v, t, ctx, 0, 42, math.inf)
    out = torch.zeros((c.rows, group * hd), dtype=to, device="cuda")
    c.run(dev, out)
    c.check(out)
    assert dev.gemm_status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,group,nodes", [(64, 1, 12), (128, 4, 12), (128, 4, 50)])
def test_rows_with_nan_queries_beside_infinities_of_v(dev, hd, group, nodes, dtype):
    """A row whose query is NaN is NaN in every column, and its neighbours are what they are without it."""
    import torch
    tq = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    c = Case(dev, [(777, nodes), (3000, nodes)], group, 1, hd, seed=4, q_dtype=tq)
    for dim, pos in [(3, 5), (4, 777 + 1), (60, 776)]:
        plant(c, c.kv.v, 0, pos, 0, dim, math.inf)
    clean = torch.zeros((c.rows, group * hd), dtype=tq, device="cuda")
    c.run(dev, clean)
    c.check(clean)
    c.q[5] = math.nan
    c.q[nodes + 2, 7] = math.nan
    out = torch.zeros_like(clean)
    c.run(dev, out)
    assert bool(out[5].isnan().all()) and bool(out[nodes + 2, :hd].isnan().all())
    clean[5] = clean[nodes + 2, :hd] = out[5] = out[nodes + 2, :hd] = 0
    assert torch.equal(clean, out) and dev.gemm_status() == 0


# ---- commit ---------------------------------------------------------------------------------------------------------

def test_commit_of_a_broken_path_counts_what_was_moved(dev):
    """Where a path breaks off, the next context ends with the last node that was moved: what lies behind it is not the
    sequence's.  Breaks in the first eight nodes, in the second eight and at the first one; whole paths beside them."""
    import torch
    kv = dev.PagedKV(1, 12, 1, 64, 16)
    up = list(range(12))
    paths = [[0, 3, 3], [0, 2, 1], [0, 60, 61], [0, -4, 5], [0, 5, 2 ** 31 - 1], up[:9] + [9, 9, 10], up[:8] + [7, 9], up, [0], []]
    good = [2, 2, 1, 1, 2, 10, 8, 12, 1, 0]
    n = len(paths)
    path = np.full((n, 12), -1)
    for t, p in enumerate(paths):
        path[t, :len(p)] = p
    table = np.arange(12).reshape(1, 12).repeat(n, 0)[:, :3]      # (all broken or in place: the trees' moves do not meet)
    ctx = np.arange(n)
    for t in range(n):
        new = torch.full((1,), -9, dtype=torch.int32, device="cuda")
        dev.paged_kv_commit(kv, i32(table[t:t + 1]), i32([0]), i32(ctx[t:t + 1]), i32(path[t:t + 1]), i32([len(paths[t])]), 3, new_ctx=new)
        assert dev.gemm_status() == (0 if good[t] == len(paths[t]) else 31), t
        assert int(new) == ctx[t] + good[t], t


def test_commit_reports_a_length_beyond_the_path(dev):
    """n_path above max_path: the path's entries are moved and counted, and the length is reported."""
    import torch
    kv = dev.PagedKV(1, 3, 1, 64, 16)
    new = torch.zeros(1, dtype=torch.int32, device="cuda")
    for n_path, status in [(3, 0), (4, 31), (2 ** 31 - 1, 31)]:
        kv.k.copy_(torch.arange(48, device="cuda").view(1, 3, 1, 16, 1).expand_as(kv.k))
        dev.paged_kv_commit(kv, i32([[0, 1, 2]]), i32([0]), i32([20]), i32([[0, 4, 9]]), i32([n_path]), 3, new_ctx=new)
        assert dev.gemm_status() == status and int(new) == 23
        assert kv.k.view(48, 64)[20:24, 0].tolist() == [20, 24, 29, 23]


# ---- refused calls --------------------------------------------------------------------------------------------------

def attention_args(dev, **over):
    import torch
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")
    a = dict(q=z(3, 256, dt=torch.float32), q_row_stride=256, kv=dev.PagedKV(2, 4, 2, 64), layer=1, block_table=z(1, 4), tree_slot=z(1), tree_ctx=z(1), tree_row0=z(2),
             tree_mask=z(3, 1), out=z(3, 256, dt=torch.float32), q_heads=4, mbps=4, max_nodes=3, scale=1.0, scratch=dev.paged_attn_tree_scratch(3, 4, 2, 64))
    a.update(over)
    return a


def test_queries_whose_rows_are_not_dense_are_refused(dev):
    import torch
    f = lambda *s: torch.zeros(s, device="cuda")
    for good in (f(3, 256), f(3, 4, 64), f(3 * 256), f(3, 600)[:, 40:], f(3, 1, 256)):
        dev.paged_attn_tree(**attention_args(dev, q=good, q_row_stride=good.stride(0) if good.dim() > 1 else 256))
    for bad in (f(256, 3).t(), f(4, 3, 64).transpose(0, 1), f(3, 64, 4).transpose(1, 2), f(2 * 3 * 256)[::2], f(3, 512)[:, ::2], f(1).expand(3, 256), f(1)[0]):
        with pytest.raises(ValueError):
            dev.paged_attn_tree(**attention_args(dev, q=bad))
    for stride in (1 << 61, 1 << 62, (1 << 63) - 8, 257 * 8):
        with pytest.raises(ValueError):
            dev.paged_attn_tree(**attention_args(dev, q_row_stride=stride))


def test_a_block_table_without_rows_is_refused(dev):
    """No tree can have a row in it; the kernels would read behind it."""
    import torch
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    for empty in (z(0, 4), z(0)):
        with pytest.raises(ValueError):
            dev.paged_attn_tree(**attention_args(dev, block_table=empty))
        with pytest.raises(ValueError):
            dev.paged_kv_commit(dev.PagedKV(1, 2, 1, 64), empty, z(1), z(1), z(1, 3), z(1), 4)
        dev.paged_kv_commit(dev.PagedKV(1, 2, 1, 64), empty, z(0), z(0), z(0, 3), z(0), 4)      # nothing to do


# ---- vocabulary probabilities ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("cols", [1, 2, 3, 4, 31, 32, 33, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 16351, 16383, 50257])
@pytest.mark.parametrize("rows", [1, 3, 400])
def test_token_probs_bf16_rows_that_begin_and_end_in_a_word(dev, rows, cols):
    """Every parity of a row's first and last column: what lies in the other half of the words at its ends is not the row's
    (NaN, and a buffer that ends with the last column).  Tolerance as for all probabilities (2^-15 of the value)."""
    import torch
    rows = min(rows, (1 << 23) // cols)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    for first in (0, 1):
        for pitch in (cols, cols + 1):
            flat = torch.full((first + (rows - 1) * pitch + cols,), math.nan, dtype=torch.bfloat16, device="cuda")
            x = flat[first:].as_strided((rows, cols), (pitch, 1), first)
            x.copy_(torch.randn((rows, cols), generator=g, device="cuda") * 3)
            for t in (None, torch.zeros(rows, device="cuda")):
                got = dev.token_probs(x, t)
                if t is None:
                    want = torch.softmax(x.double(), 1)
                    assert bool(((got.double() - want).abs() <= want * 2.0 ** -15 + 1e-38).all())
                else:
                    assert torch.equal(got.argmax(1), (x == x.amax(1, keepdim=True)).double().argmax(1)) and bool((got.sum(1) == 1).all())


# ---- accuracy in the mean -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("trees,qh,kvh,hd", [([(200, 20)], 4, 2, 128), ([(257, 5)], 12, 12, 64), ([(700, 33), (1500, 61)], 8, 2, 128), ([(9001, 3)], 4, 4, 128), ([(5000, 64)], 8, 8, 64),
                                             ([(30011, 16)], 8, 1, 128), ([(20000, 9)], 8, 2, 64)])
@pytest.mark.parametrize("tq", ["f32", "bf16"])
def test_f32_results_in_the_mean(dev, trees, qh, kvh, hd, tq):
    """Norm of the error over the norm of the result, unit-normal inputs.  A query and a weight as two bf16 parts are off by at
    most 2^-16 of themselves; with scale 1 / sqrt(hd) a score is then off by 2^-16 in the mean and a weight by that and its own
    2^-16, independently from key to key, so a sum over the keys is off by 2^-15 of itself.  The tensor pipe's sums lose one
    part of 2^-24 a step at most, a step being 16 keys: keys * 2^-28 in all.  The bar tells a lost part at every length: weights
    of one bf16 part alone exceed it, by the same emulation, which the second assertion holds."""
    import torch
    c = Case(dev, trees, qh, kvh, hd, seed=hd, q_dtype={"f32": torch.float32, "bf16": torch.bfloat16}[tq])
    out = torch.zeros((c.rows, qh * hd), device="cuda")
    c.run(dev, out)
    want, _, _ = c.expected()
    bar = 2.0 ** -15 + max(n + k for n, k in trees) * 2.0 ** -28
    assert float((out.double() - want).norm() / want.norm()) <= bar
    ctx, nodes = trees[0]
    pos = np.arange(ctx)
    pg, off = (torch.from_numpy(a).cuda() for a in (c.table[0, pos // 16], pos % 16))
    k, v = (x[0][pg, 0, off].double() for x in (c.kv.k, c.kv.v))
    p = torch.softmax(c.q[:nodes, :hd].double() @ k.T * c.scale, 1)
    p = p / p.amax(1, keepdim=True)
    short = (p.bfloat16().double() @ v) / p.sum(1, keepdim=True)
    full = (p @ v) / p.sum(1, keepdim=True)
    assert float((short - full).norm() / full.norm()) > bar


# ---- Python level ---------------------------------------------------------------------------------------------------

def test_a_full_launch_queue_does_not_stop_other_threads(dev):
    """A thread that launches faster than the GPU works waits in the driver, and the other threads go on meanwhile, as with
    the library's other calls: for most of a second the queue here is blocked by one kernel, and the longest pause of
    the counting thread stays below a third of that."""
    import threading
    import time
    import torch
    x, out = torch.zeros((1, 8), device="cuda"), torch.empty((1, 8), device="cuda")
    dev.token_probs(x, None, out)
    torch.cuda.synchronize()
    blocked = []

    def launch():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(1 << 30)
            blocked.append(time.perf_counter())
            for _ in range(6000):
                dev.token_probs(x, None, out)
            stream.synchronize()

    t0 = time.perf_counter()
    worker = threading.Thread(target=launch)
    worker.start()
    last, pause = None, 0.0
    while worker.is_alive():
        time.sleep(0.0005)
        now = time.perf_counter()
        if blocked:
            pause = max(pause, now - (last or blocked[0]))
            last = now
    whole = time.perf_counter() - t0
    assert whole > 0.45, "the GPU was not blocked"
    assert pause < 0.15, (pause, whole)


def test_errors_of_torch_keep_their_types(dev):
    """Results that do not fit the device: torch.OutOfMemoryError as from torch's own calls (logits of 2^20 equal rows, whose
    probabilities would take 2 TB)."""
    import torch
    x = torch.zeros(1 << 19, device="cuda").expand(1 << 20, 1 << 19)
    with pytest.raises(torch.OutOfMemoryError):
        dev.token_probs(x)
