"""GPU parity of the speculative-decoding operators against plain f64 implementations: attention of draft trees over the
paged cache, vocabulary probabilities, verification of drafted tokens, commit of the accepted tokens' K / V.

Attention bars, with A = scale * max sum |q||k| of the case and mag = sum_p softmax_p |v_p| per element:
  f32 out   a query as the sum of two bf16 parts is off by at most 2^-8 * 2^-8 = 2^-16 of each element, and f32 sums of
            head_dim <= 128 terms by 2^-17 of sum |q||k|: scores are off by at most 2^-15 A, the weights by that on both
            sides of the quotient; a weight as two bf16 parts by 2^-16 on both sides; the sums over the keys by keys * 2^-23.
            Together (2^-14 A + 2^-15 + keys * 2^-22) mag.
  bf16 out  additionally 2^-8 for a weight rounded to bf16, on both sides of the quotient, and 2^-8 for the result: + (2^-7 +
            2^-8) mag."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from wukong_b200 import _lib, device
    _lib.require_gpu()
    return device


def i32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def random_trees(counts, rng, reach=4):
    row0 = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    parent = np.full(row0[-1], -1, np.int64)
    for t, k in enumerate(counts):
        for i in range(1, k):
            parent[row0[t] + i] = rng.integers(max(0, i - reach), i)
    return row0, parent


def paged(lengths, page, mbps, rng, spare=2):
    need = [-(-n // page) for n in lengths]
    pool = rng.permutation(sum(need) + spare)
    table = np.zeros((len(lengths), mbps), np.int64)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = pool[at:at + k]
        at += k
    return table, len(pool)


class Case:
    """Trees [(ctx, nodes), ...] over a paged cache whose unused tokens are NaN."""

    def __init__(self, dev, trees, qh, kvh, hd, page=16, seed=0, q_dtype=None, masks="tree", q_gain=1.0, pad_rows=0):
        import torch
        rng = np.random.default_rng(seed)
        self.trees, self.qh, self.kvh, self.hd, self.page = trees, qh, kvh, hd, page
        counts = [n for _, n in trees]
        self.row0, parent = random_trees(counts, rng)
        self.rows = int(self.row0[-1]) + pad_rows
        self.max_nodes = max(1, max(counts))
        lengths = [c + n for c, n in trees]
        self.mbps = max(1, max(-(-n // page) for n in lengths)) + 1
        self.table, self.pages = paged(lengths, page, self.mbps, rng)
        if masks == "tree":
            mask = dev.tree_layout(parent, self.row0)[0]
        else:
            mask = rng.integers(0, 1 << 32, (int(self.row0[-1]), -(-self.max_nodes // 32)), dtype=np.uint64).astype(np.uint32).view(np.int32)
            if masks == "sparse":
                mask = mask & rng.integers(0, 2, mask.shape[0]).astype(np.int32)[:, None] & np.roll(mask, 1, 0)
        self.mask = np.concatenate([mask, np.full((pad_rows, mask.shape[1]), -1, np.int32)])
        self.scale = 1.0 / math.sqrt(hd)
        self.kv = dev.PagedKV(1, self.pages, kvh, hd, page)
        self.kv.k.fill_(float("nan")); self.kv.v.fill_(float("nan"))
        k, v = (torch.from_numpy(rng.standard_normal((sum(lengths) or 1, kvh, hd)).astype(np.float32)).cuda().bfloat16() for _ in range(2))
        at = 0
        for s, n in enumerate(lengths):
            pos = np.arange(n)
            pg, off = (torch.from_numpy(a).cuda() for a in (self.table[s, pos // page], pos % page))
            self.kv.k[0][pg, :, off] = k[at:at + n]
            self.kv.v[0][pg, :, off] = v[at:at + n]
            at += n
        q = torch.from_numpy((rng.standard_normal((self.rows, qh * hd)) * q_gain).astype(np.float32)).cuda()
        self.q = q.to(q_dtype or torch.float32)
        self.slot, self.ctx = np.arange(len(trees)), np.array([c for c, _ in trees])

    def run(self, dev, out, q=None, stride=None, scratch=None):
        q = self.q if q is None else q
        if scratch is None:
            scratch = dev.paged_attn_tree_scratch(self.max_nodes, self.qh, self.kvh, self.hd)
        return dev.paged_attn_tree(q, stride or q.stride(0), self.kv, 0, i32(self.table), i32(self.slot), i32(self.ctx), i32(self.row0), i32(self.mask), out,
                                   self.qh, self.mbps, self.max_nodes, self.scale, scratch)

    def expected(self):
        """(out, mag) in f64 and the largest scale * sum |q||k|; a key that a row does not see takes no part at all."""
        import torch
        want = torch.zeros((self.rows, self.qh * self.hd), dtype=torch.float64, device="cuda")
        mag, most, group = torch.zeros_like(want), 0.0, self.qh // self.kvh
        for t, (ctx, nodes) in enumerate(self.trees):
            if not nodes:
                continue
            a, pos = int(self.row0[t]), np.arange(ctx + nodes)
            pg, off = (torch.from_numpy(x).cuda() for x in (self.table[t, pos // self.page], pos % self.page))
            seen = np.ones((nodes, ctx + nodes), bool)
            words = self.mask[a:a + nodes].view(np.uint32)
            for j in range(nodes):
                seen[:, ctx + j] = (words[:, j // 32] >> np.uint32(j % 32)) & 1
            seen = torch.from_numpy(seen).cuda()
            for h in range(self.qh):
                k, v = (x[0][pg, h // group, off].double() for x in (self.kv.k, self.kv.v))
                q = self.q[a:a + nodes, h * self.hd:(h + 1) * self.hd].double()
                s = torch.where(seen, q @ torch.nan_to_num(k).T * self.scale, -math.inf)
                bad = (k != k).any(1)
                s = torch.where(seen & bad[None], math.nan, s)
                most = max(most, float((q.abs() @ torch.nan_to_num(k, posinf=0.0, neginf=0.0).abs().T).max()) * self.scale)
                top = s.amax(1, keepdim=True)
                p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
                total = p.sum(1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                fine = torch.isfinite(v)
                o = p @ torch.where(fine, v, 0.0)
                for j in torch.nonzero(~fine.all(1)).flatten().tolist():
                    see = seen[:, j] & (p[:, j] != 0)
                    o[see] += torch.where(fine[j], 0.0, v[j])[None]
                want[a:a + nodes, h * self.hd:(h + 1) * self.hd] = o
                mag[a:a + nodes, h * self.hd:(h + 1) * self.hd] = p @ torch.where(fine, v, 0.0).abs()
        return want, mag, most

    def check(self, got, expected=None):
        import torch
        want, mag, most = expected or self.expected()
        keys = max(c + n for c, n in self.trees)
        tol = 2.0 ** -14 * most + 2.0 ** -15 + keys * 2.0 ** -22 + (2.0 ** -7 + 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0)
        live = int(self.row0[-1])
        got, want, mag = got.double()[:live], want[:live], mag[:live]
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(got))
        assert torch.equal(torch.isnan(want), torch.isnan(got))
        assert torch.equal(want[~fine & ~torch.isnan(want)], got[~fine & ~torch.isnan(want)])
        err = (got - want).abs()[fine]
        assert bool((err <= tol * mag[fine] + 1e-12).all()), float((err / (mag[fine] + 1e-9)).max() / tol)


SHAPES = [   # trees, q heads, kv heads, head_dim, page
    ([(0, 1)], 1, 1, 64, 16),
    ([(0, 1), (1, 1), (127, 1), (128, 1), (129, 3)], 12, 12, 64, 16),
    ([(257, 5)], 12, 12, 64, 16),
    ([(100, 16), (5, 0), (300, 17), (16, 1), (0, 9)], 8, 2, 128, 16),
    ([(700, 33), (90, 64)], 32, 8, 128, 16),
    ([(120, 16), (112, 16), (1500, 61)], 16, 2, 128, 16),
    ([(64, 129), (640, 256)], 2, 2, 128, 16),
    ([(333, 256)], 4, 1, 64, 16),
    ([(250, 200), (0, 130)], 8, 1, 128, 16),
    ([(5000, 64)], 8, 8, 64, 16),
    ([(9001, 3), (17, 30)], 4, 4, 128, 16),
    ([(200, 20), (77, 5)], 4, 2, 64, 4),
    ([(200, 20), (77, 5)], 4, 2, 128, 8),
    ([(411, 20), (77, 5)], 4, 2, 128, 32),
    ([(411, 20), (77, 5)], 2, 2, 64, 64),
    ([(900, 20), (177, 5)], 2, 1, 128, 256),
    ([(int(c), int(n)) for c, n in zip(range(0, 900, 9), list(range(17)) * 6)], 4, 1, 64, 16),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-bf16", "bf16-f32"])
def test_tree_attention_matches_f64(dev, shape, types):
    import torch
    trees, qh, kvh, hd, page = SHAPES[shape]
    tq, to = ({"f32": torch.float32, "bf16": torch.bfloat16}[t] for t in types.split("-"))
    c = Case(dev, trees, qh, kvh, hd, page, seed=shape, q_dtype=tq, q_gain=2.0)
    out = torch.full((c.rows, qh * hd), 7.0, dtype=to, device="cuda")
    c.run(dev, out)
    c.check(out)
    again = torch.full((c.rows, qh * hd), -3.0, dtype=to, device="cuda")
    c.run(dev, again)
    assert torch.equal(out, again), "run-to-run identical"


@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-bf16"])
@pytest.mark.parametrize("hd,kvh,group,nodes", [(128, 8, 4, 16), (128, 4, 8, 61), (128, 8, 1, 5), (64, 12, 1, 16), (64, 6, 2, 100)])
def test_tree_attention_batches_with_many_units(dev, hd, kvh, group, nodes, types):
    """More units than the GPU works on at a time: a block of the kernel goes through several trees and heads, whole and in pieces."""
    import torch
    rng = np.random.default_rng(hd + nodes)
    trees = [(int(c), int(n)) for c, n in zip(rng.integers(0, 1500, 48), rng.integers(1, nodes + 1, 48))]
    tq, to = ({"f32": torch.float32, "bf16": torch.bfloat16}[t] for t in types.split("-"))
    c = Case(dev, trees, kvh * group, kvh, hd, seed=nodes, q_dtype=tq, q_gain=2.0)
    expected = c.expected()
    for _ in range(3):
        out = torch.full((c.rows, kvh * group * hd), 7.0, dtype=to, device="cuda")
        c.run(dev, out)
        c.check(out, expected)


@pytest.mark.parametrize("masks", ["random", "sparse"])
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_attention_any_mask_and_rows_that_see_nothing(dev, masks, hd):
    import torch
    c = Case(dev, [(0, 40), (130, 70), (0, 1), (255, 33)], 4, 2, hd, seed=3, masks=masks)
    c.mask[0] = 0                       # ctx 0 and no node: sees nothing
    c.mask[110:112] = 0
    out = torch.full((c.rows, 4 * hd), float("nan"), device="cuda")
    c.run(dev, out)
    c.check(out)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("hd,kvh", [(64, 1), (128, 2)])
def test_tree_attention_keeps_hidden_nonfinite_values_out(dev, hd, kvh):
    """NaN and infinities in nodes that a row does not see stay out of it; the rows that do see them get them."""
    import torch
    for seed, (ctx, nodes) in enumerate([(37, 24), (130, 60), (120, 24), (700, 140)]):
        c = Case(dev, [(ctx, nodes), (50, 3)], 4, kvh, hd, seed=seed)
        for node, what, which in [(5, math.nan, "v"), (9, math.inf, "v"), (nodes - 1, -math.inf, "v"), (11, math.nan, "k")]:
            pos = ctx + node
            cache = c.kv.v if which == "v" else c.kv.k
            cache[0, int(c.table[0, pos // 16]), kvh - 1, pos % 16, (3 + node) % hd] = what
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.zeros((c.rows, 4 * hd), dtype=dtype, device="cuda")
            c.run(dev, out)
            assert bool(torch.isfinite(out).all(1).any()) and not bool(torch.isfinite(out).all())
            c.check(out)


def test_tree_attention_large_scores_and_masked_extremes(dev):
    """Scores of several hundred: the running maximum has to move, and the largest scores sit in nodes that most rows do not see."""
    import torch
    c = Case(dev, [(300, 30), (1000, 12)], 4, 2, 128, seed=8, q_gain=30.0)
    for node in (3, 17, 29):
        pos = 300 + node
        c.kv.k[0, int(c.table[0, pos // 16]), :, pos % 16] *= 40.0
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.zeros((c.rows, 4 * 128), dtype=dtype, device="cuda")
        c.run(dev, out)
        c.check(out)


def test_tree_attention_leaves_other_rows_and_takes_strides(dev):
    import torch
    hd, qh = 64, 4
    c = Case(dev, [(40, 6), (300, 12), (9, 3)], qh, 2, hd, seed=2, pad_rows=5)
    c.slot[1] = -1                                             # switched off
    wide_q = torch.full((c.rows, 2 * qh * hd + 8), float("nan"), device="cuda")
    wide_q[:, 8:8 + qh * hd] = c.q
    wide_o = torch.full((c.rows, qh * hd + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    c.run(dev, wide_o[:, 8:8 + qh * hd], q=wide_q[:, 8:], stride=wide_q.stride(0))
    assert bool((wide_o[:, :8] == 7).all()) and bool((wide_o[:, 8 + qh * hd:] == 7).all())
    assert bool((wide_o[int(c.row0[1]):int(c.row0[2])] == 7).all()), "a tree that is switched off"
    assert bool((wide_o[int(c.row0[-1]):] == 7).all()), "rows behind the last tree"
    got = wide_o[:, 8:8 + qh * hd].clone()
    want, mag, most = c.expected()
    off = slice(int(c.row0[1]), int(c.row0[2]))
    want[off], got[off] = 0, 0
    c.check(got, (want, mag, most))


def test_tree_attention_context_past_the_table_row(dev):
    """Positions that the block-table row does not cover are not seen, and a table entry past the cache is a page of zeros."""
    import torch
    c = Case(dev, [(40, 4)], 2, 1, 64, seed=5)
    c.mbps = 2
    c.table = c.table[:, :2]
    out = torch.zeros((c.rows, 2 * 64), device="cuda")
    c.run(dev, out)
    c.trees, c.mask = [(32, 4)], np.zeros_like(c.mask)           # 32 covered positions, no node among them
    c.table = np.concatenate([c.table, c.table], 1)
    c.check(out)
    d = Case(dev, [(40, 4)], 2, 1, 64, seed=5)
    page = int(d.table[0, 1])
    d.table[0, 1] = d.pages + 1000000
    d.run(dev, out)
    d.table[0, 1] = page
    d.kv.k[0, page] = 0; d.kv.v[0, page] = 0
    d.check(out)


def test_cache_of_more_than_four_gigabytes(dev):
    """Pages beyond 2^32 bytes of a slab, in the attention and in the commit."""
    import torch
    small = Case(dev, [(300, 12), (40, 5)], 8, 8, 128, seed=13)
    pages = 150000                                        # x 8 heads x 16 tokens x 128 x 2 bytes = 4.9 GB a slab
    big = dev.PagedKV(1, 1, 8, 128)
    big.num_pages = pages
    big.k, big.v = (torch.empty((1, pages, 8, 16, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for at, used in ((pages - small.pages, small.kv), ):
        big.k[0, at:at + small.pages] = used.k[0]
        big.v[0, at:at + small.pages] = used.v[0]
    expected = small.expected()
    small.kv, small.table = big, small.table + pages - small.pages
    out = torch.zeros((small.rows, 8 * 128), device="cuda")
    small.run(dev, out)
    small.check(out, expected)
    page, off = int(small.table[0, (300 + 7) // 16]), (300 + 7) % 16
    want = big.k[0, page, :, off].clone()
    dev.paged_kv_commit(big, i32(small.table), i32([0, 1]), i32([300, 40]), i32([[0, 7, -1], [0, -1, -1]]), i32([2, 1]), small.mbps)
    assert torch.equal(big.k[0, int(small.table[0, 301 // 16]), :, 301 % 16], want) and dev.gemm_status() == 0


def test_tree_attention_one_chain_equals_decode(dev):
    """A chain's rows are ordinary decode rows with ctx + i + 1 visible keys."""
    import torch
    qh, kvh, hd = 8, 2, 128
    c = Case(dev, [(500, 9), (31, 4)], qh, kvh, hd, seed=6)
    c.mask = np.concatenate([(2 << np.arange(9)) - 1, (2 << np.arange(4)) - 1]).astype(np.int32)[:, None]
    out = torch.zeros((c.rows, qh * hd), device="cuda")
    c.run(dev, out)
    ctx = np.concatenate([500 + 1 + np.arange(9), 31 + 1 + np.arange(4)])
    dec = torch.zeros_like(out)
    dev.paged_attn_decode(c.q, qh * hd, c.kv, 0, i32(c.table), i32(np.repeat([0, 1], [9, 4])), i32(ctx), dec, c.rows, qh, c.mbps, 512, c.scale,
                          dev.paged_attn_scratch(c.rows, qh, hd, 512))
    _, mag, _ = c.expected()
    assert bool(((out - dec).abs() <= 2.0 ** -6 * mag).all())


def test_tree_attention_captured_replays_with_new_trees(dev):
    """One captured graph follows new extents, masks and tables; a second stream with its own scratch runs beside it."""
    import torch
    trees = [[(60, 7), (400, 30)], [(399, 30), (3, 1)], [(0, 12), (0, 0)]]
    cases = [Case(dev, t, 8, 2, 128, seed=20 + i, pad_rows=40) for i, t in enumerate(trees)]
    mbps, pages, rows, words = 40, max(c.pages for c in cases), max(c.rows for c in cases), 1
    kv = dev.PagedKV(1, pages, 2, 128)
    q, out = torch.zeros((rows, 1024), device="cuda"), torch.zeros((rows, 1024), device="cuda")
    table, slot, ctx, row0, mask = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((2, mbps), (2,), (2,), (3,), (rows, words)))
    scratch = dev.paged_attn_tree_scratch(32, 8, 2, 128)
    call = lambda o, sc: dev.paged_attn_tree(q, 1024, kv, 0, table, slot, ctx, row0, mask, o, 8, mbps, 32, cases[0].scale, sc)
    call(out, scratch)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call(out, scratch)
    side, out2, scratch2 = torch.cuda.Stream(), torch.zeros_like(out), dev.paged_attn_tree_scratch(32, 8, 2, 128)
    for c in cases:
        kv.k[:, :c.pages] = c.kv.k; kv.v[:, :c.pages] = c.kv.v
        table.zero_(); table[:, :c.mbps] = i32(c.table)
        slot.copy_(i32(c.slot)); ctx.copy_(i32(c.ctx)); row0.copy_(i32(c.row0)); mask[:c.rows] = i32(c.mask)
        q[:c.rows] = c.q
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            call(out2, scratch2)
        torch.cuda.synchronize()
        assert torch.equal(out[:int(c.row0[-1])], out2[:int(c.row0[-1])])
        c.check(out[:c.rows])
    del g


# ---- vocabulary probabilities ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 31), (5, 257), (2, 1000), (7, 4099), (3, 32000), (5, 50257), (1, 131073), (300, 515), (2, 270001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_probs_match_f64(dev, rows, cols, dtype):
    """The exponent (x - max) * log2(e) / t is off by 3 roundings of at most 2^-24 of itself (its magnitude is below 100
    here, so 2^-24 * 300 of the value), the exponential and the quotient by 2^-22 each, the sum by (32 + log2 cols) * 2^-24."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows * 1000 + cols)
    x = (torch.randn((rows, cols + 3), generator=g, device="cuda") * 3).to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])[:, :cols]
    t = torch.rand(rows, generator=g, device="cuda") + 0.5
    t[1::3] = 0.0
    got = dev.token_probs(x, t)
    z = x.double() / torch.where(t > 0, t, 1.0).double()[:, None]
    want = torch.softmax(z, 1)
    cold = torch.nonzero(t <= 0).flatten().tolist()
    for r in cold:
        want[r] = 0
        want[r, int(torch.nonzero(x[r] == x[r].max())[0])] = 1
    assert bool(((got.double() - want).abs() <= want * (2.0 ** -15) + 1e-38).all())
    for r in cold:
        assert torch.equal(got[r].double(), want[r])
    if dtype == "f32":      # in place, odd pitch, no temperatures
        y = x.clone() if cols == 1 else x
        plain = torch.softmax(x.double(), 1)
        dev.token_probs(y, None, out=y)
        assert bool(((y.double() - plain).abs() <= plain * 2.0 ** -15 + 1e-38).all())


@pytest.mark.parametrize("rows,cols", [(300, 8192), (300, 16320), (300, 16384), (160, 32768), (3, 65536), (150, 65281), (150, 131072), (2, 262113)])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_probs_full_runs(dev, rows, cols, shift, dtype):
    """Rows that fill every register of their threads, starting on a word of two bf16 and in the middle of one: the last
    column counts (it holds a large part of the row), and the columns beside the row do not (they are NaN).  Tolerance as above."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows + cols + shift)
    wide = torch.full((rows, cols + 2 + shift), math.nan, device="cuda", dtype={"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    x = wide[:, shift:shift + cols]
    x.copy_(torch.randn((rows, cols), generator=g, device="cuda") * 3)
    x[:, 0] = x[:, -1] = 13.0
    got = dev.token_probs(x, None)
    want = torch.softmax(x.double(), 1)
    assert bool(((got.double() - want).abs() <= want * 2.0 ** -15 + 1e-38).all())


def test_token_probs_special_rows(dev):
    import torch
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, 1.0, -inf, 1.0], [-inf] * 4, [0.0, nan, 1.0, 2.0], [inf, 0.0, 1.0, 2.0], [5.0, 7.0, 7.0, -inf], [-inf] * 4, [1.0, inf, inf, 0.0],
                      [1e30, -1e30, 0.0, 1e30], [1.0, 2.0, 3.0, 4.0]], device="cuda")
    t = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0, 0.0, 0.0, 1e-40, nan], device="cuda")
    got = dev.token_probs(x, t).cpu()
    assert got[0].tolist() == [0.0, 0.5, 0.0, 0.5]
    assert got[1].tolist() == [0.0] * 4
    assert bool(got[2].isnan().all()) and bool(got[3].isnan().all()) and bool(got[8].isnan().all())
    assert got[4].tolist() == [0.0, 1.0, 0.0, 0.0]
    assert got[5].tolist() == [0.0] * 4
    assert got[6].tolist() == [0.0, 1.0, 0.0, 0.0]
    assert got[7].tolist() == [0.5, 0.0, 0.0, 0.5]


# ---- verification ---------------------------------------------------------------------------------------------------

def weight(x):
    x = np.asarray(x, np.float32)
    return np.where((x > 0) & np.isfinite(x), x, 0).astype(np.float64)


def unit(u):
    return 0.0 if u != u else float(min(1.0, max(0.0, u)))


def verify_plain(probs, draft, token, parent, row0, u_node, u_final, max_path):
    n = len(row0) - 1
    path, tokens, n_path = np.full((n, max_path), -1), np.full((n, max_path), -1), np.zeros(n, int)
    for t in range(n):
        a, count = int(row0[t]), int(row0[t + 1] - row0[t])
        if count == 0:
            continue
        walk, cur, done = [0], 0, False
        while not done:
            r, z, done = weight(probs[a + cur]), 1.0, True
            for c in [i for i in range(cur + 1, count) if parent[a + i] == cur] if len(walk) < max_path else []:
                x = int(token[a + c])
                inside = 0 <= x < r.size
                q = 1.0 if draft is None else float(weight(draft[a + cur, x])) if inside else 0.0
                rx = r[x] if inside else 0.0
                if unit(u_node[a + c]) * q * z < rx:
                    walk.append(c)
                    cur, done = c, False
                    break
                if draft is None:
                    z -= rx
                    if inside:
                        r[x] = 0
                else:
                    r = np.maximum(r - z * weight(draft[a + cur]), 0)
                    z = r.sum()
        mass = np.cumsum(r)
        pick = -1
        if mass[-1] > 0:
            over = np.nonzero((mass > unit(u_final[t]) * mass[-1]) & (r > 0))[0]
            pick = over[0] if over.size else np.nonzero(r > 0)[0][-1]
        n_path[t] = len(walk)
        path[t, :len(walk)] = walk
        tokens[t, :len(walk)] = [token[a + i] for i in walk[1:]] + [pick]
    return path, n_path, tokens


def verify_case(dev, counts, cols, drafted, seed, max_path=None, noise=1.0, ld_extra=0):
    import torch
    rng = np.random.default_rng(seed)
    row0, parent = random_trees(counts, rng)
    rows, most = int(row0[-1]), max(1, max(counts))
    soft = lambda x: (np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)).astype(np.float32)
    base = rng.standard_normal((rows, cols)) * 2
    probs, draft = soft(base), soft(base + noise * rng.standard_normal((rows, cols)))
    token = rng.integers(0, cols, rows)
    for t in range(len(counts)):
        for i in range(int(row0[t]) + 1, int(row0[t + 1])):
            p = int(row0[t] + parent[i])
            token[i] = rng.choice(cols, p=draft[p].astype(np.float64) / draft[p].astype(np.float64).sum()) if cols <= 5000 else \
                np.argsort(-draft[p])[int(rng.integers(0, 3))]
    u_node, u_final = rng.random(rows).astype(np.float32), rng.random(len(counts)).astype(np.float32)
    return probs, draft if drafted else None, token, parent, row0, u_node, u_final, max_path or most, most


def verify_run(dev, probs, draft, token, parent, row0, u_node, u_final, max_path, most, pitch=0):
    import torch
    f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
    def rows(a):
        if a is None:
            return None
        wide = torch.full((a.shape[0], a.shape[1] + pitch), math.nan, device="cuda")
        wide[:, :a.shape[1]] = f(a)
        return wide[:, :a.shape[1]]
    got = dev.tree_verify(rows(probs), rows(draft), i32(token), i32(parent), i32(row0), f(u_node), f(u_final), most, max_path)
    path, n_path, tokens = (x.cpu().numpy() for x in got)
    return path, n_path, tokens


@pytest.mark.parametrize("counts,cols", [([1], 1), ([5], 2), ([1, 0, 7, 3], 31), ([16, 5, 16, 1, 9], 1000), ([5], 50257), ([24, 7], 32000), ([256, 64], 515),
                                         ([3], 131073), ([8] * 70, 200), ([4] * 300, 37), ([6, 6, 6], 270001)])
@pytest.mark.parametrize("drafted", [True, False])
def test_tree_verify_matches_f64(dev, counts, cols, drafted):
    for seed, noise in [(1, 1.0), (2, 0.1), (3, 3.0)]:
        if cols > 50000 and seed > 1:
            continue
        for pitch in (0, 5):
            for limit in (None, 2 if max(counts) > 2 else None):
                c = verify_case(dev, counts, cols, drafted, seed * 100 + cols % 97, limit, noise)
                want = verify_plain(*c[:8])
                got = verify_run(dev, *c, pitch=pitch)
                for w, g, what in zip(want, got, ("path", "n_path", "tokens")):
                    assert np.array_equal(w, g), (what, seed, pitch, limit)


def test_tree_verify_edges(dev):
    """Random numbers at and outside the ends of [0, 1], NaN and negative weights, rows without mass, tokens outside the
    vocabulary, a sibling offered twice, equal distributions."""
    rng = np.random.default_rng(4)
    cols, counts = 40, [6] * 12
    probs, draft, token, parent, row0, u_node, u_final, max_path, most = verify_case(dev, counts, cols, True, 5)
    u_final[:6] = [0.0, 1.0, math.nan, -2.0, 5.0, 1.0 - 2.0 ** -24]
    u_node[::5] = 0.0
    u_node[3::7] = 1.0
    u_node[4::11] = math.nan
    probs[row0[2]:row0[3]] = 0.0                                   # no mass anywhere
    probs[row0[3], ::3] = -1.0
    probs[row0[3], 1] = math.nan
    probs[row0[4], 5] = math.inf
    draft[row0[5], 7] = math.nan
    token[row0[6]:row0[7]] = [0, -1, cols, 3, 2 ** 30, 5]
    parent[row0[7]:row0[8]] = [-1, 0, 0, 0, 0, 0]                  # five siblings, the same token
    token[row0[7]:row0[8]] = 9
    draft[row0[8]:row0[9]] = probs[row0[8]:row0[9]]
    probs[row0[9]] = 0.0
    probs[row0[9], 17] = 1.0                                       # all mass on one token, which is offered and refused
    parent[row0[9] + 1], token[row0[9] + 1], u_node[row0[9] + 1] = 0, 17, 1.0
    parent[row0[10]:row0[11]] = [5, 3, 4, -7, 99, 0]               # no proper tree: forward and wild parents are no children
    for d in (draft, None):
        c = (probs, d, token, parent, row0, u_node, u_final, max_path)
        want, got = verify_plain(*c), verify_run(dev, *c, most)
        for w, g, what in zip(want, got, ("path", "n_path", "tokens")):
            assert np.array_equal(w, g), (what, d is None, np.nonzero((w != g).reshape(len(counts), -1).any(1)))


@pytest.mark.parametrize("drafted", [True, False])
def test_tree_verify_emits_the_targets_distribution(dev, drafted):
    """The first emitted token of many identical trees follows the target: chi-square over 6 tokens, 20 000 draws.  With 5
    degrees of freedom a right sampler exceeds 40 with probability 1.5e-7."""
    n, cols = 20000, 6
    rng = np.random.default_rng(12)
    p = np.array([0.4, 0.25, 0.15, 0.1, 0.07, 0.03], np.float32)
    q = np.array([0.1, 0.1, 0.3, 0.3, 0.1, 0.1], np.float32)
    counts, parent = [4] * n, np.tile([-1, 0, 0, 0], n)
    row0 = np.arange(n + 1) * 4
    token = rng.choice(cols, (n, 4), p=q.astype(np.float64) / q.astype(np.float64).sum()) if drafted else np.tile([0, 2, 4, 1], (n, 1))
    u = rng.random(5 * n).astype(np.float32)
    path, n_path, tokens = verify_run(dev, np.tile(p, (4 * n, 1)), np.tile(q, (4 * n, 1)) if drafted else None, token.reshape(-1), parent, row0, u[:4 * n],
                                      u[4 * n:], 4, 4)
    seen = np.bincount(tokens[:, 0], minlength=cols)
    chi2 = ((seen - n * p) ** 2 / (n * p)).sum()
    assert chi2 < 40, chi2


# ---- commit ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("layers,kvh,hd,page", [(1, 1, 64, 16), (12, 12, 64, 16), (3, 2, 128, 4), (2, 5, 72, 32), (5, 3, 8, 1)])
def test_kv_commit_moves_the_path(dev, layers, kvh, hd, page):
    import torch
    rng = np.random.default_rng(layers * 10 + hd)
    n, nodes = 7, 40
    ctx = np.array([0, 1, 15, 16, 33, 100, 64])
    table, pages = paged([int(c) + nodes for c in ctx], page, -(-(int(ctx.max()) + nodes) // page), rng)
    kv = dev.PagedKV(layers, pages, kvh, hd, page)
    for x in (kv.k, kv.v):
        x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
    max_path = 40
    path, n_path = np.full((n, max_path), -1), np.array([1, 2, 5, 40, 3, 12, 0])
    for t in range(n):
        k = int(n_path[t])
        if k:
            path[t, :k] = np.concatenate([[0], np.sort(rng.permutation(np.arange(1, nodes))[:k - 1])])
    slot = np.arange(n)
    slot[4] = -1                                                  # switched off
    want = [x.clone() for x in (kv.k, kv.v)]
    for t in range(n):
        for i in range(1, int(n_path[t])):
            if slot[t] < 0:
                continue
            s, d = int(ctx[t] + path[t, i]), int(ctx[t]) + i
            for x in want:
                x[:, int(table[t, d // page]), :, d % page] = x[:, int(table[t, s // page]), :, s % page].clone()
    new_ctx = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    dev.paged_kv_commit(kv, i32(table), i32(slot), i32(ctx), i32(path), i32(n_path), table.shape[1], new_ctx=new_ctx)
    assert torch.equal(kv.k, want[0]) and torch.equal(kv.v, want[1])
    expect = ctx + n_path
    expect[4] = -5
    assert new_ctx.tolist() == expect.tolist()
    assert dev.gemm_status() == 0


def test_kv_commit_refuses_bad_paths(dev):
    """A path that does not ascend, or leaves the table or the cache, ends the tree's moves there and is reported."""
    import torch
    rng = np.random.default_rng(1)
    kv = dev.PagedKV(2, 6, 2, 64, 16)
    kv.k.copy_(torch.from_numpy(rng.standard_normal(kv.k.shape).astype(np.float32)))
    table = np.array([[0, 1, 2], [3, 4, 1 << 30]])
    for path, moved in [([0, 3, 3], 1), ([0, 2, 1], 1), ([0, 60, 61], 0), ([0, -4, 5], 0), ([0, 5, 2 ** 31 - 1], 1)]:
        before = kv.k.clone()
        dev.paged_kv_commit(kv, i32(table), i32([0]), i32([1]), i32([path]), i32([3]), 3)
        assert dev.gemm_status() == 31, path
        if moved:
            before[:, 0, :, 2] = before[:, (1 + path[1]) // 16, :, (1 + path[1]) % 16].clone()
        assert torch.equal(kv.k, before), path
    before = kv.k.clone()
    dev.paged_kv_commit(kv, i32(table), i32([1]), i32([10]), i32([[0, 25, 30]]), i32([3]), 3)      # the third page lies past the cache
    assert dev.gemm_status() == 31 and torch.equal(kv.k, before)


# ---- refusals of the wrappers ---------------------------------------------------------------------------------------

def test_wrappers_refuse_wrong_tensors(dev):
    import torch
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")
    f, h = torch.float32, torch.float16
    kv = dev.PagedKV(2, 4, 2, 64)
    ok = dict(q=z(3, 256, dt=f), q_row_stride=256, kv=kv, layer=1, block_table=z(1, 4), tree_slot=z(1), tree_ctx=z(1), tree_row0=z(2), tree_mask=z(3, 1),
              out=z(3, 256, dt=f), q_heads=4, mbps=4, max_nodes=3, scale=1.0, scratch=dev.paged_attn_tree_scratch(3, 4, 2, 64))
    dev.paged_attn_tree(**ok)
    for bad in [dict(q=z(3, 256, dt=h)), dict(out=z(3, 256, dt=h)), dict(q=z(2, 256, dt=f)), dict(q=z(3, 256, dt=f).cpu()), dict(layer=2), dict(layer=-1), dict(tree_ctx=z(2)),
                dict(tree_row0=z(3)), dict(tree_slot=z(1, dt=torch.int64)), dict(tree_mask=z(2, 1)), dict(tree_mask=z(3)), dict(out=z(3, 128, dt=f)), dict(out=z(256, 3, dt=f).t()),
                dict(mbps=3), dict(mbps=0), dict(block_table=z(1, 4, dt=torch.int64)), dict(scratch=z(64)), dict(kv=dev.PagedKVInt8(2, 4, 2, 64))]:
        with pytest.raises(ValueError):
            dev.paged_attn_tree(**{**ok, **bad})
    from wukong_b200._lib import WukongB200Error
    for bad in [dict(max_nodes=0), dict(max_nodes=33), dict(q_heads=3), dict(scratch=z(64, dt=torch.uint8))]:
        with pytest.raises(WukongB200Error):
            dev.paged_attn_tree(**{**ok, **bad})
    for bad in [(z(2, 8, dt=h), None), (z(2, 8, dt=f), z(3, dt=f)), (z(2, 8, dt=f), z(2, dt=h)), (z(8, 2, dt=f).t(), None)]:
        with pytest.raises(ValueError):
            dev.token_probs(*bad)
    with pytest.raises(ValueError):
        dev.token_probs(z(2, 8, dt=f), out=z(2, 9, dt=f))
    ok = dict(probs=z(4, 8, dt=f), draft=z(4, 8, dt=f), token=z(4), parent=z(4), tree_row0=z(2), u_node=z(4, dt=f), u_final=z(1, dt=f), max_nodes=4, max_path=4)
    dev.tree_verify(**ok)
    for bad in [dict(draft=z(4, 9, dt=f)), dict(probs=z(4, 8, dt=h)), dict(token=z(5)), dict(parent=z(3)), dict(u_node=z(3, dt=f)), dict(u_final=z(2, dt=f)),
                dict(tree_row0=z(2, dt=torch.int64)), dict(out=(z(1, 3), z(1), z(1, 4)))]:
        with pytest.raises(ValueError):
            dev.tree_verify(**{**ok, **bad})
    ok = dict(kv=kv, block_table=z(1, 4), tree_slot=z(1), tree_ctx=z(1), path=z(1, 3), n_path=z(1), mbps=4)
    dev.paged_kv_commit(**ok)
    for bad in [dict(path=z(2, 3)), dict(path=z(3)), dict(n_path=z(2)), dict(new_ctx=z(2)), dict(kv=dev.PagedKVInt8(2, 4, 2, 64)), dict(mbps=5)]:
        with pytest.raises(ValueError):
            dev.paged_kv_commit(**{**ok, **bad})


# ---- together -------------------------------------------------------------------------------------------------------

def test_speculative_generation_equals_plain_greedy(dev):
    """A one-layer model decodes greedily with draft trees (some guesses right, some wrong) through append, tree attention,
    probabilities, verification and commit, and emits what token-by-token decoding over a dense cache in f64 emits."""
    import torch
    qh, kvh, hd, vocab, steps = 4, 2, 64, 101, 40
    d = qh * hd
    rng = np.random.default_rng(77)
    mat = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()
    emb, pos_emb, wq, wk, wv, wo = mat(vocab, d), mat(256, d), mat(d, d) / 16, mat(d, kvh * hd) / 16, mat(d, kvh * hd) / 16, mat(d, vocab)
    scale = 1.0 / math.sqrt(hd)
    prompts = [[5, 9, 77], [3], [50, 2, 2, 8, 100, 61, 7]]

    def plain(prompt):
        toks, margins = list(prompt), []
        while len(toks) < len(prompt) + steps:
            x = (emb[toks] + pos_emb[:len(toks)]).double()
            q, k, v = x[-1] @ wq.double(), (x.float() @ wk).bfloat16().double(), (x.float() @ wv).bfloat16().double()
            o = []
            for h in range(qh):
                g = slice(h // 2 * hd, (h // 2 + 1) * hd)
                o.append(torch.softmax(k[:, g] @ q[h * hd:(h + 1) * hd] * scale, 0) @ v[:, g])
            logits = torch.cat(o) @ wo.double()
            top = logits.topk(2).values
            margins.append(float(top[0] - top[1]))
            toks.append(int(logits.argmax()))
        return toks, min(margins)

    refs, margins = zip(*(plain(p) for p in prompts))
    n, page, mbps, most = len(prompts), 16, 8, 8
    table = rng.permutation(n * mbps).reshape(n, mbps)
    kv = dev.PagedKV(1, n * mbps, kvh, hd, page)
    bt, slot = i32(table), i32(np.arange(n))
    scratch = dev.paged_attn_tree_scratch(most, qh, kvh, hd)
    done = [list(p) for p in prompts]
    ctx = np.zeros(n, np.int64)
    first = True
    rounds = 0
    worst = 0.0
    while any(len(done[s]) < len(refs[s]) for s in range(n)):
        counts, token, parent, targets = [], [], [], []
        for s in range(n):
            if first:                                             # the prompt is a chain that is accepted by construction
                guess = list(prompts[s])
                par = [i - 1 for i in range(len(guess))]
            else:
                nxt = refs[s][len(done[s]):len(done[s]) + 3]
                guess, par = [done[s][-1]], [-1]
                tip = 0
                for g in nxt:                                     # at each level a wrong sibling first, then mostly the right one
                    guess += [(g + 1) % vocab, g if rng.random() < 0.7 else (g + 2) % vocab]
                    par += [tip, tip]
                    tip = len(guess) - 1
            counts.append(len(guess)); token += guess; parent += par
        row0 = np.concatenate([[0], np.cumsum(counts)])
        mask, depth = dev.tree_layout(np.array(parent), row0)
        base = np.repeat(ctx, counts)
        node = np.concatenate([np.arange(c) for c in counts])
        x = emb[torch.tensor(token).cuda()] + pos_emb[torch.from_numpy(base + depth).cuda()]
        qkv = torch.cat([x @ wq, x @ wk, x @ wv], 1)
        rows = len(token)
        dev.paged_kv_append(kv, 0, qkv[:, d:], qkv[:, d + kvh * hd:], qkv.stride(0), bt, i32(np.repeat(np.arange(n), counts)), i32(base + node), rows, mbps)
        att = torch.empty((rows, d), device="cuda")
        dev.paged_attn_tree(qkv, qkv.stride(0), kv, 0, bt, slot, i32(ctx), i32(row0), i32(mask), att, qh, mbps, most, scale, scratch)
        probs = dev.token_probs(att @ wo, torch.zeros(rows, device="cuda"))
        if first:
            ctx = ctx + np.array([len(p) - 1 for p in prompts])
            path = np.zeros((n, 1)); n_path = np.ones(n)
            for s in range(n):
                done[s].append(int(probs[int(row0[s + 1]) - 1].argmax()))
            ctx = ctx + 1
            first = False
            continue
        u = torch.rand(rows + n, device="cuda")
        path, n_path, tokens = dev.tree_verify(probs, None, i32(token), i32(parent), i32(row0), u[:rows].clone(), u[rows:].clone(), most, most)
        new_ctx = torch.empty(n, dtype=torch.int32, device="cuda")
        dev.paged_kv_commit(kv, bt, slot, i32(ctx), path, n_path, mbps, new_ctx=new_ctx)
        emitted, ctx, rounds = tokens.cpu().numpy(), new_ctx.cpu().numpy().astype(np.int64), rounds + 1
        for s in range(n):
            done[s] += [int(t) for t in emitted[s] if t >= 0]
            assert len(done[s]) - 1 == ctx[s]
        if max(int(c) for c in ctx) + most > mbps * page:
            break
    assert min(margins) > 1e-3, margins                            # the tokens of the comparison are not near ties
    assert rounds < steps, "some drafts were accepted"
    for s in range(n):
        upto = min(len(done[s]), len(refs[s]))
        assert done[s][:upto] == refs[s][:upto]
    assert dev.gemm_status() == 0
