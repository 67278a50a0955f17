"""Cases of the speculative-decoding operators: attention of draft trees over the paged cache, vocabulary probabilities,
verification of drafted tokens, and the commit of the accepted tokens' K / V.

A draft tree hangs off a sequence of `ctx` committed tokens: node 0 is the last token that the target model emitted, every
other node a drafted token whose parent is an earlier node.  The nodes' K / V lie at positions ctx, ctx + 1, ... of the
sequence's pages, in node order.  All trees' nodes are the rows of one flat batch; `row0` holds each tree's first row."""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE = 16


def listed():
    return [
        # one user, a short chain of guesses, GPT-2 shape: the latency of a step decides
        dict(name="tree_one", op="tree", n=1, nodes=5, ctx_lo=257, ctx_hi=257, qh=12, kvh=12, hd=64, q="f32", out="bf16", lens=1),
        # a GPT-2-shape engine's batch, trees of any size up to 16, contexts up to the model's 1024 positions
        dict(name="tree_gpt2", op="tree", n=32, nodes=16, ctx_lo=16, ctx_hi=1000, qh=12, kvh=12, hd=64, q="f32", out="bf16", lens=2),
        # one sequence with a long cache and a wide tree: the key axis has to be split over the card
        dict(name="tree_long", op="tree", n=1, nodes=64, ctx_lo=32749, ctx_hi=32749, qh=32, kvh=8, hd=128, q="bf16", out="bf16", lens=3),
        # a Llama-shape serving batch, the context draw of the decode micro-benchmark
        dict(name="tree_serving", op="tree", n=64, nodes=16, ctx_lo=128, ctx_hi=4096, qh=32, kvh=8, hd=128, q="f32", out="bf16", lens=4),
        # wide trees, eight query heads a KV head, f32 results
        dict(name="tree_wide_f32", op="tree", n=16, nodes=61, ctx_lo=500, ctx_hi=8000, qh=32, kvh=4, hd=128, q="f32", out="f32", lens=5),
        # the probabilities of one user's chain and of a whole batch of trees
        dict(name="probs_few", op="probs", rows=5, vocab=50257, dtype="f32"),
        dict(name="probs_batch", op="probs", rows=1024, vocab=32000, dtype="f32"),
        # one user's chain against the draft model's distributions
        dict(name="verify_chain", op="verify", n=1, nodes=5, vocab=50257, draft=True, lens=6),
        # a batch of trees drawn from the draft model
        dict(name="verify_trees", op="verify", n=64, nodes=16, vocab=32000, draft=True, lens=7),
        # trees of top candidates, without draft distributions
        dict(name="verify_topk", op="verify", n=32, nodes=24, vocab=50257, draft=False, lens=8),
        # the accepted tokens of one GPT-2-shape sequence, and of a Llama-shape batch
        dict(name="commit_one", op="commit", n=1, nodes=5, layers=12, kvh=12, hd=64, lens=9),
        dict(name="commit_batch", op="commit", n=64, nodes=16, layers=32, kvh=8, hd=128, lens=10),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "probs", "verify", "commit"])
    lens = rng.randrange(1 << 20)
    if op == "tree":
        hd = rng.choice([64, 128])
        kvh = rng.choice([1, 2, 4, 8, 12] if hd == 64 else [1, 2, 4, 8])
        qh = kvh * rng.choice([1, 2, 4, 8] if kvh <= 4 else [1, 2, 4] if kvh == 8 else [1, 2])
        n = _spread(rng, 1, 64)
        hi = _spread(rng, 20, min(32000, 150000 // n))
        return dict(op=op, n=n, nodes=_spread(rng, 1, 64 if n <= 16 else 16), ctx_lo=rng.randint(1, hi), ctx_hi=hi, qh=qh, kvh=kvh, hd=hd,
                    q=rng.choice(["f32", "bf16"]), out=rng.choice(["bf16", "bf16", "f32"]), lens=lens)
    if op == "probs":
        vocab = _spread(rng, 1000, 130000)
        return dict(op=op, rows=_spread(rng, 1, min(1024, 32000000 // vocab)), vocab=vocab, dtype=rng.choice(["f32", "bf16"]))
    if op == "verify":
        vocab, n = _spread(rng, 1000, 130000), _spread(rng, 1, 64)
        nodes = min(_spread(rng, 1, 32), max(1, 32000000 // (vocab * n)))
        return dict(op=op, n=n, nodes=nodes, vocab=vocab, draft=rng.random() < 0.6, lens=lens)
    kvh, hd = rng.choice([(12, 64), (8, 128), (2, 128), (5, 64)])
    return dict(op=op, n=_spread(rng, 1, 64), nodes=rng.randint(2, 32), layers=rng.randint(1, 32), kvh=kvh, hd=hd, lens=lens)


# ---- inputs ---------------------------------------------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _lens(case):
    """Nodes and committed tokens of each tree: of the case alone, so that its work is known without the inputs."""
    r = np.random.default_rng(case["lens"])
    nodes = r.integers(1, case["nodes"] + 1, case["n"])
    nodes[r.integers(case["n"])] = case["nodes"]
    ctx = r.integers(case.get("ctx_lo", 1), case.get("ctx_hi", 40) + 1, case["n"])
    return nodes.astype(np.int64), ctx.astype(np.int64)


def _trees(nodes, r):
    """Random trees: `row0` [n + 1], and for each row its node's parent (-1 for a root)."""
    row0 = np.concatenate([[0], np.cumsum(nodes)])
    parent = np.full(row0[-1], -1, np.int64)
    for t, k in enumerate(nodes):
        for i in range(1, k):
            parent[row0[t] + i] = r.integers(max(0, i - 4), i)
    return row0, parent


def _masks(row0, parent, words):
    """Bit j of a row's words: node j of its tree is the row's node itself or one of its ancestors."""
    m = np.zeros((row0[-1], words), np.uint32)
    for t in range(len(row0) - 1):
        for i in range(row0[t + 1] - row0[t]):
            r = row0[t] + i
            if parent[r] >= 0:
                m[r] = m[row0[t] + parent[r]]
            m[r, i // 32] |= np.uint32(1 << (i % 32))
    return m.view(np.int32)


def _pages(lengths, r):
    """A table of randomly ordered pages that holds `lengths` tokens a sequence."""
    need = -(-lengths // PAGE)
    pool = r.permutation(int(need.sum()) + 3)
    table = np.zeros((len(lengths), int(need.max())), np.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = pool[at:at + k]
        at += k
    return table, len(pool)


def _cache(layers, pages, case, g):
    shape = (layers, pages, case["kvh"], PAGE, case["hd"])
    k, v = (torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    return SimpleNamespace(k=k, v=v, layers=layers, num_pages=pages, kv_heads=case["kvh"], head_dim=case["hd"], page_tokens=PAGE)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = np.random.default_rng(seed)
    if case["op"] == "tree":
        nodes, ctx = _lens(case)
        row0, parent = _trees(nodes, r)
        rows, words = int(row0[-1]), -(-case["nodes"] // 32)
        table, pages = _pages(ctx + nodes, r)
        q = torch.randn((rows, case["qh"] * case["hd"]), generator=g, device="cuda") * 1.5
        return dict(case=case, q=q.to(_TYPES[case["q"]]), kv=_cache(1, pages, case, g), table=_i32(table), slot=_i32(np.arange(case["n"])),
                    ctx=_i32(ctx), row0=_i32(row0), mask=_i32(_masks(row0, parent, words)), scale=1.0 / math.sqrt(case["hd"]),
                    out=torch.zeros((rows, case["qh"] * case["hd"]), dtype=_TYPES[case["out"]], device="cuda"))
    if case["op"] == "probs":
        x = torch.randn((case["rows"], case["vocab"]), generator=g, device="cuda") * 2.5
        t = torch.rand(case["rows"], generator=g, device="cuda") + 0.5
        t[:: 7] = 0.0       # some requests of a batch decode greedily
        t[0] = 0.8
        return dict(case=case, logits=x.to(_TYPES[case["dtype"]]), temperature=t)
    if case["op"] == "verify":
        nodes, _ = _lens(case)
        row0, parent = _trees(nodes, r)
        rows = int(row0[-1])
        logits = torch.randn((rows, case["vocab"]), generator=g, device="cuda") * 2.5
        guess = logits + torch.randn((rows, case["vocab"]), generator=g, device="cuda")
        probs, draft = torch.softmax(logits, 1), torch.softmax(guess, 1)
        if case["draft"]:    # children are draws from the draft model's distribution at their parent
            picks = torch.multinomial(draft, 4, replacement=True, generator=g).cpu().numpy()
        else:                # children are the draft model's best candidates
            picks = guess.topk(4, 1).indices.cpu().numpy()
        token, used = r.integers(0, case["vocab"], rows), np.zeros(rows, np.int64)
        for t in range(case["n"]):
            for i in range(row0[t] + 1, row0[t + 1]):
                p = row0[t] + parent[i]
                token[i] = picks[p, used[p]]
                used[p] += 1
        u = torch.rand((rows + case["n"],), generator=g, device="cuda")
        return dict(case=case, probs=probs, draft=draft if case["draft"] else None, token=_i32(token), parent=_i32(parent), row0=_i32(row0),
                    u_node=u[:rows].clone(), u_final=u[rows:].clone(), nodes=case["nodes"])
    nodes, ctx = _lens(case)
    path, n_path = np.full((case["n"], case["nodes"]), -1, np.int64), np.ones(case["n"], np.int64)
    for t, k in enumerate(nodes):      # the first guess of some levels, later nodes for the rest
        n = int(r.integers(1, 1 + min(8, (k + 1) // 2)))
        lead = int(r.integers(1, n + 1))
        path[t, :lead] = np.arange(lead)
        path[t, lead:n] = np.sort(r.permutation(np.arange(n, k))[:n - lead])
        n_path[t] = n
    table, pages = _pages(ctx + nodes, r)
    return dict(case=case, kv=_cache(case["layers"], pages, case, g), table=_i32(table), slot=_i32(np.arange(case["n"])), ctx=_i32(ctx),
                path=_i32(path), n_path=_i32(n_path), new_ctx=torch.zeros(case["n"], dtype=torch.int32, device="cuda"))


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    return {"tree": _run_tree, "probs": _run_probs, "verify": _run_verify, "commit": _run_commit}[state["case"]["op"]](state)


def _run_tree(s):
    case, kv = s["case"], s["kv"]
    if own:
        from wukong_b200 import device as dev
        if "scratch" not in s:      # a program keeps one for all its layers and steps
            s["scratch"] = dev.paged_attn_tree_scratch(case["nodes"], case["qh"], kv.kv_heads, kv.head_dim)
        return dev.paged_attn_tree(s["q"], s["q"].stride(0), kv, 0, s["table"], s["slot"], s["ctx"], s["row0"], s["mask"], s["out"], case["qh"],
                                   s["table"].shape[1], case["nodes"], s["scale"], s["scratch"])
    n, qh, kvh, hd, most = case["n"], case["qh"], kv.kv_heads, kv.head_dim, case["nodes"]
    pages = s["table"][s["slot"].long()].long()
    k, v = (x[0][pages].permute(0, 2, 1, 3, 4).reshape(n, kvh, -1, hd).float() for x in (kv.k, kv.v))
    rows = s["q"].shape[0]
    row0, at = s["row0"].long(), torch.arange(rows, device="cuda")
    tree = torch.bucketize(at, row0[1:], right=True)
    node = at - row0[tree]
    q = torch.zeros((n, most, qh, hd), device="cuda")
    q[tree, node] = s["q"].float().view(rows, qh, hd)
    q = q.view(n, most, kvh, qh // kvh, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, hd)
    scores = (q @ k.transpose(2, 3) * s["scale"]).view(n, kvh, qh // kvh, most, -1)
    j = torch.arange(scores.shape[-1], device="cuda")[None, :] - s["ctx"].long()[:, None]              # node at each position
    jc = j.clamp(0, most - 1)[tree]
    bit = (torch.gather(s["mask"], 1, jc // 32) >> (jc % 32)) & 1
    count = (row0[1:] - row0[:-1])[tree, None]
    seen = torch.zeros((n, most, scores.shape[-1]), dtype=torch.bool, device="cuda")
    seen[tree, node] = (j[tree] < 0) | ((j[tree] < count) & (bit == 1))
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, kvh, -1, p.shape[-1]) @ v).view(n, kvh, qh // kvh, most, hd) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, qh * hd)[tree, node].to(s["out"].dtype)


def _run_probs(s):
    if own:
        from wukong_b200 import device as dev
        return dev.token_probs(s["logits"], s["temperature"])
    x, t = s["logits"].float(), s["temperature"][:, None]
    e = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(t > 0, t, 1.0))
    cold = torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
    return torch.where(t > 0, e / e.sum(1, keepdim=True), cold)


def _run_verify(s):
    if own:
        from wukong_b200 import device as dev
        return dev.tree_verify(s["probs"], s["draft"], s["token"], s["parent"], s["row0"], s["u_node"], s["u_final"], s["nodes"], s["nodes"])
    row0, most = s["row0"].long(), s["nodes"]
    first, count = row0[:-1], row0[1:] - row0[:-1]
    n, t = first.numel(), torch.arange(first.numel(), device="cuda")
    cur, z = torch.zeros(n, dtype=torch.long, device="cuda"), torch.ones(n, dtype=torch.float64, device="cuda")
    left = s["probs"][first].double()
    path = torch.full((n, most), -1, dtype=torch.int32, device="cuda")
    path[:, 0], length = 0, torch.ones(n, dtype=torch.long, device="cuda")
    for i in range(1, most):            # nodes in order: a node's children come after it
        row = (first + i).clamp(max=s["token"].numel() - 1)
        tried = (i < count) & (s["parent"][row].long() == cur)
        x = s["token"][row].long()
        q = torch.zeros_like(left).scatter_(1, x[:, None], 1.0) if s["draft"] is None else s["draft"][first + cur].double()
        r = left[t, x]
        accept = tried & (s["u_node"][row].double() * q[t, x] * z < r)
        lower = left.scatter(1, x[:, None], 0.0) if s["draft"] is None else (left - z[:, None] * q).clamp(min=0)
        new_z = z - r if s["draft"] is None else lower.sum(1)
        refused = tried & ~accept
        left = torch.where(refused[:, None], lower, left)
        z = torch.where(refused, new_z, z)
        cur = torch.where(accept, i, cur)
        left = torch.where(accept[:, None], s["probs"][first + cur].double(), left)
        z = torch.where(accept, 1.0, z)
        path[t[accept], length[accept]] = i
        length = length + accept
    mass = left.cumsum(1)
    index = torch.arange(left.shape[1], device="cuda")
    at = (mass <= s["u_final"].double()[:, None] * mass[:, -1:]).sum(1)
    last = torch.where(left > 0, index, -1).amax(1)
    final = torch.where(mass[:, -1] > 0, torch.minimum(at, last), -1)
    tokens = torch.where(path > 0, s["token"][(first[:, None] + path.clamp(min=0))], -1).roll(-1, 1)
    tokens[:, -1] = -1
    tokens[t, length - 1] = final.int()
    return path, length.int(), tokens


def _run_commit(s):
    kv = s["kv"]
    if own:
        from wukong_b200 import device as dev
        dev.paged_kv_commit(kv, s["table"], s["slot"], s["ctx"], s["path"], s["n_path"], s["table"].shape[1], new_ctx=s["new_ctx"])
        return kv.k, kv.v, s["new_ctx"]
    order = torch.arange(s["path"].shape[1], device="cuda")
    t, i = torch.where((order >= 1) & (order < s["n_path"][:, None]))
    src, dst = s["ctx"][t] + s["path"][t, i], s["ctx"][t] + i
    table = s["table"][s["slot"].long()].long()
    from_page, to_page = table[t, (src // PAGE).long()], table[t, (dst // PAGE).long()]
    for x in (kv.k, kv.v):
        x[:, to_page, :, (dst % PAGE).long()] = x[:, from_page, :, (src % PAGE).long()]
    s["new_ctx"].copy_(s["ctx"] + s["n_path"])
    return kv.k, kv.v, s["new_ctx"]


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "tree":
        nodes, ctx = _lens(case)
        size = {"f32": 4, "bf16": 2}
        rows, keys = int(nodes.sum()), int((ctx + nodes).sum())
        return {"bytes": keys * case["kvh"] * case["hd"] * 4 + rows * case["qh"] * case["hd"] * (size[case["q"]] + size[case["out"]]),
                "flops": 4 * case["qh"] * case["hd"] * int((nodes * (ctx + nodes)).sum())}
    if case["op"] == "probs":
        return {"bytes": case["rows"] * case["vocab"] * (4 + {"f32": 4, "bf16": 2}[case["dtype"]]), "flops": 4 * case["rows"] * case["vocab"]}
    if case["op"] == "verify":      # the row at which each walk ends, and the draft's there
        rows = int(_lens(case)[0].sum())
        return {"bytes": case["n"] * case["vocab"] * 4 * (2 if case["draft"] else 1) + rows * 20, "flops": 3 * case["n"] * case["vocab"]}
    nodes, _ = _lens(case)          # half of the tokens that a tree of this size can yield
    moved = sum(min(8, (int(k) + 1) // 2) for k in nodes) // 2 + 1
    return {"bytes": moved * case["layers"] * case["kvh"] * case["hd"] * 8, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "commit":
        return None
    s = prepare(case, seed)
    return {"tree": _exact_tree, "probs": _exact_probs, "verify": _exact_verify}[case["op"]](s)


def _exact_tree(s):
    case, kv = s["case"], s["kv"]
    group, hd = case["qh"] // case["kvh"], case["hd"]
    row0, ctx, table = (s[k].cpu().numpy() for k in ("row0", "ctx", "table"))
    mask = s["mask"].cpu().numpy().view(np.uint32)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for t in range(case["n"]):
        count, c = int(row0[t + 1] - row0[t]), int(ctx[t])
        pos = np.arange(c + count)
        page, off = (torch.from_numpy(a).cuda() for a in (table[t, pos // PAGE].astype(np.int64), pos % PAGE))
        seen = np.ones((count, c + count), bool)
        for j in range(count):
            seen[:, c + j] = (mask[row0[t]:row0[t + 1], j // 32] >> np.uint32(j % 32)) & 1
        hidden = ~torch.from_numpy(seen).cuda()
        for h in range(case["kvh"]):
            key, val = kv.k[0, page, h, off].double(), kv.v[0, page, h, off].double()
            for f in range(h * group, (h + 1) * group):
                q = s["q"][int(row0[t]):int(row0[t + 1]), f * hd:(f + 1) * hd].double()
                a = (q @ key.T) * s["scale"]
                a[hidden] = -math.inf
                w = torch.exp(a - a.max(1, keepdim=True).values)
                out[int(row0[t]):int(row0[t + 1]), f * hd:(f + 1) * hd] = (w / w.sum(1, keepdim=True)) @ val
    return out


def _exact_probs(s):
    out = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    for r, t in enumerate(s["temperature"].double().tolist()):
        x = s["logits"][r].double()
        if t > 0:
            e = torch.exp(x / t - x.max() / t)
            out[r] = e / e.sum()
        else:
            out[r] = 0.0
            out[r, int(torch.nonzero(x == x.max())[0])] = 1.0
    return out


def _exact_verify(s):
    probs, row0 = s["probs"].cpu().numpy(), s["row0"].cpu().numpy()
    draft = None if s["draft"] is None else s["draft"].cpu().numpy()
    token, parent = s["token"].cpu().numpy(), s["parent"].cpu().numpy()
    u_node, u_final = s["u_node"].cpu().numpy().astype(np.float64), s["u_final"].cpu().numpy().astype(np.float64)
    n, most = len(row0) - 1, s["nodes"]
    path, tokens = np.full((n, most), -1, np.int32), np.full((n, most), -1, np.int32)
    length = np.zeros(n, np.int32)
    for t in range(n):
        a, b = int(row0[t]), int(row0[t + 1])
        walk, cur = [0], 0
        while True:
            left, z, nxt = probs[a + cur].astype(np.float64), 1.0, None
            for c in [i for i in range(1, b - a) if parent[a + i] == cur]:
                x = token[a + c]
                q = 1.0 if draft is None else float(draft[a + cur, x])
                if u_node[a + c] * q * z < left[x]:
                    nxt = c
                    break
                if draft is None:
                    z -= left[x]
                    left[x] = 0.0
                else:
                    left = np.maximum(left - z * draft[a + cur].astype(np.float64), 0.0)
                    z = left.sum()
            if nxt is None:
                break
            walk.append(nxt)
            cur = nxt
        mass = np.cumsum(left)
        hit = np.nonzero(mass > u_final[t] * mass[-1])[0]
        last = hit[0] if len(hit) else np.nonzero(left > 0)[0][-1]
        path[t, :len(walk)], length[t] = walk, len(walk)
        tokens[t, :len(walk)] = [token[a + i] for i in walk[1:]] + [last]
    return torch.from_numpy(path), torch.from_numpy(length), torch.from_numpy(tokens)
