"""Cases of the operators that verify a tree of drafted tokens in one decode step.

A speculative step scores the drafted tokens of every request with one forward pass: attention of
the tree's nodes over the paged cache (``ops.tree_attention``), the MoE layer on those few tokens
(``ops.moe_few_tokens``), and the acceptance of one path of the tree with the move of that path's
cache rows (``ops.tree_commit``).

``run`` computes the plain form with elementary torch operations while ``own`` is false, and calls
the package's operators while it is true.
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One request drafts 8 nodes behind a short prompt: what a step costs when nothing hides latency.
        dict(name="attn_one_request", op="attention", batch=1, nodes_min=8, nodes_max=8, ctx_min=500, ctx_max=500,
             q_heads=32, kv_heads=4, head_dim=128, block=256, chain=False),
        # A busy server: 32 requests of about 1,100 tokens, 16 nodes each.
        dict(name="attn_serving", op="attention", batch=32, nodes_min=16, nodes_max=16, ctx_min=1000, ctx_max=1300,
             q_heads=32, kv_heads=4, head_dim=128, block=256, chain=False),
        # Drafted chains of 4 tokens for 64 requests: the cache is all there is to read.
        dict(name="attn_chains", op="attention", batch=64, nodes_min=4, nodes_max=4, ctx_min=4000, ctx_max=4200,
             q_heads=32, kv_heads=4, head_dim=128, block=256, chain=True),
        # Long context with large trees on 16 query heads per KV head: bound by the products.
        dict(name="attn_long_context", op="attention", batch=4, nodes_min=64, nodes_max=64, ctx_min=32000,
             ctx_max=32768, q_heads=64, kv_heads=4, head_dim=128, block=256, chain=False),
        # Ragged batch on small blocks and heads of 64: empty contexts, single nodes, pages that end inside a tile.
        dict(name="attn_ragged", op="attention", batch=13, nodes_min=1, nodes_max=23, ctx_min=0, ctx_max=2777,
             q_heads=4, kv_heads=2, head_dim=64, block=16, chain=False),
        # The acceptance of one request's step over the 48 layers of the cache.
        dict(name="commit_one_request", op="commit", batch=1, nodes_min=8, nodes_max=8, accept_max=4, layers=48,
             kv_heads=4, head_dim=128, block=64, int8=False),
        # The same for a batch, paths of one to eight nodes.
        dict(name="commit_serving", op="commit", batch=32, nodes_min=16, nodes_max=32, accept_max=8, layers=48,
             kv_heads=4, head_dim=128, block=64, int8=False),
        # An int8 cache: payload and scales move together.
        dict(name="commit_int8", op="commit", batch=24, nodes_min=3, nodes_max=40, accept_max=6, layers=48, kv_heads=4,
             head_dim=128, block=64, int8=True),
        # One token through a MoE layer of 128 experts, top-8: eight experts' weights and little else.
        dict(name="moe_one_token", op="moe", tokens=1, hidden=2048, inter=768, experts=128, topk=8, fp8=True),
        # Two requests' trees of eight nodes.
        dict(name="moe_16_tokens", op="moe", tokens=16, hidden=2048, inter=768, experts=128, topk=8, fp8=True),
        # Four trees of 16: nearly every expert is read.
        dict(name="moe_64_tokens", op="moe", tokens=64, hidden=2048, inter=768, experts=128, topk=8, fp8=True),
        # bf16 weights in their natural layout, a small layer, an odd number of tokens.
        dict(name="moe_bf16_small", op="moe", tokens=5, hidden=256, inter=128, experts=8, topk=2, fp8=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "commit", "moe"))
    if op == "attention":
        q_heads, kv_heads, head_dim = rng.choice(((32, 4, 128), (64, 4, 128), (16, 2, 128), (8, 8, 128), (4, 2, 64),
                                                  (12, 4, 128), (16, 1, 64)))
        n = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, 32768)
        # no more cache rows than the listed cases read, no more products than the largest
        batch = max(1, min(_log_int(rng, 1, 64), 260000 // (ctx + n),
                           int(2.5e11 / (4.0 * (ctx + n) * n * q_heads * head_dim))))
        lo = rng.choice((ctx, max(0, ctx - ctx // 3), 0))
        return dict(op=op, batch=batch, nodes_min=rng.choice((n, 1)), nodes_max=n, ctx_min=lo, ctx_max=ctx,
                    q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, block=rng.choice((16, 32, 64, 128, 256)),
                    chain=rng.random() < 0.25)
    if op == "commit":
        n = _log_int(rng, 1, 64)
        return dict(op=op, batch=_log_int(rng, 1, 32), nodes_min=rng.choice((n, 1)), nodes_max=n,
                    accept_max=rng.randint(1, min(8, n)), layers=rng.choice((2, 24, 48)),
                    kv_heads=rng.choice((1, 2, 4)), head_dim=rng.choice((64, 128)), block=rng.choice((16, 64)),
                    int8=rng.random() < 0.4)
    fp8 = rng.random() < 0.7
    return dict(op=op, tokens=_log_int(rng, 1, 64), hidden=128 * _log_int(rng, 2, 16), inter=128 * _log_int(rng, 1, 6),
                experts=_log_int(rng, 8, 128 if fp8 else 64), topk=rng.choice((1, 2, 4, 6, 8, 8, 8)), fp8=fp8)


# -------------------------------------------------------------- their sizes
def _spread(lo, hi, n, step):
    """n whole numbers over [lo, hi], both ends among them, in an order that is not sorted."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _coprime(n, start):
    s = start
    while math.gcd(s, n) != 1:
        s += 1
    return s


def _lens(case):
    """(nodes, committed context) of every request, from the case alone."""
    b = case["batch"]
    nodes = _spread(case["nodes_min"], case["nodes_max"], b, _coprime(b, 5))
    if case["op"] == "commit":
        ctx = [(37 * i + 11) % (3 * case["block"]) for i in range(b)]
    else:
        ctx = _spread(case["ctx_min"], case["ctx_max"], b, _coprime(b, 3))
    return nodes, ctx


def _paths(case):
    """The accepted path of every request (node indices), from the case alone."""
    nodes, _ = _lens(case)
    out = []
    for i, n in enumerate(nodes):
        m = min(n, 1 + (3 * i + case["accept_max"] - 1) % case["accept_max"])
        step = (n - 1) // (m - 1) if m > 1 else 1
        out.append([j * step for j in range(m)])
    return out


def work(case):
    if case["op"] == "attention":
        nodes, ctx = _lens(case)
        d, h, q = case["head_dim"], case["kv_heads"], case["q_heads"]
        keys = sum(n + c for n, c in zip(nodes, ctx))
        pairs = sum(n * (n + c) for n, c in zip(nodes, ctx))
        return {"bytes": keys * 2 * h * d * 2 + 2 * sum(nodes) * q * d * 2 + 4 * sum(nodes),
                "flops": 4.0 * pairs * q * d}
    if case["op"] == "commit":
        moved = sum(sum(1 for j, p in enumerate(path) if p != j) for path in _paths(case))
        rows = moved * case["layers"] * 2 * case["kv_heads"]
        per = case["head_dim"] * (1 if case["int8"] else 2) + (4 if case["int8"] else 0)
        nodes, _ = _lens(case)
        return {"bytes": 2 * rows * per + 20 * sum(nodes) + 12 * case["batch"], "flops": 0}
    t, h, i, e, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "topk"))
    touched = e * (1.0 - (1.0 - k / e) ** t)   # experts that at least one token is expected to pick
    wbytes = 1 if case["fp8"] else 2
    return {"bytes": touched * 3 * h * i * wbytes + e * h * 2 + 2 * t * h * 2,
            "flops": 2.0 * t * k * 3 * h * i + 2.0 * t * h * e}


# ------------------------------------------------------------------ the inputs
def _trees(case, seed, paths=None):
    """Parents of every node: a random tree per request (node 0 its root); with `paths` each of
    those paths is a chain of the tree."""
    nodes, _ = _lens(case)
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    out = []
    for b, n in enumerate(nodes):
        r = torch.rand(n, generator=g).tolist()
        if case.get("chain"):
            par = list(range(-1, n - 1))
        else:
            par = [-1] + [max(0, i - 1 - int(r[i] * min(i, 6))) for i in range(1, n)]
        if paths is not None:
            for a, c in zip(paths[b], paths[b][1:]):
                par[c] = a
        out.append(par)
    return out


def _tables(case, nodes, ctx, seed):
    """Block tables of a shuffled pool: (tables [batch, max_blocks], blocks in the pool)."""
    bs = case["block"]
    need = [max(1, -(-(n + c) // bs)) for n, c in zip(nodes, ctx)]
    total = sum(need)
    g = torch.Generator().manual_seed(seed * 31 + 7)
    ids = torch.randperm(total, generator=g).to(torch.int32)
    tab = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        tab[b, :k] = ids[at:at + k]
        at += k
    return tab.to(DEV), total + 1   # the last block is the pool's scratch block


def _ragged(nodes, ctx):
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    i32 = dict(dtype=torch.int32, device=DEV)
    return torch.tensor(cu, **i32), torch.tensor([n + c for n, c in zip(nodes, ctx)], **i32)


def _prepare_attention(case, seed):
    nodes, ctx = _lens(case)
    tab, blocks = _tables(case, nodes, ctx, seed)
    cu, lens = _ragged(nodes, ctx)
    g = torch.Generator(device=DEV).manual_seed(seed)
    h, d, q = case["kv_heads"], case["head_dim"], case["q_heads"]
    pool = torch.randn(blocks, 1, 2, h, case["block"], d, generator=g, device=DEV, dtype=torch.bfloat16)
    qs = (torch.randn(sum(nodes), q, d, generator=g, device=DEV) * 2.0).to(torch.bfloat16)
    par = torch.tensor([p for t in _trees(case, seed) for p in t], dtype=torch.int32, device=DEV)
    return dict(case=case, q=qs, k=pool[:, 0, 0], v=pool[:, 0, 1], tables=tab, cu=cu, lens=lens, parents=par,
                max_nodes=max(nodes), max_len=max(n + c for n, c in zip(nodes, ctx)), scale=d ** -0.5)


def _prepare_commit(case, seed):
    nodes, ctx = _lens(case)
    paths = _paths(case)
    tab, blocks = _tables(case, nodes, ctx, seed)
    cu, lens = _ragged(nodes, ctx)
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (blocks, case["layers"], 2, case["kv_heads"], case["block"])
    scales = None
    if case["int8"]:
        data = torch.randint(-127, 128, (*shape, case["head_dim"]), generator=g, device=DEV, dtype=torch.int8)
        scales = torch.rand(*shape, generator=g, device=DEV) * 0.05 + 0.001
    else:
        data = torch.randn(*shape, case["head_dim"], generator=g, device=DEV, dtype=torch.bfloat16)
    trees = _trees(case, seed, paths)
    gc = torch.Generator().manual_seed(seed * 17 + 3)
    vocab = 151936
    draft, target = [], []
    for n, path in zip(nodes, paths):
        base, step = (int(v) for v in torch.randint(1, vocab // 256, (2,), generator=gc))
        ids = [(base + i * step) % (vocab - 1) for i in range(n)]     # distinct within a tree
        t = torch.randint(0, vocab - 1, (n,), generator=gc).tolist()
        for a, c in zip(path, path[1:]):
            t[a] = ids[c]                                             # the model agrees with the path ...
        t[path[-1]] = vocab - 1                                       # ... and then picks a token nobody drafted
        draft += ids
        target += t
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(case=case, data=data, scales=scales, tables=tab, cu=cu, lens=lens, max_nodes=max(nodes),
                parents=torch.tensor([p for t in trees for p in t], **i32), draft=torch.tensor(draft, **i32),
                target=torch.tensor(target, **i32))


def _tile(w):
    """[.., N, K] e4m3 -> the same bytes tile-major, [N / 128, K / 64, 128, 64] with the four 16-byte
    chunks of a row at u ^ ((row >> 1) & 3): how the engine lays its weights out once after loading."""
    e, n, k = w.shape
    b = w.view(torch.uint8).view(e, n // 128, 128, k // 64, 4, 16).permute(0, 1, 3, 2, 4, 5)
    row = torch.arange(128, device=w.device)
    src = torch.arange(4, device=w.device)[None] ^ ((row >> 1) & 3)[:, None]
    src = src.view(1, 1, 1, 128, 4, 1).expand(*b.shape)
    return torch.gather(b, 4, src).contiguous().view(e, n, k).view(torch.float8_e4m3fn)


def _prepare_moe(case, seed):
    t, h, i, e = (case[n] for n in ("tokens", "hidden", "inter", "experts"))
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(t, h, generator=g, device=DEV).to(torch.bfloat16)           # normalised activations
    rows = -(-e // 128) * 128                                                   # the router is padded to 128 rows
    router = torch.zeros(rows, h, device=DEV, dtype=torch.bfloat16)
    router[:e] = (torch.randn(e, h, generator=g, device=DEV) * (2.0 / math.sqrt(h))).to(torch.bfloat16)
    out = dict(case=case, x=x, router=router, s13=None, s2=None)
    for name, n, k in (("w13", 2 * i, h), ("w2", h, i)):
        w = torch.empty(e, n, k, device=DEV, dtype=torch.float8_e4m3fn if case["fp8"] else torch.bfloat16)
        for j in range(0, e, 16):
            r = torch.randn(min(16, e - j), n, k, generator=g, device=DEV)
            w[j:j + 16] = (r * 100.0).clamp(-448, 448).to(w.dtype) if case["fp8"] else (r * 0.03).to(w.dtype)
        if case["fp8"]:
            # 128 x 128 block scales around 0.03 / 100
            out["s" + name[1:]] = (torch.rand(e, n // 128, k // 128, generator=g, device=DEV) + 0.5) * 3e-4
            out[name + "_tiled"] = _tile(w)
        out[name] = w
    return out


def prepare(case, seed):
    return {"attention": _prepare_attention, "commit": _prepare_commit, "moe": _prepare_moe}[case["op"]](case, seed)


# ------------------------------------------------------------- the plain forms
def _node_places(s):
    """Request and place in its tree of every node, as [tokens] index tensors."""
    cu = s["cu"].long()
    tok = torch.arange(s["parents"].shape[0], device=DEV)
    b = torch.searchsorted(cu, tok, right=True) - 1
    return b, tok - cu[b]


def _plain_attention(s):
    q, lens = s["q"], s["lens"].long()
    nb, n, length = lens.shape[0], s["max_nodes"], s["max_len"]
    nq, d = q.shape[1], q.shape[2]
    hk = s["k"].shape[1]
    b, i = _node_places(s)
    # parents -> who sees whom inside the tree (each node itself and its ancestors)
    see = torch.zeros(nb, n + 1, n + 1, device=DEV)
    see[b, i, torch.where(s["parents"] < 0, n, s["parents"].long())] = 1.0
    see = see[:, :n, :n] + torch.eye(n, device=DEV)
    for _ in range(max(1, (n - 1).bit_length())):
        see = ((see @ see) > 0).float()
    # keys and values of every request, padded to the longest
    blocks = s["tables"].long()

    def rows(pool):
        x = pool[blocks].permute(0, 2, 1, 3, 4)            # [batch, heads, blocks, block, d]
        return x.reshape(nb, hk, -1, d)[:, :, :length].float()

    k, v = rows(s["k"]), rows(s["v"])
    qp = torch.zeros(nb, n, nq, d, device=DEV)
    qp[b, i] = q.float()
    qp = qp.view(nb, n, hk, nq // hk, d).permute(0, 2, 3, 1, 4).reshape(nb, hk, -1, d)
    key = torch.arange(length, device=DEV)
    node = key[None] - (lens - (s["cu"][1:] - s["cu"][:-1]).long())[:, None]     # [batch, key]: its node, < 0 in the prefix
    ok = torch.gather(see, 2, node.clamp(0, n - 1)[:, None].expand(nb, n, length)) > 0
    ok = (ok | (node < 0)[:, None]) & (key[None] < lens[:, None])[:, None]        # [batch, node, key]
    score = ((qp @ k.transpose(2, 3)) * s["scale"]).view(nb, hk, nq // hk, n, length)
    score.masked_fill_(~ok[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp_(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    o = (p.view(nb, hk, -1, length) @ v).view(nb, hk, nq // hk, n, d)
    o = o / p.sum(dim=-1, keepdim=True).clamp_min(1e-38)
    return o.permute(0, 3, 1, 2, 4).reshape(nb, n, nq, d)[b, i].to(torch.bfloat16)


def _plain_commit(s):
    nb, n = s["lens"].shape[0], s["max_nodes"]
    b, i = _node_places(s)
    par = torch.full((nb, n), -2, dtype=torch.long, device=DEV)
    draft, target = torch.full_like(par, -1), torch.full_like(par, -1)
    par[b, i], draft[b, i], target[b, i] = s["parents"].long(), s["draft"].long(), s["target"].long()
    count = (s["cu"][1:] - s["cu"][:-1]).long()
    row, col = torch.arange(nb, device=DEV), torch.arange(n, device=DEV)[None]
    path = torch.full((nb, n), -1, dtype=torch.long, device=DEV)
    at, alive = torch.zeros(nb, dtype=torch.long, device=DEV), count > 0
    for step in range(n):
        path[:, step] = torch.where(alive, at, -1)
        fits = (par == at[:, None]) & (draft == target[row, at][:, None]) & (col > at[:, None])
        alive = alive & fits.any(dim=1)
        at = torch.where(alive, torch.where(fits, col, n).amin(dim=1), at)
    taken = (path >= 0).sum(dim=1)
    tokens = torch.where(path >= 0, torch.gather(target, 1, path.clamp(min=0)), -1)
    # the cache rows of the path move up behind the committed prefix
    bs = s["case"]["block"]
    first = s["lens"].long() - count
    rb, rj = torch.nonzero(path > col, as_tuple=True)      # the moves: more than one place to go
    src, dst = first[rb] + path[rb, rj], first[rb] + rj
    tab = s["tables"].long()
    sb, so, db, do = tab[rb, src // bs], src % bs, tab[rb, dst // bs], dst % bs
    for t in (s["data"], s["scales"]):
        if t is not None:
            t[db, :, :, :, do] = t[sb, :, :, :, so]
    out = dict(accepted=taken.int(), path=path.int(), tokens=tokens.int(), data=s["data"])
    return out if s["scales"] is None else dict(out, scales=s["scales"])


def _bf16_of(x64):
    """float64 -> the nearest bf16 value (ties to even), rounded once."""
    m, e = torch.frexp(x64)
    return torch.ldexp(torch.round(m * 256.0), e - 8)


def _plain_route(s, dtype):
    case = s["case"]
    logits = _bf16_of(s["x"].double() @ s["router"][:case["experts"]].double().t()).to(dtype)
    p = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["topk"]]   # ties: lowest id
    w = torch.gather(p, 1, ids)
    return ids, (w / w.sum(dim=1, keepdim=True)).to(torch.bfloat16).to(dtype)


def _scaled(w, s):
    w = w.float()
    if s is None:
        return w
    e, n, k = w.shape
    return (w.view(e, n // 128, 128, k // 128, 128) * s[:, :, None, :, None]).view(e, n, k)


def _plain_moe(s):
    case = s["case"]
    t, i, k = case["tokens"], case["inter"], case["topk"]
    ids, w = _plain_route(s, torch.float32)
    x = s["x"].float()
    if t * k <= case["experts"]:                           # few pairs: their experts' weights alone
        e = ids.reshape(-1)
        gu = (_scaled(s["w13"][e], None if s["s13"] is None else s["s13"][e])
              @ x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
        h = gu[:, :i] / (1.0 + torch.exp(-gu[:, :i])) * gu[:, i:]
        y = (_scaled(s["w2"][e], None if s["s2"] is None else s["s2"][e]) @ h[:, :, None])[:, :, 0]
        return (y.view(t, k, -1) * w[:, :, None]).sum(dim=1).to(torch.bfloat16)
    gate = torch.zeros(t, case["experts"], device=DEV)
    gate.scatter_(1, ids, w)
    gu = x[None] @ _scaled(s["w13"], s["s13"]).transpose(1, 2)              # [experts, tokens, 2 inter]
    h = gu[:, :, :i] / (1.0 + torch.exp(-gu[:, :, :i])) * gu[:, :, i:]
    y = h @ _scaled(s["w2"], s["s2"]).transpose(1, 2)
    return (y * gate.t()[:, :, None]).sum(dim=0).to(torch.bfloat16)


# ------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if not own:
        return {"attention": _plain_attention, "commit": _plain_commit, "moe": _plain_moe}[case["op"]](s)
    from b200moe import ops
    if case["op"] == "attention":
        from b200moe.engine.kv_cache import KVLayer
        kv = KVLayer(s["k"], s["v"], None, None, case["block"], s["k"].stride(0), 0, case["kv_heads"])
        return ops.tree_attention(s["q"], kv, s["cu"], s["lens"], s["tables"], s["parents"], s["max_nodes"],
                                  s["scale"])
    if case["op"] == "commit":
        taken, path, tokens = ops.tree_commit(s["data"], s["cu"], s["lens"], s["tables"], s["parents"], s["draft"],
                                              s["target"], s["max_nodes"], kv_scales=s["scales"])
        out = dict(accepted=taken, path=path, tokens=tokens, data=s["data"])
        return out if s["scales"] is None else dict(out, scales=s["scales"])
    tiled = case["fp8"]
    return ops.moe_few_tokens(s["x"], s["router"], s["w13_tiled"] if tiled else s["w13"], s["s13"],
                              s["w2_tiled"] if tiled else s["w2"], s["s2"], case["experts"], case["topk"],
                              tiled=tiled)


# --------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "commit":
        return None                                        # whole numbers, and cache rows moved as they are
    if case["op"] == "attention":
        nodes, ctx = _lens(case)
        q = s["q"].double()
        out = torch.zeros_like(q)
        group = case["q_heads"] // case["kv_heads"]
        parents = s["parents"].tolist()
        at = 0
        for b, (n, c) in enumerate(zip(nodes, ctx)):
            slot = torch.arange(c + n, device=DEV)
            blk = s["tables"][b].long()[slot // case["block"]]
            allow = torch.zeros(n, c + n, dtype=torch.bool)
            allow[:, :c] = True
            for i in range(n):
                j = i
                while j >= 0:
                    allow[i, c + j] = True
                    j = parents[at + j]
            allow = allow.to(DEV)
            for head in range(case["q_heads"]):
                k = s["k"][blk, head // group, slot % case["block"]].double()
                v = s["v"][blk, head // group, slot % case["block"]].double()
                z = (q[at:at + n, head] @ k.t()) * s["scale"]
                out[at:at + n, head] = torch.softmax(z.masked_fill(~allow, -math.inf), dim=1) @ v
            at += n
        return out
    x = s["x"].double()
    ids, w = _plain_route(s, torch.float64)
    out = torch.zeros_like(x)
    inter = case["inter"]

    def weight(name, e):
        a = s[name][e].double()
        sc = s["s" + name[1:]]
        if sc is None:
            return a
        return a * sc[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)

    for e in sorted(set(ids.flatten().tolist())):
        tok, k = torch.nonzero(ids == e, as_tuple=True)
        z = x[tok] @ weight("w13", e).t()
        a, u = z[:, :inter], z[:, inter:]
        y = (a * torch.sigmoid(a) * u) @ weight("w2", e).t()
        out.index_add_(0, tok, y * w[tok, k, None])
    return out
