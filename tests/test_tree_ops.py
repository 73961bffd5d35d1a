"""Draft-tree operators: tree attention over the paged pool, the commit of the accepted path and the
few-token MoE layer, against plain 64-bit implementations written here."""
import math

import pytest
import torch

from b200moe import ops
from b200moe.config import preset_args
from b200moe.engine.kv_cache import KVPool
from b200moe.models.qwen3_moe import Qwen3MoeForCausalLM, StepInputs
from b200moe.utils.weights import quantize_block_fp8, random_init_

HALF = torch.finfo(torch.bfloat16).eps / 2   # a bf16 rounding is off by at most this, relative to the value
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _tree(n, kind, gen):
    """Parents of a tree of n nodes."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":   # several nodes follow the prefix directly
        return [-1 if i % 3 == 0 else i - 1 for i in range(n)]
    r = torch.rand(n, generator=gen).tolist()
    return ([-1] + [int(r[i] * i) for i in range(1, n)])[:n]


def _sees(par):
    n = len(par)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            m[i, j] = True
            j = par[j]
    return m


class Batch:
    """Pool, tables and trees of a ragged batch; ``pad`` rows of q behind the last sequence."""

    def __init__(self, dev, nodes, ctx, nq, nkv, D, bs, kind="random", int8=False, mode="token", pad=0, seed=0,
                 dtype=torch.bfloat16, layers=2, layer=1):
        g = torch.Generator().manual_seed(seed)
        need = [max(1, -(-(n + c) // bs)) for n, c in zip(nodes, ctx)]
        self.pool = KVPool(sum(need) + 1, layers, nkv, bs, D, dtype, dev, int8=int8, int8_mode=mode)
        ids = torch.randperm(sum(need), generator=g).tolist()
        tab = torch.zeros(len(nodes), max(need) + 1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            tab[b, :k] = torch.tensor(ids[at:at + k])
            at += k
        self.tables = tab.to(dev)
        if int8:
            self.pool.data.copy_(torch.randint(-127, 128, self.pool.data.shape, generator=g, dtype=torch.int8))
            if self.pool.scales is not None:
                self.pool.scales.copy_(torch.rand(self.pool.scales.shape, generator=g) * 0.02 + 0.002)
            else:
                self.pool.side.copy_(torch.randn(self.pool.side.shape, generator=g))
                self.pool.ch_scale.copy_(torch.rand(self.pool.ch_scale.shape, generator=g) * 0.02 + 0.002)
                self.pool.ch_dscale.copy_(self.pool.ch_scale)
                self.pool.n_out.fill_(2)
                self.pool.out_idx[..., 0] = 3
                self.pool.out_idx[..., 1] = D - 1
                for d in (3, D - 1):
                    self.pool.ch_dscale[..., d] = 0.0
        else:
            self.pool.data.copy_(torch.randn(self.pool.data.shape, generator=g))
        self.nodes, self.ctx, self.D, self.nq, self.nkv = nodes, ctx, D, nq, nkv
        cu = [0]
        for n in nodes:
            cu.append(cu[-1] + n)
        self.cu_list = cu
        self.trees = [_tree(n, kind, g) for n in nodes]
        par = [p for t in self.trees for p in t] + [-1] * pad
        i32 = dict(dtype=torch.int32, device=dev)
        self.cu = torch.tensor(cu, **i32)
        self.lens = torch.tensor([n + c for n, c in zip(nodes, ctx)], **i32)
        self.parents = torch.tensor(par, **i32)
        self.q = (torch.randn(cu[-1] + pad, nq, D, generator=g) * 2).to(dtype).to(dev)
        self.layer = self.pool.layer(layer)
        self.scale = D ** -0.5
        self.max_nodes = max(max(nodes), 1)

    def args(self):
        return (self.q, self.layer, self.cu, self.lens, self.tables, self.parents, self.max_nodes, self.scale)

    def exact(self):
        """(o, sum_j p_ij |v_j|) in 64 bits."""
        q = self.q.double().cpu()
        out, mass = torch.zeros_like(q), torch.zeros_like(q)
        for b, (n, c) in enumerate(zip(self.nodes, self.ctx)):
            if n == 0:
                continue
            k, v = (t.double().cpu() for t in self.layer.gather(self.tables[b], n + c))
            see = torch.cat([torch.ones(n, c, dtype=torch.bool), _sees(self.trees[b])], dim=1)
            s0 = self.cu_list[b]
            for h in range(self.nq):
                kv = h // (self.nq // self.nkv)
                z = q[s0:s0 + n, h] @ k[:, kv].t() * self.scale
                p = torch.softmax(z.masked_fill(~see, -math.inf), dim=1)
                out[s0:s0 + n, h] = p @ v[:, kv]
                mass[s0:s0 + n, h] = p @ v[:, kv].abs()
        return out, mass

    def check(self, got):
        """The output is rounded to bf16 once (HALF of its value), and a kernel may round each p_ij to
        bf16 in front of the product and in the sum that divides it (HALF of the mass, twice).  fp32
        scores of at most a few hundred add less than 2^-13 of the mass."""
        o, mass = self.exact()
        n = self.cu_list[-1]
        err = (got[:n].double().cpu() - o[:n]).abs()
        lim = HALF * o[:n].abs() + (2 * HALF + 2 ** -13) * mass[:n] + 1e-30
        assert bool((err <= lim).all()), float((err / lim).max())


ATTN = [
    # nodes, ctx, nq, nkv, D, block
    ([1], [0], 4, 2, 64, 16),
    ([8], [500], 32, 4, 128, 256),
    ([5, 1, 17, 0, 3], [0, 1, 130, 40, 255], 8, 4, 128, 64),
    ([16, 9], [128, 127], 16, 1, 128, 128),          # 16 query heads on one KV head
    ([7, 33], [100, 300], 6, 2, 64, 32),             # a group of three
    ([4, 3, 2], [1023, 1025, 64], 8, 8, 128, 128),   # one query head per KV head
    ([40, 64], [700, 65], 32, 4, 128, 16),           # several row tiles, pages that end inside a key tile
    ([3, 20], [50, 77], 4, 2, 64, 24),               # a block size that no tile divides into
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nodes,ctx,nq,nkv,D,bs", ATTN)
@pytest.mark.parametrize("kind", ["random", "chain", "forest"])
def test_tree_attention(dev, nodes, ctx, nq, nkv, D, bs, kind):
    b = Batch(dev, nodes, ctx, nq, nkv, D, bs, kind)
    got = ops.tree_attention(*b.args())
    b.check(got)
    if dev == "cuda":
        ops.check_status(got.device)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,ctx,nq,nkv,D,bs", [
    ([64], [9000], 32, 4, 128, 256),                 # one request over every SM: parts of one item joined
    ([256, 100], [2500, 4001], 8, 2, 128, 64),       # the largest tree
    ([200], [6000], 16, 1, 64, 128),                 # 25 row tiles of one KV head, key chunks
    ([3, 0, 31, 1, 90], [5000, 7, 1290, 0, 777], 32, 4, 128, 32),
    ([1] * 7, [1500, 20, 3000, 1, 900, 4000, 130], 4, 2, 64, 16),
    ([2] * 300, list(range(300)), 8, 8, 64, 16),
    ([1] * 2300, [i % 5 for i in range(2300)], 4, 4, 64, 8),   # more sequences than one launch takes
])
@pytest.mark.parametrize("kind", ["random", "chain"])
def test_tree_attention_large(nodes, ctx, nq, nkv, D, bs, kind):
    b = Batch("cuda", nodes, ctx, nq, nkv, D, bs, kind)
    out = torch.full_like(b.q, 7.0)
    b.check(ops.tree_attention(*b.args(), out=out))
    ops.check_status(out.device)
    again = ops.tree_attention(*b.args())
    assert torch.equal(out, again)                   # the same shares, joined in the same order


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("mode", ["token", "channel"])
@pytest.mark.parametrize("D,bs", [(128, 64), (64, 16)])
def test_tree_attention_int8(dev, mode, D, bs):
    b = Batch(dev, [9, 1, 24], [40, 300, 0], 8, 2, D, bs, int8=True, mode=mode)
    b.check(ops.tree_attention(*b.args()))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["token", "channel"])
@pytest.mark.parametrize("limit", [None, 1, 3 << 20])
@pytest.mark.parametrize("nodes,ctx,nq,nkv,D,bs", [
    ([64], [9000], 32, 4, 128, 256), ([5, 0, 17, 1, 40], [0, 7, 130, 1500, 255], 8, 2, 64, 8),
    ([3, 90, 31], [5000, 777, 1290], 16, 2, 128, 32), ([4, 3, 2], [50, 77, 9], 4, 2, 64, 24),
])
def test_tree_attention_int8_large(monkeypatch, mode, limit, nodes, ctx, nq, nkv, D, bs):
    """The whole batch, one sequence, or some of them at a time in the bf16 stage; a block size without one."""
    if limit is not None:
        monkeypatch.setattr(ops, "INT8_STAGE_MAX_BYTES", limit)
    b = Batch("cuda", nodes, ctx, nq, nkv, D, bs, int8=True, mode=mode, pad=2)
    out = torch.full_like(b.q, 7.0)
    b.check(ops.tree_attention(*b.args(), out=out))
    assert bool((out[-2:] == 7.0).all())
    ops.check_status(out.device)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_int8_ignores_what_it_does_not_see(dev):
    """NaN factors behind the sequence and in other branches change nothing."""
    b = Batch(dev, [6], [25], 8, 2, 128, 16, "star", int8=True)
    want = ops.tree_attention(*b.args()).clone()
    last, node = b.tables[0, 30 // 16].item(), 25 + 4
    for sc in (b.layer.k_scale, b.layer.v_scale):
        sc[last, :, 15:] = math.nan
        sc[b.tables[0, node // 16].item(), :, node % 16] = math.nan
    got = ops.tree_attention(*b.args())
    keep = [i for i in range(6) if i != 4]
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[4].float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["token", "channel"])
def test_tree_int8_bad_block_sets_status(mode):
    b = Batch("cuda", [4, 3], [40, 20], 8, 2, 128, 16, int8=True, mode=mode)
    want = ops.tree_attention(*b.args()).clone()
    b.tables[0, 0], b.tables[0, 1] = 1 << 20, -5
    got = ops.tree_attention(*b.args())
    assert torch.equal(got[4:], want[4:])
    with pytest.raises(RuntimeError):
        ops.check_status(got.device)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_chain_is_prefill(dev):
    """A chain sees what causal prefill sees."""
    b = Batch(dev, [6, 13], [33, 190], 8, 2, 128, 32, "chain")
    got = ops.tree_attention(*b.args())
    ref = ops.prefill_attention(b.q, b.layer, b.cu, b.lens, b.tables, 13, b.scale, torch.empty_like(b.q))
    _, mass = b.exact()
    lim = 2 * (HALF + 2 * HALF + 2 ** -13) * mass    # both are within check()'s bound of the exact value
    assert bool(((got.double() - ref.double()).abs().cpu() <= lim).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_leaves_padding_rows(dev):
    b = Batch(dev, [3, 5], [20, 70], 8, 2, 128, 16, pad=4)
    out = torch.full_like(b.q, 7.0)
    assert ops.tree_attention(*b.args(), out=out) is out
    assert bool((out[8:] == 7.0).all())
    b.check(out)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_ignores_what_it_does_not_see(dev):
    """NaN and infinite keys and values behind the sequence and in other branches change nothing."""
    b = Batch(dev, [6], [25], 8, 2, 128, 16, "star")
    want = ops.tree_attention(*b.args()).clone()
    last = b.tables[0, 30 // 16].item()
    b.layer.k[last, :, 15:] = math.nan      # slot 31: behind the last node (30 keys + 1)
    b.layer.v[last, :, 15:] = math.inf
    node = 25 + 4                            # node 4: a leaf that only itself sees
    blk = b.tables[0, node // 16].item()
    b.layer.k[blk, :, node % 16] = math.nan
    b.layer.v[blk, :, node % 16] = math.nan
    got = ops.tree_attention(*b.args())
    keep = [i for i in range(6) if i != 4]
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[4].float()).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_large_scores(dev):
    """Scores of many hundreds: the running maximum keeps the exponentials in range."""
    b = Batch(dev, [10], [300], 4, 2, 64, 16)
    b.q *= 50
    got = ops.tree_attention(*b.args())
    assert bool(torch.isfinite(got.float()).all())
    o, mass = b.exact()
    # fp32 products of 64 terms are off by at most 64 * 2^-24 of their absolute sum (below 12,000 here
    # in units of log 2), which moves p by that factor
    z = (b.q.double().abs().amax() * b.layer.k.double().abs().amax() * 64 * b.scale).item()
    lim = HALF * o.abs() + (2 * HALF + 2 * 64 * 2 ** -24 * z) * mass
    assert bool(((got.double().cpu() - o).abs() <= lim).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_attention_empty(dev):
    b = Batch(dev, [0, 0], [5, 0], 4, 2, 64, 16)
    assert ops.tree_attention(*b.args()).shape == (0, 4, 64)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_operators_without_sequences(dev):
    i32 = dict(dtype=torch.int32, device=dev)
    pool = KVPool(3, 2, 2, 16, 64, torch.bfloat16, dev)
    cu, lens, tab = torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 2, **i32)
    for rows in (0, 3):                              # rows that belong to no sequence
        q, par = torch.ones(rows, 4, 64, dtype=torch.bfloat16, device=dev), torch.zeros(rows, **i32)
        out = torch.full_like(q, 7.0)
        ops.tree_attention(q, pool.layer(0), cu, lens, tab, par, 4, 0.1, out=out)
        assert bool((out == 7.0).all())
        acc, path, tokens = ops.tree_commit(pool.data, cu, lens, tab, par, par, par, 4)
        assert acc.shape == (0,) and path.shape == tokens.shape == (0, 4)


@pytest.mark.gpu
def test_tree_operators_in_a_long_pool():
    """Blocks behind 2^31 elements and 2^32 bytes."""
    bs, D, nkv, layers = 256, 128, 4, 8
    need = (1 << 31) // (layers * 2 * nkv * bs * D) + 40
    b = Batch("cuda", [20, 7], [300, 1000], 8, nkv, D, bs, layers=1, layer=0)
    big = KVPool(need, layers, nkv, bs, D, torch.bfloat16, "cuda")
    shift = need - b.pool.num_blocks
    big.data[shift:, layers - 1].copy_(b.pool.data[:, 0])
    tables = (b.tables + shift).to(torch.int32)
    want = ops.tree_attention(*b.args())
    got = ops.tree_attention(b.q, big.layer(layers - 1), b.cu, b.lens, tables, b.parents, b.max_nodes, b.scale)
    assert torch.equal(got, want)
    draft = torch.ones_like(b.parents)
    a = ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, draft, draft, b.max_nodes)
    c = ops.tree_commit(big.data, b.cu, b.lens, tables, b.parents, draft, draft, b.max_nodes)
    assert all(torch.equal(x, y) for x, y in zip(a, c)) and int(a[0].max()) > 1
    assert torch.equal(big.data[shift:, layers - 1], b.pool.data[:, 0])
    ops.check_status(got.device)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_refusals(dev):
    b = Batch(dev, [4], [20], 8, 2, 128, 16)
    q, kv, cu, lens, tab, par, n, sc = b.args()
    bad = [
        (q, kv, cu, lens, tab, par[:3], n, sc), (q, kv, cu[:1], lens, tab, par, n, sc),
        (q, kv, cu.long(), lens, tab, par, n, sc), (q, kv, cu, lens, tab[0], par, n, sc),
        (q, kv, cu, lens, tab, par, 0, sc), (q, kv, cu, lens, tab, par, ops.TREE_MAX_NODES + 1, sc),
        (q.transpose(0, 1), kv, cu, lens, tab, par, n, sc), (q[:, :3].contiguous(), kv, cu, lens, tab, par, n, sc),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            ops.tree_attention(*args)
    for out in (torch.empty(3, 8, 128, dtype=q.dtype, device=dev), torch.empty_like(q, dtype=torch.float16), q):
        with pytest.raises(ValueError):
            ops.tree_attention(*b.args(), out=out)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            ops.tree_attention(q, kv, cu, lens, tab, par, n, scale)
    if dev == "cuda":   # metadata left on the host, a head size without a kernel
        with pytest.raises(ValueError):
            ops.tree_attention(q, kv, cu.cpu(), lens, tab, par, n, sc)
        c = Batch(dev, [4], [20], 8, 2, 32, 16)
        with pytest.raises(ValueError):
            ops.tree_attention(*c.args())
    d = torch.zeros_like(par)
    for args in [(b.pool.data[0], cu, lens, tab, par, d, d, n), (b.pool.data, cu, lens, tab, par, d[:2], d, n),
                 (b.pool.data, cu, lens, tab, par, d, d.long(), n), (b.pool.data, cu, lens, tab, par, d, d, 0)]:
        with pytest.raises(ValueError):
            ops.tree_commit(*args)
    with pytest.raises(ValueError):
        ops.tree_commit(b.pool.data, cu, lens, tab, par, d, d, n, kv_scales=torch.ones(3, device=dev))


@pytest.mark.gpu
def test_tree_bad_metadata_sets_status():
    """Block ids outside the pool, tables that are too short and trees that do not fit are left out."""
    for what in ("block", "short", "cu", "prefix"):
        b = Batch("cuda", [4, 3], [40, 20], 8, 2, 128, 16)
        q, kv, cu, lens, tab, par, n, sc = b.args()
        if what == "block":
            tab[0, 0], tab[0, 1] = 1 << 20, -5
        elif what == "short":
            tab = tab[:, :1].contiguous()
        elif what == "cu":
            cu[2] = 1 << 20
        else:
            lens[0] = 2
        d = torch.zeros_like(par)
        before = b.pool.data.clone()
        ops.tree_attention(q, kv, cu, lens, tab, par, n, sc)
        with pytest.raises(RuntimeError):
            ops.check_status(q.device)
        if what != "block":   # the commit touches the nodes' own blocks only
            t = torch.full_like(par, 1)
            d[2] = 1          # accepts a node that has to move
            par[:4] = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
            ops.tree_commit(b.pool.data, cu, lens, tab, par, d, t, n)
            with pytest.raises(RuntimeError):
                ops.check_status(q.device)
            assert what == "cu" or torch.equal(before, b.pool.data)


def _commit_case(dev, seed, nodes, ctx, int8=False, mode="token", bs=16, layers=3, nkv=2, D=64):
    b = Batch(dev, nodes, ctx, 2 * nkv, nkv, D, bs, int8=int8, mode=mode, seed=seed, layers=layers, pad=2)
    g = torch.Generator().manual_seed(seed + 100)
    rows = b.parents.shape[0]
    # few tokens, so that siblings often draft the same one and paths are long
    draft = torch.randint(0, 3, (rows,), generator=g, dtype=torch.int32)
    target = torch.randint(0, 3, (rows,), generator=g, dtype=torch.int32)
    return b, draft.to(dev), target.to(dev)


def _commit_expect(b, draft, target):
    """Paths by walking lists; moved rows by copying through a snapshot."""
    paths, toks = [], []
    dr, ta = draft.tolist(), target.tolist()
    for q0, par in zip(b.cu_list, b.trees):
        path = [0] if par else []
        while path:
            kids = [c for c in range(len(par)) if par[c] == path[-1] and dr[q0 + c] == ta[q0 + path[-1]]]
            if not kids:
                break
            path.append(min(kids))
        paths.append(path)
        toks.append([ta[q0 + i] for i in path])
    return paths, toks


def _commit_moved(b, paths, t):
    want = t.clone()
    bs = b.pool.block_size
    for i, (n, c, path) in enumerate(zip(b.nodes, b.ctx, paths)):
        for j, node in enumerate(path):
            s, d = c + node, c + j
            want[b.tables[i, d // bs].item(), :, :, :, d % bs] = t[b.tables[i, s // bs].item(), :, :, :, s % bs]
    return want


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("int8,mode", [(False, "token"), (True, "token"), (True, "channel")])
@pytest.mark.parametrize("nodes,ctx", [([1], [0]), ([12, 0, 7, 31], [3, 9, 16, 44]), ([64], [15]), ([2, 2, 200], [0, 31, 5])])
def test_tree_commit(dev, int8, mode, nodes, ctx):
    for seed in range(3):
        b, draft, target = _commit_case(dev, seed, nodes, ctx, int8, mode)
        paths, toks = _commit_expect(b, draft, target)
        tensors = [t for t in (b.pool.data, b.pool.scales, b.pool.side) if t is not None]
        want = [_commit_moved(b, paths, t) for t in tensors]
        acc, path, tokens = ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, draft, target,
                                            b.max_nodes, kv_scales=b.pool.scales, kv_side=b.pool.side)
        assert acc.tolist() == [len(p) for p in paths]
        for i, (p, t) in enumerate(zip(paths, toks)):
            pad = [-1] * (b.max_nodes - len(p))
            assert path[i].tolist() == p + pad and tokens[i].tolist() == t + pad
        for t, w in zip(tensors, want):
            assert torch.equal(t, w)


# ------------------------------------------------------------------ few-token MoE
def _moe_weights(dev, E, H, I, fp8, seed):
    g = torch.Generator().manual_seed(seed)
    router = torch.zeros(-(-E // 128) * 128, H)
    router[:E] = torch.randn(E, H, generator=g) * 2 / math.sqrt(H)
    w13, w2 = (torch.randn(E, n, k, generator=g) * 0.05 for n, k in ((2 * I, H), (H, I)))
    if fp8:
        (w13, s13), (w2, s2) = quantize_block_fp8(w13.to(dev)), quantize_block_fp8(w2.to(dev))
        return router.to(dev, torch.bfloat16), w13, s13, w2, s2
    return router.to(dev, torch.bfloat16), w13.to(dev, torch.bfloat16), None, w2.to(dev, torch.bfloat16), None


def _moe_check(x, router, w13, s13, w2, s2, E, k, renorm, out, ids, wts):
    """Routing exactly, then the outputs for that routing within the bound of its roundings."""
    T, H = x.shape
    I = w2.shape[2]
    xd = x.double()
    logits = (xd @ router[:E].double().t())
    m, e = torch.frexp(logits)
    logits = torch.ldexp(torch.round(m * 256), e - 8)     # bf16, rounded once
    want = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids.long(), want)
    p = torch.softmax(logits, dim=1).gather(1, want)
    if renorm:
        p = p / p.sum(dim=1, keepdim=True)
    # (below 2^-126 a bf16 is a multiple of 2^-133: half of that more)
    assert bool(((wts.double() - p).abs() <= (HALF + 2 ** -18) * p + 2.0 ** -134).all())
    deq = (lambda w, s, g: w[g].double()) if s13 is None else \
        (lambda w, s, g: w[g].double() * s[g].double().repeat_interleave(128, 0).repeat_interleave(128, 1))
    y, lim = torch.zeros_like(xd), torch.zeros_like(xd)
    u32 = 2.0 ** -24
    for g in torch.unique(want).tolist():
        t, j = (want == g).nonzero(as_tuple=True)
        a13, a2 = deq(w13, s13, g), deq(w2, s2, g)
        z, az = xd[t] @ a13.t(), xd[t].abs() @ a13.abs().t()
        gt, up, ag, au = z[:, :I], z[:, I:], az[:, :I], az[:, I:]
        s = gt * torch.sigmoid(gt)
        h = s * up
        # fp32 sums of H terms (H u32 of their absolute sum; the scale adds two roundings), |silu'| < 1.1;
        # silu and the product: a few roundings; the hidden value may be rounded to bf16
        # with e4m3 weights a token may enter as two e4m3 terms, off by 2^-21 of its largest value at most
        dg, du = (H + 4) * u32 * ag, (H + 4) * u32 * au
        if s13 is not None:
            off = 2 ** -21 * xd[t].abs().amax(1, keepdim=True) * a13.abs().sum(1)
            dg, du = dg + off[:, :I], du + off[:, I:]
        dh = 1.1 * dg * up.abs() + s.abs() * du + (HALF + 2 ** -20) * h.abs()
        w = wts.double()[t, j, None]
        y.index_add_(0, t, w * (h @ a2.t()))
        lim.index_add_(0, t, w * (dh @ a2.abs().t() + (I + 8) * u32 * (h.abs() @ a2.abs().t())))
    lim += HALF * y.abs()
    err = (out.double() - y).abs()
    assert bool((err <= lim).all()), float((err / lim).max())


MOE = [  # T, H, I, E, topk, fp8, tiled, renorm
    (1, 256, 128, 8, 2, True, True, True), (5, 256, 128, 8, 2, False, False, True),
    (3, 128, 128, 1, 1, True, False, False), (64, 256, 256, 8, 8, True, True, True),
    (17, 1280, 640, 24, 6, True, True, False), (33, 384, 128, 40, 4, True, False, True),
    (64, 512, 128, 4, 1, False, False, True), (9, 2048, 768, 128, 8, True, True, True),
    (2, 640, 1152, 200, 3, False, False, True),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,H,I,E,k,fp8,tiled,renorm", MOE)
def test_moe_few_tokens(dev, T, H, I, E, k, fp8, tiled, renorm):
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, fp8, seed=T + E)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dev, torch.bfloat16)
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(T, k, dtype=torch.float32, device=dev)
    a13, a2 = (ops.tile_fp8(w13), ops.tile_fp8(w2)) if tiled else (w13, w2)
    out = ops.moe_few_tokens(x, router, a13, s13, a2, s2, E, k, renorm, ids=ids, weights=wts, tiled=tiled)
    _moe_check(x, router, w13, s13, w2, s2, E, k, renorm, out, ids, wts)
    if dev == "cuda":
        ops.check_status(out.device)


@pytest.mark.parametrize("dev", DEVICES)
def test_moe_few_tokens_all_to_one_expert(dev):
    """Every token picks the same experts, and experts that tie: the lowest id wins."""
    E, H, I, k, T = 8, 256, 128, 2, 50
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, True, seed=3)
    router[:E] = router[0]                       # all experts tie
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(9)).to(dev, torch.bfloat16)
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(T, k, dtype=torch.float32, device=dev)
    out = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k, ids=ids, weights=wts)
    assert bool((ids == torch.tensor([0, 1], dtype=torch.int32, device=dev)).all())
    _moe_check(x, router, w13, s13, w2, s2, E, k, True, out, ids, wts)


@pytest.mark.parametrize("dev", DEVICES)
def test_moe_few_tokens_one_bad_token(dev):
    """A token with a NaN gives a NaN row; the other rows do not change."""
    E, H, I, k = 8, 256, 128, 2
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, True, seed=4)
    x = torch.randn(6, H, generator=torch.Generator().manual_seed(2)).to(dev, torch.bfloat16)
    want = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k)
    x[2, 5] = math.nan
    got = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k)
    keep = [0, 1, 3, 4, 5]
    assert bool(torch.isnan(got[2].float()).all())
    # (the CPU path multiplies an expert's rows together: another row may change its last bits)
    assert torch.equal(got[keep], want[keep]) if dev == "cuda" else bool(torch.isfinite(got[keep].float()).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("scale", [2.0 ** -50, 2.0 ** 40])
def test_moe_few_tokens_of_any_size(dev, fp8, scale):
    """Small and large tokens in one batch: every row has its own power of two."""
    E, H, I, k, T = 8, 384, 256, 3, 7
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, fp8, seed=6)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(7))
    x[::2] *= scale
    x[1, 5] *= 1e4                                   # one value far above its row
    x = x.to(dev, torch.bfloat16)
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    wts = torch.empty(T, k, dtype=torch.float32, device=dev)
    out = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k, ids=ids, weights=wts)
    _moe_check(x, router, w13, s13, w2, s2, E, k, True, out, ids, wts)


@pytest.mark.parametrize("dev", DEVICES)
def test_moe_few_tokens_zero_and_infinite_rows(dev):
    """Logits of -0 tie with 0; an infinity spoils its own row alone."""
    E, H, I, k = 8, 256, 128, 3
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, True, seed=8)
    x = torch.randn(5, H, generator=torch.Generator().manual_seed(3)).to(dev, torch.bfloat16)
    want = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k)
    x[0] = 0
    x[1] = 0
    x[1, 9] = 2.0 ** -133                            # logits below the smallest bf16: +0 and -0
    x[2, 4] = math.inf
    ids = torch.empty(5, k, dtype=torch.int32, device=dev)
    got = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, k, ids=ids)
    assert ids[:2].tolist() == [[0, 1, 2]] * 2
    assert bool((got[:2] == 0).all()) and not bool(torch.isfinite(got[2].float()).any())
    assert torch.equal(got[3:], want[3:]) if dev == "cuda" else bool(torch.isfinite(got[3:].float()).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_moe_few_refusals(dev):
    E, H, I, k = 8, 256, 128, 2
    router, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, True, seed=4)
    x = torch.zeros(ops.MOE_FEW_MAX_TOKENS + 1, H, dtype=torch.bfloat16, device=dev)
    ok = (router, w13, s13, w2, s2, E, k)
    for xx, args in [(x, ok), (x[:4, ::2], ok), (x[:4], (router, w13, None, w2, None, E, k)),
                     (x[:4], (router, w13, s13, w2, s2, E, 9)), (x[:4], (router, w13[:4], s13, w2, s2, E, k)),
                     (x[:4], (router, w13, s13, w2.transpose(1, 2), s2, E, k))]:
        with pytest.raises(ValueError):
            ops.moe_few_tokens(xx, *args)
    for out in (x[:3], x[:4], x[2:6]):
        with pytest.raises(ValueError):
            ops.moe_few_tokens(x[:4], *ok, out=out)
    assert ops.moe_few_tokens(x[:0], *ok).shape == (0, H)


# ------------------------------------------------------------------ together, in the model
class Decoder:
    """Sequences with a block table each, stepped through a tiny model."""

    def __init__(self, dev, prompts, preset="tiny-moe", int8=False, blocks=12, bs=16):
        self.args = preset_args(preset)
        self.dev, self.bs = dev, bs
        self.model = Qwen3MoeForCausalLM(self.args, dev)
        random_init_(self.model, seed=5, std=0.1)
        self.model.reserve_workspace(256, 16, 8)
        a = self.args
        self.pool = KVPool(len(prompts) * blocks + 1, a.num_hidden_layers, a.num_key_value_heads, bs, a.head_dim,
                           self.model.dtype, dev, int8=int8)
        g = torch.Generator().manual_seed(1)
        self.tables = torch.randperm(len(prompts) * blocks, generator=g).view(len(prompts), blocks).tolist()
        self.seqs = [list(p) for p in prompts]      # the last token's key is not stored yet

    def inputs(self, rows, ids, parents=None, num_decode=0):
        """rows: (sequence, keys already stored, tokens); parents per row: trees."""
        i32 = dict(dtype=torch.int32, device=self.dev)
        pos, slots, cu = [], [], [0]
        for j, (s, p, n) in enumerate(rows):
            depth = list(range(n))
            if parents is not None:
                for i, up in enumerate(parents[j]):
                    depth[i] = 0 if up < 0 else depth[up] + 1
            pos += [p + d for d in depth]
            slots += [self.tables[s][(p + i) // self.bs] * self.bs + (p + i) % self.bs for i in range(n)]
            cu.append(cu[-1] + n)
        lens = [p + n for _, p, n in rows]
        want = list(range(cu[-1])) if parents is not None else [c - 1 for c in cu[1:]]
        return StepInputs(torch.tensor(ids, **i32), torch.tensor(pos, **i32), torch.tensor(slots, **i32),
                          torch.tensor(cu, **i32), torch.tensor(lens, **i32),
                          torch.tensor([self.tables[s] for s, _, _ in rows], **i32), torch.tensor(want, **i32),
                          num_decode, max(n for _, _, n in rows), max(lens), len(rows),
                          tree_parents=None if parents is None else
                          torch.tensor([p for t in parents for p in t], **i32))

    def prefill(self):
        rows = [(s, 0, len(t) - 1) for s, t in enumerate(self.seqs)]
        self.model(self.inputs(rows, [i for t in self.seqs for i in t[:-1]]), self.pool)

    def greedy(self, steps):
        for _ in range(steps):
            rows = [(s, len(t) - 1, 1) for s, t in enumerate(self.seqs)]
            h = self.model(self.inputs(rows, [t[-1] for t in self.seqs], num_decode=len(rows)), self.pool)
            for t, n in zip(self.seqs, ops.argmax(self.model.compute_logits(h)).tolist()):
                t.append(n)

    def drafts(self, truth, right, g):
        """A random tree per sequence; along one of its paths ``right`` drafts are what comes next."""
        parents, ids = [], []
        for s, t in enumerate(self.seqs):
            n = int(torch.randint(2, 10, (1,), generator=g))
            par = _tree(n, "random", g)
            tok = [t[-1]] + torch.randint(0, self.args.vocab_size, (n - 1,), generator=g).tolist()
            at, deep = 0, 0
            for i in range(1, n):
                if par[i] == at and deep < right:
                    tok[i] = truth[s][len(t) + deep]
                    at, deep = i, deep + 1
            parents.append(par)
            ids.append(tok)
        return parents, ids

    def verify(self, parents, ids):
        rows = [(s, len(t) - 1, len(p)) for s, (t, p) in enumerate(zip(self.seqs, parents))]
        inp = self.inputs(rows, [i for t in ids for i in t], parents)
        acc, path, tokens = self.model.verify_trees(inp, self.pool)
        for t, a, tok in zip(self.seqs, acc.tolist(), tokens.tolist()):
            t += tok[:a]
        return acc.tolist()


PROMPTS = [[5, 900, 33, 7], [1, 2], list(range(40, 75)), [8] * 17]


@pytest.mark.parametrize("int8", [False, True])
def test_verified_trees_emit_the_greedy_tokens(int8):
    """Steps that verify trees emit what one decode step per token emits (fp32 model on the CPU)."""
    ref, got = Decoder("cpu", PROMPTS, int8=int8), Decoder("cpu", PROMPTS, int8=int8)
    ref.prefill()
    ref.greedy(40)
    got.prefill()
    g = torch.Generator().manual_seed(2)
    steps = []
    for _ in range(5):
        steps += got.verify(*got.drafts(ref.seqs, 4, g))
    for a, b, p in zip(got.seqs, ref.seqs, PROMPTS):
        assert a == b[:len(a)] and len(a) >= len(p) + 5
    assert max(steps) > 2                            # paths were accepted
    # The rows kept are those of the sequences.  A layer-0 row depends on its token and position alone: it is
    # rounded to bf16, where the fp32 noise of another batch size (2^-20) may fall on the other side of a
    # border (one step, 2 HALF of the value); the int8 pool adds one step of the row's scale, amax / 127.
    for s, t in enumerate(got.seqs):
        for x, y in zip(*(d.pool.layer(0).gather(torch.tensor(d.tables[s]), len(t) - 1) for d in (got, ref))):
            lim = 2 * HALF * x.abs() + 2 ** -20
            if int8:
                lim = x.abs().amax(-1, keepdim=True) * (1.01 / 127 + 2 * HALF)
            assert bool(((x - y).abs() <= lim).all())


def test_decode_and_tree_rows_in_one_step():
    """Decode rows in front of tree rows: each gets what it gets alone."""
    g = torch.Generator().manual_seed(3)
    trees = [_tree(n, "random", g) for n in (5, 1, 8)]
    ids = [[t[-1]] + torch.randint(0, 1000, (len(p) - 1,), generator=g).tolist() for t, p in zip(PROMPTS[1:], trees)]

    def step(decode, tree):
        d = Decoder("cpu", PROMPTS)
        d.prefill()
        rows = ([(0, len(d.seqs[0]) - 1, 1)] if decode else []) + \
            ([(s + 1, len(PROMPTS[s + 1]) - 1, len(p)) for s, p in enumerate(trees)] if tree else [])
        toks = ([d.seqs[0][-1]] if decode else []) + ([i for t in ids for i in t] if tree else [])
        inp = d.inputs(rows, toks, ([[-1]] if decode else []) + (trees if tree else []), num_decode=int(decode))
        inp.tree_parents = inp.tree_parents[int(decode):].contiguous() if tree else None
        if decode:
            inp.prefill_cu = (inp.cu_seqlens_q[1:] - 1).contiguous()
        return d.model(inp, d.pool)

    both = step(True, True)
    # (fp32 sums in another order; a K or V at the border of two bf16 values may move by one of their steps)
    torch.testing.assert_close(both, torch.cat([step(True, False), step(False, True)]), atol=2e-2, rtol=0)


def test_verify_refuses_other_steps():
    d = Decoder("cpu", PROMPTS)
    rows = [(s, len(t) - 1, 1) for s, t in enumerate(d.seqs)]
    with pytest.raises(ValueError):
        d.model.verify_trees(d.inputs(rows, [t[-1] for t in d.seqs], num_decode=len(rows)), d.pool)
    inp = d.inputs(rows, [t[-1] for t in d.seqs], [[-1]] * len(rows))
    inp.logits_indices = inp.logits_indices[:2]
    with pytest.raises(ValueError):
        d.model.verify_trees(inp, d.pool)


@pytest.mark.gpu
@pytest.mark.parametrize("preset,int8,few", [("tiny-moe-fp8", False, 0), ("tiny-moe-fp8", False, 64),
                                             ("tiny-moe", False, 64), ("tiny-moe-fp8", True, 64)])
def test_verified_trees_in_the_model_gpu(monkeypatch, preset, int8, few):
    """Every operator call inside a verification step, on what the model hands it, against the exact values."""
    d = Decoder("cuda", PROMPTS, preset, int8=int8)
    d.model.MOE_FEW_ROWS = few
    d.prefill()
    seen = {"attn": 0, "moe": 0, "commit": 0}
    attn, moe, commit = ops.tree_attention, ops.moe_few_tokens, ops.tree_commit
    g = torch.Generator().manual_seed(2)

    def check_attn(q, layer, cu, lens, tables, parents, max_q, scale, out):
        got = attn(q, layer, cu, lens, tables, parents, max_q, scale, out)
        b = Batch.__new__(Batch)
        b.q, b.layer, b.scale, b.tables, b.nq = q, layer, scale, tables, q.shape[1]
        b.cu_list, b.nkv = cu.tolist(), layer.num_kv_heads
        b.nodes = [y - x for x, y in zip(b.cu_list, b.cu_list[1:])]
        b.ctx = [n - k for n, k in zip(lens.tolist(), b.nodes)]
        b.trees = [parents.tolist()[x:y] for x, y in zip(b.cu_list, b.cu_list[1:])]
        b.check(got)
        seen["attn"] += 1
        return got

    def check_moe(x, router, w13, s13, w2, s2, E, k, renorm, out, tiled):
        ids = torch.empty(x.shape[0], k, dtype=torch.int32, device=x.device)
        wts = torch.empty(x.shape[0], k, device=x.device)
        moe(x, router, w13, s13, w2, s2, E, k, renorm, out=out, ids=ids, weights=wts, tiled=tiled)
        _moe_check(x, router, w13, s13, w2, s2, E, k, renorm, out, ids, wts)
        seen["moe"] += 1
        return out

    def check_commit(data, cu, lens, tables, parents, draft, target, max_q, kv_scales=None, kv_side=None):
        b = Batch.__new__(Batch)
        b.cu_list, b.tables, b.pool = cu.tolist(), tables, d.pool
        b.nodes = [y - x for x, y in zip(b.cu_list, b.cu_list[1:])]
        b.ctx = [n - k for n, k in zip(lens.tolist(), b.nodes)]
        b.trees = [parents.tolist()[x:y] for x, y in zip(b.cu_list, b.cu_list[1:])]
        paths, toks = _commit_expect(b, draft, target)
        kept = [t for t in (data, kv_scales, kv_side) if t is not None]
        want = [_commit_moved(b, paths, t) for t in kept]
        res = commit(data, cu, lens, tables, parents, draft, target, max_q, kv_scales=kv_scales, kv_side=kv_side)
        assert res[0].tolist() == [len(p) for p in paths]
        assert [t[:len(p)] for t, p in zip(res[2].tolist(), paths)] == toks
        for t, w in zip(kept, want):
            assert torch.equal(t, w)
        seen["commit"] += 1
        return res

    monkeypatch.setattr(ops, "tree_attention", check_attn)
    monkeypatch.setattr(ops, "moe_few_tokens", check_moe)
    monkeypatch.setattr(ops, "tree_commit", check_commit)
    truth = [t + list(range(1, 99)) for t in d.seqs]
    for _ in range(3):
        d.verify(*d.drafts(truth, 4, g))
    layers = d.args.num_hidden_layers
    assert seen == {"attn": 3 * layers, "moe": 3 * layers if few else 0, "commit": 3}
    ops.check_status(d.pool.data.device)


@pytest.mark.gpu
def test_verify_step_replays_from_a_graph():
    """A captured step (three operators on their workspaces) run over new inputs in its buffers gives what
    the eager step gives."""
    g = torch.Generator().manual_seed(4)
    eager, graph = Decoder("cuda", PROMPTS, "tiny-moe-fp8"), Decoder("cuda", PROMPTS, "tiny-moe-fp8")
    n = 6
    for d in (eager, graph):
        d.model.MOE_FEW_ROWS = 64
        d.prefill()

    def step_inputs(d, trees, ids):
        return d.inputs([(s, len(t) - 1, n) for s, t in enumerate(d.seqs)], [i for t in ids for i in t], trees)

    batches = [([_tree(n, "random", g) for _ in PROMPTS],
                [torch.randint(0, 1000, (n,), generator=g).tolist() for _ in PROMPTS]) for _ in range(3)]
    static = step_inputs(graph, *batches[0])
    start = graph.pool.data.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.model.verify_trees(static, graph.pool)     # warm-up
    torch.cuda.current_stream().wait_stream(side)
    cg = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        res = graph.model.verify_trees(static, graph.pool)
    graph.pool.data.copy_(start)
    for trees, ids in batches:
        want = eager.model.verify_trees(step_inputs(eager, trees, ids), eager.pool)
        new = step_inputs(graph, trees, ids)
        for name in ("input_ids", "positions", "slot_mapping", "seq_lens", "tree_parents"):
            getattr(static, name).copy_(getattr(new, name))
        cg.replay()
        for a, b in zip(res, want):
            assert torch.equal(a, b)
        assert torch.equal(eager.pool.data, graph.pool.data)
        for d in (eager, graph):
            for t, a, tok in zip(d.seqs, want[0].tolist(), want[2].tolist()):
                t += tok[:a]
    ops.check_status(static.input_ids.device)


@pytest.mark.gpu
def test_operators_on_two_streams():
    """Calls in flight on two streams at once keep their results: each has its own workspace."""
    b = [Batch("cuda", [64, 3], [3000, 200], 32, 4, 128, 64, seed=s) for s in range(2)]
    m = [_moe_weights("cuda", 24, 256, 128, True, seed=s) for s in range(2)]
    x = [torch.randn(32, 256, generator=torch.Generator().manual_seed(s)).to("cuda", torch.bfloat16) for s in range(2)]
    want = [(ops.tree_attention(*b[i].args()), ops.moe_few_tokens(x[i], *m[i], 24, 4)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.tree_attention(*b[i].args()), ops.moe_few_tokens(x[i], *m[i], 24, 4)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, y in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(y, want[i][1])
    ops.check_status(x[0].device)


@pytest.mark.gpu
def test_operators_in_two_graphs_of_one_pool():
    """Two captured graphs that share a memory pool, replayed in turn over new inputs: a workspace holds nothing
    from one call to the next."""
    def case(seed):
        b = Batch("cuda", [30, 7], [2500, 300], 32, 4, 128, 32, seed=seed)
        w = _moe_weights("cuda", 24, 256, 128, True, seed=seed)
        x = torch.randn(20, 256, generator=torch.Generator().manual_seed(seed)).to("cuda", torch.bfloat16)
        return b, w, x

    def run(b, w, x):
        return ops.tree_attention(*b.args()), ops.moe_few_tokens(x, *w, 24, 4)

    cases, graphs, outs = [case(s) for s in range(2)], [], []
    run(*cases[0])                                   # warm-up
    torch.cuda.synchronize()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(run(*c))
        graphs.append(g)
    for r in range(3):
        for c in cases:
            c[0].q.copy_(torch.randn(c[0].q.shape, generator=torch.Generator().manual_seed(r)))
            c[2].mul_(1.25)
        for g in graphs:
            g.replay()
        for c, got in zip(cases, outs):
            assert all(torch.equal(a, b) for a, b in zip(got, run(*c)))
    ops.check_status("cuda:0")


# ------------------------------------------------------------------ what the cases above do not reach
FORMS = [(16, False, "token"), (64, False, "token"), (24, False, "token"), (48, False, "token"), (96, False, "token"),
         (16, True, "token"), (48, True, "token"), (16, True, "channel"), (48, True, "channel")]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs,int8,mode", FORMS)
def test_tree_attention_nan_query(dev, bs, int8, mode):
    """A NaN in one head of one query makes that head of that node NaN and changes nothing else."""
    b = Batch(dev, [7, 1, 12], [50, 0, 170], 8, 2, 64, bs, int8=int8, mode=mode)
    want = ops.tree_attention(*b.args()).clone()
    b.q[9, 3, 5] = b.q[7, 0, 0] = math.nan       # a node of the third tree, the only one of the second
    got = ops.tree_attention(*b.args())
    hit = torch.zeros(20, 8, dtype=torch.bool, device=dev)
    hit[9, 3] = hit[7, 0] = True
    assert bool(torch.isnan(got[hit].float()).all())
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs", [16, 64, 24, 48, 96])
@pytest.mark.parametrize("keys", [1, 32, 75])
def test_tree_attention_nan_keys_in_front(dev, bs, keys):
    """The first keys of a prefix are NaN: so is every node of that sequence, and no other."""
    b = Batch(dev, [7, 5], [120, 60], 8, 2, 64, bs)
    want = ops.tree_attention(*b.args()).clone()
    for y in range(keys):
        b.layer.k[b.tables[0, y // bs].item(), :, y % bs] = math.nan
    got = ops.tree_attention(*b.args())
    assert bool(torch.isnan(got[:7].float()).all())
    assert torch.equal(got[7:], want[7:])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs,ctx", [(16, 60), (64, 60), (64, 9000), (48, 60)])
def test_tree_attention_infinite_keys(dev, bs, ctx):
    """Keys that score -inf weigh nothing; a node that sees no other has no softmax and is NaN."""
    b = Batch(dev, [4, 1], [ctx, 200], 8, 2, 64, bs, "star")
    b.q.copy_(b.q.abs() + 1)
    some = {y for y in range(ctx) if y % 3 == 0}
    for y in some:
        b.layer.k[b.tables[0, y // bs].item(), :, y % bs] = -math.inf
    got = ops.tree_attention(*b.args())
    b.check(got)
    for y in set(range(ctx + 2)) - some:         # all that node 1 sees: the prefix, node 0 and itself
        b.layer.k[b.tables[0, y // bs].item(), :, y % bs] = -math.inf
    last = ops.tree_attention(*b.args())
    assert bool(torch.isnan(last[:2].float()).all())
    assert torch.equal(last[4], got[4])          # the other sequence
    assert bool(torch.isfinite(last[2:4].float()).all())   # nodes 2 and 3 see themselves


@pytest.mark.gpu
@pytest.mark.parametrize("bs,int8", [(16, False), (48, False), (16, True)])
def test_tree_offsets_whose_difference_wraps(bs, int8):
    """Offsets 2^31 - 1 and -2^31 + 3: their difference, 4 in 32 bits, is not a tree of 4 nodes."""
    b = Batch("cuda", [3, 5, 4, 6, 2], [40, 9, 40, 43, 70], 8, 2, 64, bs, int8=int8)
    want = ops.tree_attention(*b.args()).clone()
    b.cu[2], b.cu[3] = (1 << 31) - 1, -(1 << 31) + 3
    out = torch.full_like(b.q, 7.0)
    ops.tree_attention(*b.args(), out=out)
    assert torch.equal(out[:3], want[:3]) and bool((out[3:18] == 7.0).all())
    with pytest.raises(RuntimeError):
        ops.check_status(out.device)
    draft = torch.zeros_like(b.parents)
    acc = ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, draft, draft, b.max_nodes,
                          kv_scales=b.pool.scales)[0]
    assert [int(n) > 0 for n in acc.tolist()] == [True, False, False, False, True]
    with pytest.raises(RuntimeError):
        ops.check_status(out.device)


# offsets past the rows, below zero, that descend
BAD_CU = [(1, 1 << 20), (2, 1 << 20), (1, -7), (2, 0), (2, -(1 << 31))]


@pytest.mark.gpu
@pytest.mark.parametrize("bs,int8", [(16, False), (128, False), (48, False), (16, True)])
@pytest.mark.parametrize("ctx", [40, 5000])
@pytest.mark.parametrize("at,value", BAD_CU)
def test_tree_bad_offset_leaves_the_other_trees(bs, int8, ctx, at, value):
    """An offset outside the rows spoils the two trees that it bounds; the others are right."""
    if bs == 48 and ctx > 1000:
        ctx = 300                                # the form without tensor cores
    b = Batch("cuda", [3, 5, 4, 6, 2], [ctx, 9, ctx, ctx + 3, 70], 8, 2, 64, bs, int8=int8)
    want = ops.tree_attention(*b.args()).clone()
    b.cu[at] = value
    out = torch.full_like(b.q, 7.0)
    ops.tree_attention(*b.args(), out=out)
    rows = torch.zeros(20, dtype=torch.bool, device="cuda")   # of the trees between at - 1 and at + 1
    rows[b.cu_list[at - 1]:b.cu_list[at + 1]] = True
    kept = out.clone()
    kept[rows] = want[rows]
    b.check(kept)
    with pytest.raises(RuntimeError):
        ops.check_status(out.device)
    # the commit too accepts nothing of the two
    draft = torch.zeros_like(b.parents)
    acc, path, _ = ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, draft, draft, b.max_nodes,
                                   kv_scales=b.pool.scales)
    bad = [i for i in range(5) if i in (at - 1, at)]
    assert [i for i, n in enumerate(acc.tolist()) if n == 0] == bad and bool((path[bad] == -1).all())
    with pytest.raises(RuntimeError):
        ops.check_status(out.device)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 64])
@pytest.mark.parametrize("at", [0, 1, 6])
def test_moe_few_tokens_logit_beside_a_tie(dev, T, at):
    """Logits 1 + 2^-8 + 2^-30 and 1 + 2^-8 - 2^-30 lie beside a border of two bf16 values, 1 and 1 + 2^-7:
    the bit far below decides, and with it the expert."""
    E, H, I = 8, 256, 128
    _, w13, s13, w2, s2 = _moe_weights(dev, E, H, I, True, seed=5)
    router = torch.zeros(128, H)
    router[:E, 3] = -4.0
    x = torch.zeros(T, H)
    x[:, [at, 7, 200]] = 1.0
    lo, up = 2, 5
    router[lo, :] = 0
    router[up, :] = 0
    router[lo, [at, 7, 200]] = torch.tensor([1.0, 2.0 ** -8, -2.0 ** -30])
    router[up, [at, 7, 200]] = torch.tensor([1.0, 2.0 ** -30, 2.0 ** -8])
    router[:2, [at]] = -1.0
    x, router = x.to(dev, torch.bfloat16), router.to(dev, torch.bfloat16)
    ids = torch.empty(T, 2, dtype=torch.int32, device=dev)
    wts = torch.empty(T, 2, dtype=torch.float32, device=dev)
    out = ops.moe_few_tokens(x, router, w13, s13, w2, s2, E, 2, ids=ids, weights=wts)
    assert ids.tolist() == [[up, lo]] * T
    _moe_check(x, router, w13, s13, w2, s2, E, 2, True, out, ids, wts)


@pytest.mark.gpu
def test_tree_operators_count_their_launches(monkeypatch):
    def launches(b, limit=None):
        if limit is not None:
            monkeypatch.setattr(ops, "INT8_STAGE_MAX_BYTES", limit)
        before = ops.launch_count()
        ops.tree_attention(*b.args())
        return ops.launch_count() - before

    assert launches(Batch("cuda", [4, 3], [40, 20], 8, 2, 64, 16)) == 1
    assert launches(Batch("cuda", [4, 3], [40, 20], 8, 2, 64, 48)) == 1
    assert launches(Batch("cuda", [1] * 1025, [2] * 1025, 4, 2, 64, 8)) == 2     # 1024 sequences at a time
    b = Batch("cuda", [4, 3, 2], [40, 20, 9], 8, 2, 64, 16, int8=True)
    assert launches(b) == 2                      # the stage and the attention that reads it
    assert launches(b, limit=1) == 6             # one sequence at a time
    assert launches(Batch("cuda", [4, 3], [40, 20], 8, 2, 64, 24, int8=True)) == 1
    assert launches(Batch("cuda", [0, 0], [5, 0], 8, 2, 64, 16)) == 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs,int8", [(16, False), (48, False), (16, True), (48, True)])
def test_tree_operators_take_a_view_of_a_wider_table(dev, bs, int8):
    b = Batch(dev, [5, 1, 9], [70, 0, 130], 8, 2, 64, bs, int8=int8)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=dev)
    wide[:, :b.tables.shape[1]] = b.tables
    view = wide[:, :b.tables.shape[1]]
    assert not view.is_contiguous()
    want = ops.tree_attention(*b.args())
    got = ops.tree_attention(b.q, b.layer, b.cu, b.lens, view, b.parents, b.max_nodes, b.scale)
    assert torch.equal(got, want)
    data, scales = b.pool.data.clone(), None if b.pool.scales is None else b.pool.scales.clone()
    draft = torch.ones_like(b.parents)
    args = (draft, draft, b.max_nodes)
    x = ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, *args, kv_scales=b.pool.scales)
    y = ops.tree_commit(data, b.cu, b.lens, view, b.parents, *args, kv_scales=scales)
    assert all(torch.equal(s, t) for s, t in zip(x, y)) and torch.equal(data, b.pool.data)
    with pytest.raises(ValueError):              # rows that are not contiguous
        ops.tree_attention(b.q, b.layer, b.cu, b.lens, wide.t().contiguous().t(), b.parents, b.max_nodes, b.scale)


def test_verify_step_narrows_the_tables_of_an_int8_pool(monkeypatch):
    """The stage of an int8 pool is as wide as the tables: the model hands over the columns that the step uses."""
    attn, widths = ops.tree_attention, []

    def spy(q, layer, cu, lens, tables, *rest):
        widths.append(tables.shape[1])
        return attn(q, layer, cu, lens, tables, *rest)

    monkeypatch.setattr(ops, "tree_attention", spy)
    for int8 in (False, True):
        d = Decoder("cpu", PROMPTS, int8=int8)
        d.prefill()
        truth = [t + list(range(1, 99)) for t in d.seqs]
        parents, ids = d.drafts(truth, 2, torch.Generator().manual_seed(3))
        longest = max(len(t) - 1 + len(p) for t, p in zip(d.seqs, parents))
        widths.clear()
        d.verify(parents, ids)
        assert set(widths) == {-(-longest // d.bs) if int8 else 12}


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["token", "channel"])
def test_tree_int8_stage_stays_within_its_limit(mode):
    """64 short sequences in tables of 200 blocks would fill a stage of 1.7 GB: the call allocates no more than the
    limit, and with the columns in use alone a small stage and two launches."""
    b = Batch("cuda", [8] * 64, [300] * 64, 32, 4, 128, 64, int8=True, mode=mode)
    wide = torch.zeros(64, 200, dtype=torch.int32, device="cuda")
    wide[:, :b.tables.shape[1]] = b.tables
    want = ops.tree_attention(*b.args())

    def call(tables):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        mem, before = torch.cuda.memory_allocated(), ops.launch_count()
        out = ops.tree_attention(b.q, b.layer, b.cu, b.lens, tables, b.parents, b.max_nodes, b.scale)
        torch.cuda.synchronize()
        return out, torch.cuda.max_memory_allocated() - mem, ops.launch_count() - before

    rest = 148 * 2 * 128 * (128 * 4 + 8) + want.nbytes + (4 << 20)   # partial results, the output, rounding
    out, used, _ = call(wide)
    b.check(out)
    assert used <= (512 << 20) + rest
    out, used, launches = call(wide[:, :b.tables.shape[1]])
    assert torch.equal(out, want) and launches == 2
    assert used <= 64 * b.tables.shape[1] * 64 * 4 * (128 * 4 + 8) + rest


@pytest.mark.parametrize("what", ["long", "descend", "outside", "prefix", "table", "block", "negative"])
def test_tree_operators_on_the_cpu_refuse_what_does_not_fit(what):
    """What the kernels leave out and report in the status word is a ValueError on the CPU."""
    b = Batch("cpu", [4, 9, 3], [40, 20, 5], 8, 2, 64, 16, "star")
    q, kv, cu, lens, tab, par, n, sc = b.args()
    draft = torch.zeros_like(par)
    target = torch.zeros_like(par)
    draft[4 + 1:4 + 9] = 1                       # the second tree accepts its last node alone: a row moves
    draft[4 + 8] = 0
    if what == "long":
        n = 8                                    # of 9 nodes
    elif what == "descend":
        cu[1], cu[2] = 13, 4
    elif what == "outside":
        cu[3] = 17
    elif what == "prefix":
        lens[1] = 8
    elif what == "table":
        tab = tab[:, :1].contiguous()            # the nodes lie in the second block
    else:
        tab[1, 1] = b.pool.num_blocks if what == "block" else -1
    before = b.pool.data.clone()
    with pytest.raises(ValueError):
        ops.tree_attention(q, kv, cu, lens, tab, par, n, sc)
    with pytest.raises(ValueError):
        ops.tree_commit(b.pool.data, cu, lens, tab, par, draft, target, n)
    assert torch.equal(before, b.pool.data)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_operators_refuse_a_pool_without_slots(dev):
    b = Batch(dev, [4], [20], 8, 2, 128, 16)
    d = torch.zeros_like(b.parents)
    shape = list(b.pool.data.shape)
    for dim in (1, 3, 4):                        # no layers, no heads, blocks of no rows
        data = b.pool.data.new_zeros([0 if i == dim else n for i, n in enumerate(shape)])
        with pytest.raises(ValueError):
            ops.tree_commit(data, b.cu, b.lens, b.tables, b.parents, d, d, b.max_nodes)
    empty = KVPool(3, 1, 2, 0, 128, torch.bfloat16, dev)
    with pytest.raises(ValueError):
        ops.tree_attention(b.q, empty.layer(0), b.cu, b.lens, b.tables, b.parents, b.max_nodes, b.scale)


@pytest.mark.parametrize("dev", DEVICES)
def test_tree_commit_refuses_int8_rows_without_their_scales(dev):
    """Moving the payload alone would leave every moved row with another row's scale."""
    for mode in ("token", "channel"):
        b, draft, target = _commit_case(dev, 1, [6, 3], [10, 4], True, mode)
        before = b.pool.data.clone()
        with pytest.raises(ValueError):
            ops.tree_commit(b.pool.data, b.cu, b.lens, b.tables, b.parents, draft, target, b.max_nodes)
        assert torch.equal(before, b.pool.data)


@pytest.mark.gpu
def test_tree_commit_of_more_sequences_than_a_grid_is_high():
    """65,540 trees of three nodes: a grid has 65,535 rows of blocks at most."""
    B, n, bs = 65540, 3, 4
    i32 = dict(dtype=torch.int32, device="cuda")
    data = torch.randn(B, 1, 2, 1, bs, 8, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    cu, lens = torch.arange(0, B * n + 1, n, **i32), torch.full((B,), n + 1, **i32)
    tables = torch.arange(B, **i32).flip(0).unsqueeze(1).contiguous()
    parents = torch.tensor([-1, 0, 0], **i32).repeat(B)
    draft = torch.tensor([9, 1, 2], **i32).repeat(B)
    target = torch.tensor([2, 0, 0], **i32).repeat(B)        # node 2 is accepted: slot 3 moves to slot 2
    want = data.clone()
    want[:, :, :, :, 2] = data[:, :, :, :, 3]
    before = ops.launch_count()
    acc, path, tokens = ops.tree_commit(data, cu, lens, tables, parents, draft, target, n)
    assert ops.launch_count() - before == 2
    assert bool((acc == 2).all()) and torch.equal(data, want)
    assert bool((path == torch.tensor([0, 2, -1], **i32)).all())
    assert bool((tokens == torch.tensor([2, 0, -1], **i32)).all())
    ops.check_status(data.device)


class Spy:
    """The tree operators of a model's steps, each call checked against the exact values."""

    def __init__(self, monkeypatch, pool):
        self.attn, self.commit, self.pool = ops.tree_attention, ops.tree_commit, pool
        self.calls = {"attn": 0, "commit": 0}
        monkeypatch.setattr(ops, "tree_attention", self.check_attn)
        monkeypatch.setattr(ops, "tree_commit", self.check_commit)

    @staticmethod
    def batch(cu, lens, tables, parents):
        b = Batch.__new__(Batch)
        b.cu_list, b.tables = cu.tolist(), tables
        b.nodes = [y - x for x, y in zip(b.cu_list, b.cu_list[1:])]
        b.ctx = [n - k for n, k in zip(lens.tolist(), b.nodes)]
        b.trees = [parents.tolist()[x:y] for x, y in zip(b.cu_list, b.cu_list[1:])]
        return b

    def check_attn(self, q, layer, cu, lens, tables, parents, max_q, scale, out):
        got = self.attn(q, layer, cu, lens, tables, parents, max_q, scale, out)
        b = self.batch(cu, lens, tables, parents)
        b.q, b.layer, b.scale, b.nq, b.nkv = q, layer, scale, q.shape[1], layer.num_kv_heads
        b.check(got)
        self.calls["attn"] += 1
        return got

    def check_commit(self, data, cu, lens, tables, parents, draft, target, max_q, kv_scales=None, kv_side=None):
        b = self.batch(cu, lens, tables, parents)
        b.pool = self.pool
        paths, toks = _commit_expect(b, draft, target)
        kept = [t for t in (data, kv_scales, kv_side) if t is not None]
        want = [_commit_moved(b, paths, t) for t in kept]
        res = self.commit(data, cu, lens, tables, parents, draft, target, max_q, kv_scales=kv_scales, kv_side=kv_side)
        assert res[0].tolist() == [len(p) for p in paths]
        assert [t[:len(p)] for t, p in zip(res[2].tolist(), paths)] == toks
        assert all(torch.equal(t, w) for t, w in zip(kept, want))
        self.calls["commit"] += 1
        return res


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 48])
@pytest.mark.parametrize("mode", [None, "token", "channel"])
def test_verify_steps_on_every_pool_gpu(monkeypatch, bs, mode):
    """Verification steps of a model on bf16 and both int8 pools, with and without the tensor-core form."""
    d = Decoder("cuda", PROMPTS, "tiny-moe-fp8", int8=mode == "token", bs=bs)
    if mode == "channel":
        a = d.args
        d.pool = KVPool(d.pool.num_blocks, a.num_hidden_layers, a.num_key_value_heads, bs, a.head_dim, d.model.dtype,
                        "cuda", int8=True, int8_mode="channel")
        d.pool.calibrate_begin()
        d.prefill()
        torch.cuda.synchronize()
        d.pool.calibrate_freeze(sum(len(p) - 1 for p in PROMPTS))
        # two dimensions of every head in the side values, whatever the calibration found
        d.pool.n_out.fill_(2)
        d.pool.out_idx[..., 0], d.pool.out_idx[..., 1] = 1, a.head_dim - 2
        for x in (1, a.head_dim - 2):
            d.pool.ch_dscale[..., x] = 0
    d.prefill()
    spy = Spy(monkeypatch, d.pool)
    g = torch.Generator().manual_seed(6)
    truth = [t + list(range(1, 99)) for t in d.seqs]
    for _ in range(2):
        d.verify(*d.drafts(truth, 4, g))
    assert spy.calls == {"attn": 2 * d.args.num_hidden_layers, "commit": 2}
    ops.check_status(d.pool.data.device)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_decode_and_tree_rows_in_one_step_gpu(monkeypatch, int8):
    """Decode rows in front of tree rows: the tree rows of q, the output and the tables start behind them."""
    d = Decoder("cuda", PROMPTS, "tiny-moe-fp8", int8=int8)
    d.prefill()
    spy = Spy(monkeypatch, d.pool)
    decode, decoded = ops.decode_attention, []

    def check_decode(q, layer, tables, lens, scale, out, split_len, nsplit, ws):
        got = decode(q, layer, tables, lens, scale, out, split_len, nsplit, ws)
        b = Spy.batch(torch.arange(q.shape[0] + 1), lens, tables, torch.full((q.shape[0],), -1))
        b.q, b.layer, b.scale, b.nq, b.nkv = q, layer, scale, q.shape[1], layer.num_kv_heads
        decoded.append((b, got.clone(), b.exact()))
        return got

    monkeypatch.setattr(ops, "decode_attention", check_decode)
    g = torch.Generator().manual_seed(3)
    trees = [_tree(n, "random", g) for n in (5, 8)]
    rows = [(s, len(d.seqs[s]) - 1, 1) for s in (0, 1)] + [(s + 2, len(d.seqs[s + 2]) - 1, len(p))
                                                           for s, p in enumerate(trees)]
    toks = [d.seqs[0][-1], d.seqs[1][-1]] + [d.seqs[2][-1], 5, 6, 7, 8] + [d.seqs[3][-1]] + list(range(11, 18))
    inp = d.inputs(rows, toks, [[-1], [-1]] + trees, num_decode=2)
    inp.tree_parents = inp.tree_parents[2:].contiguous()
    inp.prefill_cu = (inp.cu_seqlens_q[2:] - 2).contiguous()
    h = d.model(inp, d.pool)
    assert bool(torch.isfinite(h.float()).all())
    assert spy.calls["attn"] == len(decoded) == d.args.num_hidden_layers
    for b, got, (o, mass) in decoded:            # one query: the output and P rounded to bf16, as in Batch.check
        lim = HALF * o.abs() + (2 * HALF + 2 ** -13) * mass + 1e-30
        assert bool(((got.double().cpu() - o).abs() <= lim).all())
    ops.check_status(d.pool.data.device)
