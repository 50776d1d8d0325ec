"""The operators for several continuations of a request against their plain forms in 64 bits."""
import types

import numpy as np
import pytest
import torch

from plain import branch_plain as plain
from return_b200.ext import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def tree(kind, n, rs):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    return [-1] + [int(rs.randint(max(0, i - 5), i)) for i in range(1, n)]


def tree_batch(cached, parents, tokens=None):
    cu = np.concatenate([[0], np.cumsum([len(p) for p in parents])]).astype(np.int32)
    flat = [x for p in parents for x in p]
    return types.SimpleNamespace(host=types.SimpleNamespace(cu_q=cu, seg_pos0=np.asarray(cached, np.int32)), scratch={}, cu_q=ints(cu),
                                 seg_pos0=ints(cached), tree_parent=ints(flat), tokens=ints(tokens if tokens is not None else [0] * len(flat)))


def page_tables(rs, ends, page, width=None, spare=2):
    blocks = [(e + page - 1) // page for e in ends]
    order = rs.permutation(sum(blocks) + spare).tolist()
    tables, at = [], 0
    for b in blocks:
        tables.append(order[at:at + b])
        at += b
    width = width or max(blocks)
    return tables, ints([t + [-1] * (width - len(t)) for t in tables]), len(order)


class Attention:
    """A step of drafted trees: inputs on the device, and what it has to give."""

    def __init__(self, seed, dtype, heads, kv_heads, D, page, cached, nodes, kind="random", window=None, softcap=None, sink=False, pad=0, poison=True):
        rs, g = np.random.RandomState(seed), torch.Generator().manual_seed(seed)
        self.args = (heads, kv_heads, D, D ** -0.5)
        self.cached, self.parents = cached, [tree(kind, n, rs) for n in nodes]
        self.batch = tree_batch(cached, self.parents)
        ends = [c + n for c, n in zip(cached, nodes)]
        self.tables, self.block_table, pages = page_tables(rs, ends, page)
        self.page, self.window, self.softcap, T = page, window, softcap, sum(nodes)
        self.qkv = torch.randn((T, (heads + 2 * kv_heads) * D + pad), generator=g).to(dtype)
        self.k, self.v = (torch.randn((pages, kv_heads, page, D), generator=g).to(dtype) for _ in range(2))
        if poison:                      # what no node sees: rows behind a tree, pages of nobody
            held = torch.zeros((pages, page), dtype=torch.bool)
            for t, e in zip(self.tables, ends):
                for j in range(e):
                    held[t[j // page], j % page] = True
            for pool in (self.k, self.v):
                pool.permute(0, 2, 1, 3)[~held] = float("nan")
        self.sink = torch.randn((heads,), generator=g) * 2 if sink else None

    def want(self):
        heads, kv_heads, D, scale = self.args
        q = self.qkv[:, :heads * D].reshape(-1, heads, D)
        return plain.tree_attention(q, self.k, self.v, self.parents, self.cached, self.tables, self.page, kv_heads, scale, self.window, self.sink, self.softcap)

    def bound(self, out, size):
        """Per value.  Scores: a sum of D products in float32, and the scale's rounding; the cap is no steeper than 1 and adds a few units of
        its own value (|tanh| error of 2^-22 at most, times the cap).  Probabilities carry twice that, the sums over L keys a unit each;
        bfloat16 rounds the probabilities and the result by half a step each."""
        D, L = self.args[2], max(c + len(p) for c, p in zip(self.cached, self.parents))
        u = 2.0 ** -24
        score = (D + 4) * u * size + ((self.softcap or 0.0) * 2.0 ** -22)
        vmax = float(torch.nan_to_num(self.v.float(), nan=0.0, posinf=0.0, neginf=0.0).abs().max())
        b = (2 * score + (2 * L + 16) * u)[..., None] * vmax
        half = torch.finfo(self.qkv.dtype).eps / 2
        if self.qkv.dtype == torch.bfloat16:
            b = b + half * vmax + half * out.abs()
        return b

    def run(self, out=None):
        heads, kv_heads, D, scale = self.args
        qkv, k, v = (x.to(DEV) for x in (self.qkv, self.k, self.v))
        if out is None:
            out = torch.full((qkv.shape[0], heads * D), float("nan"), dtype=qkv.dtype, device=DEV)
        ops.tree_attention(qkv, k, v, self.batch, self.block_table, self.page, out, heads, kv_heads, D, scale, self.window,
                           self.sink.to(DEV) if self.sink is not None else None, self.softcap)
        return out

    def check(self, got):
        want, size = self.want()
        got = got.double().cpu().reshape(want.shape)
        assert torch.isfinite(got).all()
        off = (got - want).abs() - self.bound(want, size)
        assert off.max() <= 0, f"off by {(got - want).abs().max():.3e}, {off.max():.3e} beyond the bound"


SHAPES = [  # heads, kv heads, head size, page, cached, nodes, kind
    (4, 2, 128, 16, [0], [1], "random"),
    (4, 2, 128, 16, [1, 0, 63, 64, 65], [1, 7, 2, 64, 3], "random"),
    (16, 8, 128, 16, [500], [8], "random"),
    (32, 8, 128, 64, [130, 700], [16, 33], "random"),
    (64, 8, 128, 16, [300, 7], [40, 17], "random"),
    (5, 1, 64, 8, [129, 3, 1000], [31, 1, 12], "random"),
    (8, 8, 64, 16, [40], [130], "chain"),
    (2, 2, 128, 16, [250], [256], "random"),
    (3, 1, 128, 16, [90, 5], [129, 90], "star"),
    (6, 3, 48, 8, [77, 12], [9, 20], "random"),
    (4, 1, 256, 16, [33, 200], [5, 11], "random"),
    (2, 1, 16, 5, [31], [6], "chain"),
    (8, 2, 256, 16, [300, 64, 2], [70, 33, 8], "random"),
    (8, 2, 128, 32, [300, 64, 2], [20, 3, 8], "random"),
    (8, 2, 128, 128, [300, 64, 2], [12, 3, 8], "random"),
    (8, 2, 64, 24, [300, 64, 2], [12, 3, 40], "random"),
    (12, 2, 128, 16, [700, 1], [16, 5], "random"),
    (2, 1, 8, 4, [100], [9], "random"),
    (2, 1, 6, 4, [100], [9], "random"),
    (4, 2, 200, 16, [100], [30], "random"),
]


EITHER = [  # head sizes between the kernels' shapes
    (8, 2, 80, 16, [300, 64, 2], [40, 3, 8], "random"),
    (8, 2, 96, 24, [300, 64, 2], [12, 3, 70], "random"),
    (8, 2, 136, 16, [300, 64, 2], [40, 3, 8], "random"),
    (4, 1, 40, 64, [700], [100], "random"),
    (4, 1, 24, 12, [700, 9], [20, 9], "random"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_tree_attention(shape, dtype):
    a = Attention(3, dtype, *shape[:4], list(shape[4]), list(shape[5]), kind=shape[6])
    a.check(a.run())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("options", [dict(window=1), dict(window=3), dict(window=70), dict(window=5000), dict(softcap=2.0), dict(sink=True),
                                     dict(window=100, softcap=5.0, sink=True)], ids=str)
@pytest.mark.parametrize("D", [64, 128, 256, 32])
def test_tree_attention_options(D, options, dtype):
    a = Attention(5, dtype, 8, 2, D, 16, [200, 0, 65, 1500], [20, 9, 1, 40], kind="random", pad=16, **options)
    a.check(a.run())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,nodes", [(8, 8), (32, 40)])
@pytest.mark.parametrize("splits,share", [(2, 9), (5, 4), (17, 1), (64, 1)])
def test_tree_attention_shares(splits, share, heads, nodes, dtype, monkeypatch):
    """However the keys are shared out; shorter segments have fewer shares, one a single one."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    a = Attention(7, dtype, heads, 4, 128, 16, [1050, 3, 400, 64], [nodes, 2, 1, nodes - 3], sink=True)
    a.check(a.run())


@pytest.fixture(params=["tcgen05", "bfloat16"])
def kernel(request, monkeypatch):
    """One of the two kernels that a bfloat16 step may run on, whatever it costs."""
    monkeypatch.setitem(ops.TREE_COSTS, request.param, (0.0,) * 7)
    launch = ops._tree_launch

    def watched(*a):
        got = launch(*a)
        assert (got[0] > 0) == (request.param == "tcgen05" and a[7] == torch.bfloat16 and a[5] % 8 == 0)
        return got

    monkeypatch.setattr(ops, "_tree_launch", watched)


@pytest.mark.parametrize("shape", [x for x in SHAPES if x[2] % 8 == 0] + EITHER, ids=lambda s: "-".join(map(str, s[:4])))
def test_tree_attention_on_either_kernel(shape, kernel):
    a = Attention(3, torch.bfloat16, *shape[:4], list(shape[4]), list(shape[5]), kind=shape[6])
    a.check(a.run())


@pytest.mark.parametrize("options", [dict(window=3), dict(window=70), dict(softcap=2.0), dict(window=100, softcap=5.0, sink=True)], ids=str)
@pytest.mark.parametrize("splits,share", [(1, 0), (7, 4)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_attention_options_on_either_kernel(D, options, splits, share, kernel, monkeypatch):
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    a = Attention(5, torch.bfloat16, 8, 2, D, 16, [200, 0, 65, 1500], [20, 9, 1, 40], pad=16, **options)
    a.check(a.run())


@pytest.mark.parametrize("joined", [True, False])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float32, 128), (torch.float32, 6), (torch.bfloat16, 48)])
@pytest.mark.parametrize("splits,share", [(2, 9), (3, 6), (8, 3), (8, 2)])
def test_tree_attention_shares_joined_or_merged(splits, share, D, dtype, joined, kernel, monkeypatch):
    """Shares that join as clusters, or by a launch of their own; segments of one share, and of none in some clusters' CTAs."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    monkeypatch.setattr(ops, "tree_joins", lambda *a: joined)
    for heads, nodes in ((8, [8, 2, 1]), (16, [70, 3, 33])):
        a = Attention(23, dtype, heads, 2, D, 16, [1000, 3, 250], nodes, window=None if heads == 8 else 300, sink=heads == 8)
        a.check(a.run())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,D,nodes", [(1, 1, 5, [1]), (3, 1, 33, [5]), (3, 3, 7, [1, 3, 1]), (1, 1, 255, [3])])
@pytest.mark.parametrize("splits,share", [(3, 4), (11, 1), (5, 3)])
def test_tree_attention_odd_sizes_merged(splits, share, heads, kv_heads, D, nodes, dtype, monkeypatch):
    """An odd number of floats lies in front of the shares' maxima and sums."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    monkeypatch.setattr(ops, "tree_joins", lambda *a: False)
    a = Attention(37, dtype, heads, kv_heads, D, 16, [700, 3, 65][:len(nodes)], nodes)
    a.check(a.run())


def test_tree_attention_of_one_row_of_an_odd_size():
    a = Attention(41, torch.float32, 1, 1, 5, 16, [700], [1])
    a.check(a.run())


@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("splits,share", [(1, 0), (4, 5)])
@pytest.mark.parametrize("softcap", [None, 60.0])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_that_outrun_the_reference(D, softcap, splits, share, falling, kernel, monkeypatch):
    """Scores that grow along the keys to some 150 (or shrink from there): a row's maximum moves in many tiles, and by far."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    for heads, nodes in ((8, [8, 2, 1]), (16, [40, 3, 33])):
        a = Attention(29, torch.bfloat16, heads, 2, D, 16, [1200, 3, 250], nodes, softcap=softcap)
        for t, c in zip(a.tables, a.cached):
            for j in range(c):
                at = c - 1 - j if falling else j
                a.k[t[j // 16], :, j % 16] *= 1 + at / 32
        a.check(a.run())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads,D", [(4, 128), (16, 64), (4, 256), (4, 48), (8, 104)])
def test_what_a_node_does_not_see_does_not_reach_it_on_either_kernel(heads, D, value, kernel):
    test_what_a_node_does_not_see_does_not_reach_it(heads, D, value, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads,D", [(4, 128), (16, 64), (4, 48), (4, 256)])
def test_what_a_node_does_not_see_does_not_reach_it(heads, D, value, dtype):
    """One node's value (and, in another run, its key) is no number: only its descendants may show it."""
    for name in ("v", "k"):
        a = Attention(11, dtype, heads, 2, D, 16, [70, 10], [60, 5], window=50)
        clean = a.run()
        want, size = a.want()
        bad = 20
        slot = a.cached[0] + bad
        old = getattr(a, name)[a.tables[0][slot // 16], :, slot % 16].clone()
        getattr(a, name)[a.tables[0][slot // 16], :, slot % 16, 1 if name == "v" else slice(None)] = value
        # a cached key outside the later nodes' window, seen by the root alone
        first = a.cached[0] - 50 + 1
        getattr(a, name)[a.tables[0][first // 16], :, first % 16, 3 if name == "v" else slice(None)] = value
        got = a.run()
        sees = [bad in plain.line_of(a.parents[0], x) or x == 0 for x in range(60)] + [False] * 5
        assert 0 < sum(sees) < 40
        for t, hit in enumerate(sees):
            if hit:
                if name == "v":
                    assert not torch.isfinite(got[t].float()).all(), t
            else:
                assert torch.equal(got[t], clean[t]), t
        del old


@pytest.mark.parametrize("splits,share,joined", [(1, 0, False), (3, 8, True), (5, 4, False)])
@pytest.mark.parametrize("heads,D", [(4, 128), (8, 128), (16, 128), (4, 64), (8, 64), (4, 256), (8, 256), (8, 104), (4, 48)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_values_that_every_node_sees(heads, D, dtype, splits, share, joined, kernel, monkeypatch):
    """In tiles seen in full, of 16, 32 and 64 rows a tile and more: what the definition gives, and every other column as it was."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    monkeypatch.setattr(ops, "tree_joins", lambda *a: joined)
    inf = float("inf")
    for nodes, softcap in (([8, 2, 1], None), ([16, 3, 33], 30.0)):
        a = Attention(43, dtype, heads, 2, D, 16, [1200, 3, 250], nodes, softcap=softcap)
        for t, j, column, value in ((0, 100, 0, inf), (0, 127, 7, -inf), (0, 700, 33, inf), (0, 130, 33, inf), (0, 64, 40, inf), (0, 900, 40, -inf),
                                    (0, 0, D - 1, inf), (0, 511, 20, float("nan")), (2, 5, 2, inf), (2, 64, 3, -inf), (2, 200, 3, inf)):
            a.v[a.tables[t][j // 16], :, j % 16, column] = value
        want, size = a.want()
        got = a.run().double().cpu().reshape(want.shape)
        odd = ~torch.isfinite(want)
        assert odd[:, :, :].any(-1).all(-1).tolist() == [True] * nodes[0] + [False] * nodes[1] + [True] * nodes[2]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
        off = (got - want).abs() - a.bound(want, size)
        assert off[~odd].max() <= 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("D", [128, 48])
def test_blocks_that_are_gone_read_as_zeros(D, page, dtype):
    """A table's -1, and a page that the pool does not have."""
    a = Attention(17, dtype, 8, 2, D, page, [150, 20], [9, 3])
    for t, block in ((0, 1), (0, 4), (1, 0)):
        a.k[a.tables[t][block]] = a.v[a.tables[t][block]] = 0.0
    a.check(a.run())
    want = a.run()
    pages = a.k.shape[0]
    a.block_table[0, 1], a.block_table[0, 4], a.block_table[1, 0] = -1, pages, 2 ** 31 - 1
    assert torch.equal(a.run(), want)


def test_float32_values_near_the_end_of_the_type():
    """The products' parts are scaled up; values that the scale would take beyond the type are added by themselves."""
    a = Attention(19, torch.float32, 8, 2, 64, 16, [150, 20], [9, 3])
    held = torch.isfinite(a.v)
    for exponent in (100, 103, 104, 105, 111, 118):
        a.v[held] = torch.sign(a.v[held]) * 2.0 ** exponent
        a.check(a.run())


def test_tree_attention_takes_what_the_documentation_allows():
    """Another stream, an output that other rows surround, two calls on one step's tables at once, a captured and replayed call."""
    a = Attention(13, torch.bfloat16, 8, 2, 128, 16, [900, 30], [12, 5])
    want = a.run()
    wide = torch.full((19, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    a.run(wide[1:18])
    assert torch.equal(wide[1:18], want) and (wide[0] == 7).all() and (wide[18] == 7).all()
    heads, kv_heads, D, scale = a.args
    qkv, k, v = (x.to(DEV) for x in (a.qkv, a.k, a.v))
    call = lambda out: ops.tree_attention(qkv, k, v, a.batch, a.block_table, 16, out, heads, kv_heads, D, scale)  # noqa: E731
    outs = [torch.empty_like(want) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                call(o)
    torch.cuda.synchronize()
    graphs = []
    for o in outs[2:]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(o)
        graphs.append(graph)
    for o in outs[2:]:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    ops.check_status(torch.device(DEV))


@pytest.mark.parametrize("splits,share", [(2, 8), (5, 3), (8, 2)])
def test_joined_shares_on_two_streams_and_in_graphs(splits, share, kernel, monkeypatch):
    """Clusters of two calls, and of two captured graphs, side by side on the device."""
    monkeypatch.setattr(ops, "tree_shares", lambda *a: (splits, share))
    monkeypatch.setattr(ops, "tree_joins", lambda *a: True)
    a = Attention(31, torch.bfloat16, 16, 4, 128, 16, [1000, 30, 700, 500, 900, 1000], [8, 5, 1, 8, 8, 8])
    want = a.run()
    a.check(want)
    heads, kv_heads, D, scale = a.args
    qkv, k, v = (x.to(DEV) for x in (a.qkv, a.k, a.v))
    call = lambda out: ops.tree_attention(qkv, k, v, a.batch, a.block_table, 16, out, heads, kv_heads, D, scale)  # noqa: E731
    outs = [torch.empty_like(want) for _ in range(4)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for o in outs[2:]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(o)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(30):
        for s, o, graph in zip(streams, outs, graphs):
            with torch.cuda.stream(s):
                call(o)
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    ops.check_status(torch.device(DEV))


# ---------------------------------------------------------------------------------------- commit

def commit_case(seed, layers, heads, D, page, cached, nodes, dtype, latent=False, twice=False):
    rs, g = np.random.RandomState(seed), torch.Generator().manual_seed(seed)
    parents = [tree("random", n, rs) for n in nodes]
    # few different tokens, so that paths go on; with `twice` siblings may name the same one
    tokens = [[int(x) for x in rs.randint(0, 2 if twice else 4, n)] for n in nodes]
    sampled = [[int(x) for x in rs.randint(0, 2 if twice else 4, n)] for n in nodes]
    tables, block_table, pages = page_tables(rs, [c + n for c, n in zip(cached, nodes)], page)
    shape = (layers, pages, page, D) if latent else (layers, 2, pages, heads, page, D)
    pool = torch.randn(shape, generator=g).to(dtype)
    return parents, tokens, sampled, tables, block_table, pool


@pytest.mark.parametrize("case", [
    (2, 2, 128, 16, [40], [8], torch.bfloat16, False, False),
    (3, 4, 64, 8, [0, 7, 100, 15], [1, 20, 33, 9], torch.bfloat16, False, True),
    (5, 1, 48, 16, [3] * 9, [30] * 9, torch.float32, False, True),
    (2, 3, 33, 5, [11, 2], [17, 200], torch.bfloat16, False, True),
    (4, 1, 160, 16, [5, 31], [12, 64], torch.bfloat16, True, False),
    (1, 1, 16, 16, [0], [256], torch.float32, False, True),
], ids=str)
def test_tree_commit(case):
    for seed in range(6):
        layers, heads, D, page, cached, nodes, dtype, latent, twice = case
        parents, tokens, sampled, tables, block_table, pool = commit_case(seed, *case)
        paths = [plain.walk(t, p, s) for t, p, s in zip(tokens, parents, sampled)]
        flat = lambda lists: [x for one in lists for x in one]  # noqa: E731
        batch = tree_batch(cached, parents, flat(tokens))
        n, width = len(nodes), max(nodes) + 2
        path, emitted = (torch.full((n, width), 99, dtype=torch.int32, device=DEV) for _ in range(2))
        count = torch.full((n,), 99, dtype=torch.int32, device=DEV)
        here = pool.to(DEV)
        ops.tree_commit(ints(flat(sampled)), batch, [(here, block_table)], path, count, emitted)
        assert count.tolist() == [len(p) for p in paths]
        assert path.tolist() == [p + [-1] * (width - len(p)) for p in paths]
        assert emitted.tolist() == [[s[x] for x in p] + [-1] * (width - len(p)) for p, s in zip(paths, sampled)]
        assert torch.equal(here.cpu(), plain.commit(pool, tables, cached, paths, page))


def test_tree_commit_several_groups_and_gone_pages():
    parents, tokens, sampled = [[-1, 0, 0, 2, 3]], [[9, 1, 2, 3, 4]], [[2, 0, 3, 4, 8]]
    batch = tree_batch([14], parents, tokens[0])
    pools = [torch.randn((2, 2, 3, 1, 16, 32)).to(torch.bfloat16), torch.randn((3, 5, 8, 24)).to(torch.float32)]
    tables = [[2, 0], [4, -1, 1]]                       # slots 8 to 15 of the second group are gone
    here = [p.to(DEV) for p in pools]
    path, emitted = (torch.empty((1, 5), dtype=torch.int32, device=DEV) for _ in range(2))
    count = torch.empty((1,), dtype=torch.int32, device=DEV)
    ops.tree_commit(ints(sampled[0]), batch, [(h, ints([t])) for h, t in zip(here, tables)], path, count, emitted)
    assert path.tolist() == [[0, 2, 3, 4, -1]] and emitted.tolist() == [[2, 3, 4, 8, -1]] and count.tolist() == [4]
    for h, p, t, page in zip(here, pools, tables, (16, 8)):
        assert torch.equal(h.cpu(), plain.commit(p, [t], [14], [[0, 2, 3, 4]], page))
    path.zero_()
    ops.tree_commit(ints(sampled[0]), batch, [], path, count, emitted)          # the walk alone
    assert path.tolist() == [[0, 2, 3, 4, -1]]


# ---------------------------------------------------------------------------------------- copies

@pytest.mark.parametrize("shape,dtype", [((3, 2, 9, 2, 16, 64), torch.bfloat16), ((2, 2, 9, 1, 5, 33), torch.bfloat16),
                                         ((2, 9, 16, 72), torch.float32), ((1, 2, 9, 8, 64, 128), torch.bfloat16)])
def test_copy_pages(shape, dtype):
    pool = torch.randn(shape).to(dtype)
    pool.view(-1)[::7] = float("nan")
    src, dst, rows = [0, 0, 3, -1, 5], [1, 2, 4, 6, -1], [1, 100, 3, 2, 2]
    here = pool.to(DEV)
    ops.copy_pages(here, ints(src), ints(dst), ints(rows))
    want = plain.copy_pages(pool, src, dst, rows)
    assert torch.equal(here.cpu().view(torch.int16 if dtype == torch.bfloat16 else torch.int32),
                       want.view(torch.int16 if dtype == torch.bfloat16 else torch.int32))
    ops.copy_pages(here, ints([]), ints([]), ints([]))
    ops.copy_pages(here, ints([9, 0]), ints([0, 9]), ints([1, 1]))             # pages that the pool does not have
    ops.copy_pages(here, ints([0]), ints([3]), ints([0]))
    assert torch.equal(here.cpu().view(torch.int16 if dtype == torch.bfloat16 else torch.int32),
                       want.view(torch.int16 if dtype == torch.bfloat16 else torch.int32))


def test_copy_slots():
    states = [torch.randn(7, 300, device=DEV), torch.randint(0, 99, (7, 1), dtype=torch.int32, device=DEV), torch.randn(7, 3, 20001, device=DEV),
              torch.randn(7, 5, device=DEV).to(torch.bfloat16), torch.randint(0, 255, (7, 3), dtype=torch.uint8, device=DEV)]
    states += [torch.randn(7, 4, device=DEV) for _ in range(70)]               # more than one launch takes
    want = [t.clone() for t in states]
    for t in want:
        for a, b in ((2, 0), (2, 6), (5, 3)):
            t[b] = t[a]
    table = ops.slot_table(states)
    ops.copy_slots(table, ints([2, 2, 5, 7, -1]), ints([0, 6, 3, 1, 1]))
    for a, b in zip(states, want):
        assert torch.equal(a, b)
    ops.copy_slots(table, ints([]), ints([]))


# ---------------------------------------------------------------------------------------- beams

def beams_run(logits, scores, beams, keep):
    requests = logits.shape[0] // beams
    out = torch.empty((requests, keep), device=DEV)
    b, t = (torch.empty((requests, keep), dtype=torch.int32, device=DEV) for _ in range(2))
    ops.beam_select(logits, scores, beams, out, b, t)
    return out.cpu(), b.cpu(), t.cpu()


def beams_check(logits, scores, beams, keep):
    """Places have to be equal; totals are off by the rounding at the store, by the float32 sum of exponentials (each off by
    2^-21 relative at most: two units of the hardware's 2^x and its argument's rounding where the term counts) and of the chunk."""
    out, b, t = beams_run(logits.to(DEV) if not logits.is_cuda else logits, scores.to(DEV), beams, keep)
    want = plain.beam_select(logits.cpu(), scores.cpu(), beams, keep)
    for r, row in enumerate(want):
        assert list(zip(b[r].tolist(), t[r].tolist())) == [(x[1], x[2]) for x in row]
        for got, (total, _, _) in zip(out[r].tolist(), row):
            assert got == total or abs(got - total) <= 2.0 ** -24 * abs(total) + 2.0 ** -19


@pytest.mark.parametrize("requests,beams,V,keep", [(1, 1, 1, 1), (1, 4, 32768, 8), (2, 3, 1000, 6), (3, 8, 151936, 16), (1, 2, 5, 10), (40, 5, 8193, 11),
                                                   (1, 64, 700, 128), (20, 8, 32771, 1), (1, 1, 100000, 128), (16, 8, 8960, 16), (1, 2, 2300, 4)])
def test_beam_select(requests, beams, V, keep):
    g = torch.Generator().manual_seed(V + keep)
    logits = torch.randn((requests * beams, V), generator=g) * 3
    beams_check(logits, -30 * torch.rand((requests * beams,), generator=g), beams, keep)


@pytest.mark.parametrize("V", [50, 2048, 40000])
def test_beam_select_ties_and_masked_words(V):
    g = torch.Generator().manual_seed(V)
    same = torch.zeros((6, V))
    beams_check(same, torch.zeros(6), 3, 7)                                     # everything is equal: the first beam's first words
    beams_check(same, torch.tensor([-1.0, 0.0, 0.0, -1.0, -1.0, -1.0]), 3, 7)
    grid = torch.round(torch.randn((6, V), generator=g))
    beams_check(grid, torch.zeros(6), 3, 20)
    beams_check(grid.repeat(1, 1)[[0, 0, 1, 2, 2, 2]], torch.zeros(6), 3, 20)   # beams alike
    signed = torch.where(torch.rand((2, V), generator=g) < 0.5, -0.0, 0.0)
    beams_check(signed, torch.zeros(2), 2, 9)                                   # -0 is 0
    masked = torch.full((4, V), float("-inf"))
    masked[:, [3, 9, V - 1]] = torch.randn((4, 3), generator=g)
    beams_check(masked, -torch.rand(4, generator=g), 2, 12)                     # fewer words than are asked for
    masked[1] = float("-inf")
    beams_check(masked, -torch.rand(4, generator=g), 2, 12)
    beams_check(masked, -torch.rand(4, generator=g), 4, 2)


@pytest.mark.parametrize("V", [60, 9000])
def test_beam_select_dead_beams_and_numbers_that_are_none(V):
    g = torch.Generator().manual_seed(V)
    logits = torch.randn((8, V), generator=g)
    scores = -torch.rand(8, generator=g)
    beams_check(logits, torch.where(torch.arange(8) % 4 == 0, scores, float("-inf")), 4, 8)
    beams_check(logits, torch.full((8,), float("-inf")), 4, 8)
    beams_check(logits, torch.where(torch.arange(8) == 2, float("nan"), scores), 4, 8)
    for value in (float("nan"), float("inf")):
        bad = logits.clone()
        bad[1, V // 2] = bad[5, 0] = value
        beams_check(bad, scores, 4, 8)
        beams_check(bad[:2], scores[:2], 2, 8)


def test_beam_select_strides_streams_and_graphs():
    g = torch.Generator().manual_seed(1)
    wide = (torch.randn((6, 5003), generator=g)).to(DEV)
    scores = -torch.rand(6, generator=g)
    beams_check(wide[:, 2:5001], scores, 3, 6)                                  # rows that begin anywhere
    beams_check(wide[:, 1:2], scores, 3, 3)
    beams_check(torch.full((1, 7000), 1.0, device=DEV).expand(6, 7000), scores, 3, 6)        # all rows the same memory
    x, s = wide[:, :5000].contiguous(), scores.to(DEV)
    want = beams_run(x, s, 3, 6)
    outs = [(torch.empty((2, 6), device=DEV), *(torch.empty((2, 6), dtype=torch.int32, device=DEV) for _ in range(2))) for _ in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.beam_select(x, s, 3, *o)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(o, want))


@pytest.mark.parametrize("rows,V,keep", [(296, 4096, 64), (592, 1000, 5), (40, 40000, 128)])
def test_beam_select_gives_the_same_every_time(rows, V, keep):
    """A first tile's selection counts what all threads collected: late warps and early ones see one count, run after run."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn((rows, V), generator=g)
    x[::2] = torch.round(x[::2] * 2)                                            # some rows of many equal values
    s = -torch.rand(rows, generator=g)
    beams_check(x, s, 4, keep)
    x, s = x.to(DEV), s.to(DEV)
    want = beams_run(x, s, 4, keep)
    for _ in range(200):
        assert all(torch.equal(a, b) for a, b in zip(beams_run(x, s, 4, keep), want))


@pytest.mark.parametrize("rows,V,keep", [(600, 2048, 100), (600, 2500, 128), (600, 5000, 7), (600, 3001, 64), (300, 16388, 128), (300, 24576, 128), (300, 40000, 3)])
def test_beam_select_walks_rising_rows_twice(rows, V, keep):
    """Rows that rise overflow what is collected and are walked again; nothing of the first walk's tiles may reach the second's."""
    x = torch.linspace(-30, 0, V).expand(rows, V) + torch.linspace(0, 5, rows)[:, None]
    s = torch.zeros(rows)
    beams_check(x, s, 1, keep)
    x, s = x.to(DEV), s.to(DEV)
    want = beams_run(x, s, 1, keep)
    for _ in range(50):
        assert all(torch.equal(a, b) for a, b in zip(beams_run(x, s, 1, keep), want))


LOWEST = [torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -1e38, -1e30, -1e20, -1e10, -65504.0]


def masked_rows(rows, V, value, seed):
    """Most words masked, in long runs and one by one, and whole rows of the mask."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, V), generator=g) * 3
    x[torch.rand((rows, V), generator=g) < 0.5] = value
    x[:, V // 5:V - V // 5] = value
    x[3] = value
    return x, -torch.rand(rows, generator=g)


def shifted_rows(rows, V, shift):
    g = torch.Generator().manual_seed(V)
    return torch.randn((rows, V), generator=g) * 3 + shift, -30 * torch.rand(rows, generator=g)


def certain_rows(rows, V, top):
    """One word takes nearly everything."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn((rows, V), generator=g)
    x[torch.arange(rows), torch.randint(0, V, (rows,), generator=g)] = top + torch.rand(rows, generator=g)
    return x, -torch.rand(rows, generator=g)


@pytest.mark.parametrize("value", LOWEST, ids=str)
@pytest.mark.parametrize("V", [100, 2048, 40000, 151936])
def test_beam_select_masks_of_finite_values(V, value):
    x, s = masked_rows(6, V, value, V)
    beams_check(x, s, 3, 7)
    beams_check(x[3:4], s[3:4], 1, 20)                                          # nothing but the mask


@pytest.mark.parametrize("shift", [100.0, -100.0, 1000.0, -1000.0, 10000.0, -10000.0])
@pytest.mark.parametrize("V", [1000, 32771, 151936])
def test_beam_select_of_shifted_rows(V, shift):
    """A constant added to a row changes nothing, but for what it rounds off the logits."""
    x, s = shifted_rows(8, V, shift)
    beams_check(x, s, 4, 8)


@pytest.mark.parametrize("top", [20.0, 40.0, 57.0, 100.0, 1003.0, 10007.0, 1e30])
@pytest.mark.parametrize("V", [1000, 40000])
def test_beam_select_of_words_that_are_certain(V, top):
    x, s = certain_rows(6, V, top)
    beams_check(x, s, 3, 3)


@pytest.mark.parametrize("value", LOWEST, ids=str)
@pytest.mark.parametrize("V", [100, 9000, 151936])
def test_beam_select_of_fewer_words_than_are_asked_for(V, value):
    """Masked words of finite value fill the places behind the others: the lowest ones of the beam that is ahead, or of the first where none is."""
    g = torch.Generator().manual_seed(V)
    x = torch.full((6, V), value)
    for b in range(6):
        x[b, torch.randint(0, V, (2,), generator=g)] = torch.randn(2, generator=g)
    beams_check(x, -torch.rand(6, generator=g), 3, 16)
