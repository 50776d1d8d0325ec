"""Refusals of the operators for several continuations of a request, and what they work out on the host.  No GPU."""
import types

import numpy as np
import pytest
import torch

from return_b200.ext import ops


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def tree_batch(cached, nodes):
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    T = int(cu[-1])
    return types.SimpleNamespace(host=types.SimpleNamespace(cu_q=cu, seg_pos0=np.asarray(cached, np.int32)), scratch={},
                                 cu_q=torch.from_numpy(cu.copy()), seg_pos0=ints(*cached), tokens=torch.zeros(T, dtype=torch.int32),
                                 tree_parent=torch.full((T,), -1, dtype=torch.int32))


def attention_args(**changes):
    a = dict(cached=[5, 20], nodes=[3, 1], heads=4, kv_heads=2, head_dim=16, page=8, dtype=torch.bfloat16)
    a.update(changes)
    T, D = sum(a["nodes"]), a["head_dim"]
    pool = torch.zeros((6, a["kv_heads"], a["page"], D), dtype=a["dtype"])
    return dict(qkv=torch.zeros((T, (a["heads"] + 2 * a["kv_heads"]) * D), dtype=a["dtype"]), k_pool=pool, v_pool=pool.clone(),
                batch=tree_batch(a["cached"], a["nodes"]), block_table=torch.zeros((len(a["nodes"]), 3), dtype=torch.int32), page_size=a["page"],
                out=torch.zeros((T, a["heads"] * D), dtype=a["dtype"]), num_heads=a["heads"], num_kv_heads=a["kv_heads"], head_dim=D, scale=0.25)


def refuse(match, call, *args, **kwargs):
    with pytest.raises(ops.KernelError, match=match):
        call(*args, **kwargs)


def test_tree_attention_refuses():
    good = attention_args()
    refuse("CPU tensor", ops.tree_attention, **good)
    refuse("kernels take 256", ops.tree_attention, **attention_args(nodes=[3, 257], cached=[0, 0]))
    refuse("at least one node", ops.tree_attention, **attention_args(nodes=[3, 0]))
    refuse("block table holds", ops.tree_attention, **attention_args(cached=[5, 24]))
    refuse("block table holds", ops.tree_attention, **attention_args(cached=[-1, 3]))
    refuse("multiple of the kv heads", ops.tree_attention, **attention_args(heads=3))
    refuse("up to 256", ops.tree_attention, **attention_args(head_dim=272))
    for change, match in ((dict(qkv=good["qkv"][:3]), "row per node"), (dict(qkv=good["qkv"][:, :63]), "row per node"),
                          (dict(v_pool=good["v_pool"].float()), "one type"), (dict(v_pool=good["v_pool"][:5]), "pools"),
                          (dict(k_pool=good["k_pool"].transpose(1, 2)), "pools"), (dict(out=good["out"].float()), "one type"),
                          (dict(out=torch.zeros((4, 128), dtype=torch.bfloat16)[:, ::2]), "out"),
                          (dict(block_table=good["block_table"].long()), "block_table"), (dict(window=-1), "window"), (dict(softcap=-1.0), "softcap"), (dict(scale=0.0), "scale")):
        refuse(match, ops.tree_attention, **{**attention_args(), **change})
    bad = attention_args()
    bad["batch"].tree_parent = bad["batch"].tree_parent.long()
    refuse("tree_parent", ops.tree_attention, **bad)


def test_tree_commit_refuses():
    def args(n=2, width=3):
        b = tree_batch([5, 20], [3, 1])
        pool = torch.zeros((2, 2, 6, 2, 8, 16), dtype=torch.bfloat16)
        return dict(sampled=ints(0, 0, 0, 0), batch=b, caches=[(pool, torch.zeros((2, 3), dtype=torch.int32))],
                    path=torch.zeros((n, width), dtype=torch.int32), count=torch.zeros(n, dtype=torch.int32),
                    emitted=torch.zeros((n, width), dtype=torch.int32))
    refuse("CPU tensor", ops.tree_commit, **args())
    refuse("CPU tensor", ops.tree_commit, **{**args(), "caches": []})
    refuse("3 columns", ops.tree_commit, **args(width=2))
    refuse("path", ops.tree_commit, **args(n=3))
    refuse("sampled", ops.tree_commit, **{**args(), "sampled": ints(0, 0, 0)})
    refuse("count", ops.tree_commit, **{**args(), "count": torch.zeros(2)})
    pool, table = args()["caches"][0]
    refuse("a pool", ops.tree_commit, **{**args(), "caches": [(pool[0], table)]})
    refuse("a pool", ops.tree_commit, **{**args(), "caches": [(pool.transpose(3, 4), table)]})
    refuse("a pool", ops.tree_commit, **{**args(), "caches": [(pool.to(torch.uint8), table)]})
    refuse("block table holds", ops.tree_commit, **{**args(), "caches": [(pool, table[:, :2])]})
    refuse("block_table", ops.tree_commit, **{**args(), "caches": [(pool, table.long())]})


def test_copies_refuse():
    pool = torch.zeros((2, 2, 6, 2, 8, 16), dtype=torch.bfloat16)
    refuse("CPU tensor", ops.copy_pages, pool, ints(0), ints(1), ints(3))
    refuse("dst", ops.copy_pages, pool, ints(0), ints(1, 2), ints(3))
    refuse("rows", ops.copy_pages, pool, ints(0), ints(1), ints(3).long())
    refuse("a pool", ops.copy_pages, pool[:, :, ::2], ints(0), ints(1), ints(3))
    refuse("at least one", ops.slot_table, [])
    refuse("CUDA device", ops.slot_table, [torch.zeros(3, 4)])


def test_beam_select_refuses():
    def args(rows=6, V=10, requests=2, keep=4, beams=3):
        return dict(logits=torch.zeros((rows, V)), scores=torch.zeros(rows), beams=beams, scores_out=torch.zeros((requests, keep)),
                    beams_out=torch.zeros((requests, keep), dtype=torch.int32), tokens_out=torch.zeros((requests, keep), dtype=torch.int32))
    refuse("CPU tensor", ops.beam_select, **args())
    refuse("request and beam", ops.beam_select, **args(rows=5))
    refuse("request and beam", ops.beam_select, **args(rows=130, beams=65))
    refuse("request and beam", ops.beam_select, **args(rows=0, requests=2, beams=0))
    refuse("continuations", ops.beam_select, **args(keep=31))
    refuse("continuations", ops.beam_select, **args(keep=0))
    refuse("continuations", ops.beam_select, **args(keep=129, V=1000))
    refuse("logits", ops.beam_select, **{**args(), "logits": torch.zeros((6, 20))[:, ::2]})
    refuse("logits", ops.beam_select, **{**args(), "logits": torch.zeros((6, 10), dtype=torch.bfloat16)})
    refuse("scores", ops.beam_select, **{**args(), "scores": torch.zeros(5)})
    refuse("tokens_out", ops.beam_select, **{**args(), "tokens_out": torch.zeros((2, 4))})
    refuse("65,535", ops.beam_select, **{**args(rows=65538, requests=21846, V=1, keep=1)})


def test_beam_select_refuses_rows_that_its_counters_do_not_hold():
    for rows, V, beams in ((1, 2 ** 29 + 1, 1), (1, 2 ** 31 - 2, 1), (4, 2 ** 29, 4)):
        out = torch.zeros((rows // beams, 1))
        refuse("29 words", ops.beam_select, torch.zeros((1, 1)).expand(rows, V), torch.zeros(rows), beams, out, out.int(), out.int())


def test_limits_of_a_library_are_those_of_the_checks():
    lib = types.SimpleNamespace(rb_a=lambda: 3, rb_b=lambda: 4)
    ops._same_limits(lib, rb_a=3, rb_b=4)
    refuse("rb_b: 4 in the compiled library, 5 here", ops._same_limits, lib, rb_a=3, rb_b=5)


@pytest.mark.parametrize("kind", sorted(ops.TREE_COSTS))
def test_tree_shares_cover_the_keys(monkeypatch, kind):
    """Every share is within the launch's splits, and the shares cover the longest walk; a full launch of long CTAs, and a short one, are not split."""
    monkeypatch.setattr(ops, "num_sms", lambda: 148)
    for nodes, cached, window, split in (([8], [500], 0, None), ([16] * 8, [2040] * 8, 0, True), ([64] * 32, [250 * i for i in range(32)], 0, None),
                                         ([5, 1], [9000, 3], 700, True), ([1], [0], 0, False), ([256], [130000], 0, True), ([8] * 64, [2000] * 64, 0, False if kind == "tcgen05" else None)):
        ends = [c + k for c, k in zip(cached, nodes)]
        splits, share = ops.tree_shares(nodes, ends, window, 4, 8, sum(nodes) * 32, 128, 128, 1, kind)
        tiles = [(e - 1) // 64 - (max(0, e - k - window + 1) if window else 0) // 64 + 1 for e, k in zip(ends, nodes)]
        assert 1 <= splits <= ops.TREE_MAX_SPLITS and split in (None, splits > 1)
        if splits == 1:
            assert share == 0
        else:
            assert share >= 1 and splits * share >= max(tiles) > (splits - 1) * share


def test_scratch_of_shares_that_a_launch_merges():
    """Odd head sizes, heads, nodes and splits: pairs begin where eight bytes can be moved, behind all outputs, and fit."""
    for splits in range(2, ops.TREE_MAX_SPLITS + 1):
        for rows in (1, 2, 3, 7, 35):
            for head_dim in (1, 3, 5, 6, 33, 128, 255):
                floats, pairs = ops.tree_scratch(splits, rows, head_dim)
                assert pairs % 4 == 0 and splits * rows * head_dim <= pairs < splits * rows * head_dim + 4 and floats == pairs + 2 * splits * rows


# ---------------------------------------------------------------------------------------- drafted trees on the host

def test_batch_of_drafted_trees():
    from return_b200.cache.manager import CacheManager, GroupSpec
    from return_b200.engine.batch import StepEntry, build_host_batch
    from return_b200.parts.base import Tiling
    m = CacheManager([GroupSpec("full", 4, 20)], max_requests=3)
    for rid, cached in (("a", 5), ("b", 2)):
        m.add(rid)
        m.append(rid, cached)
    entries = [StepEntry("a", [7, 8, 9, 8], [0, 3], m.append("a", 4), [-1, 0, 0, 2]), StepEntry("b", [6], [0], m.append("b", 1))]
    b = build_host_batch(entries, m, 100, 50, {"x": Tiling(2)})
    assert b.tree_parent.tolist() == [-1, 0, 0, 2, -1] and b.slots.tolist() == [5, 6, 7, 8, 2]
    assert b.pos.tolist() == [5, 6, 6, 7, 2] and b.tiles["x"].shape == (0, 2) and b.num_multi == 0
    assert b.seg_pos0.tolist() == [5, 2] and b.seg_kv_len.tolist() == [9, 3] and b.want_rows.tolist() == [0, 3, 4]
    for parents in ([-1, 0, 3, 0], [0, 0, 0, 0], [-1, 0, -1, 0], [-1, 1, 0, 0], [-1, 0, 0], None):
        entries[0].parents = parents
        if parents is None:             # a prompt's portion is no tree, and no tree step has one
            entries[1].parents = [-1]
        with pytest.raises(ValueError, match="parent"):
            build_host_batch(entries, m)
    entries[0].parents = entries[1].parents = None
    plain = build_host_batch(entries, m)
    assert plain.tree_parent is None and plain.slots is None and plain.pos.tolist() == [5, 6, 7, 8, 2]
    alone = [StepEntry("b", [1], [0], m.append("b", 1), [-1])]
    assert build_host_batch(alone, m).tree_parent is None                       # single tokens: an ordinary decode step


def test_forked_requests_share_full_pages():
    from return_b200.cache.manager import CacheManager, GroupSpec, KVCapacityError
    m = CacheManager([GroupSpec("full", 4, 9), GroupSpec("win", 4, 12, window=6)], max_requests=4)
    m.add("a")
    m.append("a", 10)
    m.append("a", 1)
    fork = m.fork_all([("a", "b"), ("a", "c")])
    m.check()
    full = m.block_table("a", 0)
    assert m.length("b") == m.length("c") == 11 and m.block_table("b", 0)[:2] == full[:2] and m.block_table("b", 0)[2] != full[2]
    assert fork[0].src_slot == m.slot("a") and fork[0].dst_slot == m.slot("b") != m.slot("c")
    assert [x[::3] for x in fork[1].pages] == [(0, 3), (1, 3)] and fork[1].pages[0][1:3] == (full[2], m.block_table("c", 0)[2])
    assert m.block_table("b", 1)[0] == m.block_table("a", 1)[0] == -1           # what the window has passed
    assert m.pages_used()[0] == 5 and m.pools[0].holders(full[0]) == 3
    for rid in "abc":
        m.append(rid, 5)
        m.check()
    assert m.pages_used()[0] == 8
    with pytest.raises(KVCapacityError):                                        # three copies, one free page
        m.append("a", 1), m.append("b", 1)
        m.fork_all([("a", "d")])
    m.check()
    m.free("a")
    m.check()
    assert m.pools[0].holders(full[0]) == 2
    m.free("b"), m.free("c")
    assert m.pages_used() == [0, 0]
    m.check()


def test_forks_refuse():
    from return_b200.cache.manager import CacheManager, GroupSpec, KVCapacityError
    m = CacheManager([GroupSpec("full", 4, 4)], max_requests=3)
    m.add("a")
    m.append("a", 9)
    before = (m.pages_used(), m.free_slots)
    for pairs, error in (([("a", "a")], KeyError), ([("a", "b"), ("a", "b")], KeyError), ([("x", "b")], KeyError),
                         ([("a", "b"), ("a", "c")], KVCapacityError), ([("a", "b")] * 0 + [("a", "b"), ("a", "c"), ("a", "d")], KVCapacityError)):
        with pytest.raises(error):
            m.fork_all(pairs)
        assert (m.pages_used(), m.free_slots) == before
        m.check()
    m.fork_all([("a", "b")])
    m.truncate("a", 8)
    with pytest.raises(ValueError, match="shares the page"):                    # position 6 lies in a page that b holds too
        m.truncate("a", 6)
    m.free("b")
    m.truncate("a", 6)
    m.check()


def test_pages_that_another_holds_do_not_come_back():
    from return_b200.cache.manager import CacheManager, GroupSpec
    m = CacheManager([GroupSpec("win", 4, 6, window=4)], max_requests=2)
    m.add("a")
    m.append("a", 8)
    m.fork_all([("a", "b")])
    m.append("a", 4)                                                            # passes block 0, which b still holds
    assert m.pages_needed("b", 4) == [0] and m.pools[0].num_free == 3
    m.append("b", 4)
    m.check()
    assert m.pools[0].num_free == 3


def test_prompt_lookup():
    from return_b200.engine.draft import PromptLookup
    from return_b200.engine.request import Request
    d = PromptLookup(6, longest=3, shortest=2, places=2)
    r = Request("x", [1, 2, 3, 4, 9, 1, 2, 3, 5, 9, 7, 1, 2, 3])
    tokens, parents = d.propose(r, 100)
    assert tokens[0] == 3 and parents[0] == -1 and len(tokens) <= 7
    # the latest place first: 5 9 7 ..., then 4 9 1 ... as a second branch where there is room
    assert tokens[1:4] == [5, 9, 7] and parents[1:4] == [0, 1, 2]
    wide = PromptLookup(9, longest=3, shortest=2, places=2).propose(Request("y", r.prompt_ids), 3)
    assert wide == ([3, 5, 9, 7], [-1, 0, 1, 2])
    tokens, parents = PromptLookup(20, longest=3, shortest=2, places=2).propose(Request("z", r.prompt_ids), 100)
    branch = [t for t, p in zip(tokens, parents) if p == 0]
    assert branch == [5, 4] and len(set(zip(parents, tokens))) == len(tokens)
    r.push(4)
    assert d.propose(r, 100)[0][:3] == [4, 9, 1]                                # 2 3 4 stood once before: 9 1 2 ...
    r.push(77)
    assert d.propose(r, 100) == ([77], [-1]) and d.propose(r, 0) == ([77], [-1])
    assert PromptLookup(4).propose(Request("w", [5]), 9) == ([5], [-1])
    again = Request("v", list(r.prompt_ids) + r.output)
    assert d.propose(again, 5) == d.propose(r, 5)
    with pytest.raises(ValueError):
        PromptLookup(4, longest=1, shortest=2)


def test_draft_settings_refuse():
    from return_b200.engine.config import EngineConfig
    for bad in (-1, ops.TREE_MAX_NODES):
        with pytest.raises(ValueError, match="draft_tokens"):
            EngineConfig(draft_tokens=bad)


@pytest.mark.parametrize("chunk,lengths", [(1, [1, 1]), (1, [3, 1, 2]), (2, [1, 1, 1, 1, 1]), (4, [5, 1, 1, 6])])
def test_prompts_of_a_beam_search_keep_their_logits(chunk, lengths):
    """A step of single tokens hands out the captured graph's own logits, which the next one writes over."""
    from return_b200.engine.beams import BeamSearch

    class Runner:
        vocab_size, max_positions = 7, 100
        config = types.SimpleNamespace(max_reside=8, prefill_chunk=chunk)
        static = torch.zeros((8, 7))

        def add_request(self, rid):
            pass

        def reserve(self, rid, tokens, want):
            return tokens, want

        def step(self, entries):
            ends = [tokens[-1] for tokens, want in entries if want]
            out = self.static if all(len(tokens) == 1 for tokens, _ in entries) else torch.zeros_like(self.static)
            out.fill_(-1)
            for i, t in enumerate(ends):
                out[i] = t
            return out[:len(ends)]

    search = BeamSearch(Runner(), 1, 4)
    from return_b200.engine.beams import _Search
    group = [_Search(i, [0] * (n - 1) + [10 + i]) for i, n in enumerate(lengths)]
    assert search._prompts(group)[:, 0].tolist() == [10 + i for i in range(len(lengths))]


class BeamRunner:
    """A runner on the host: a real cache manager, logits that follow from a request's tokens alone."""

    def __init__(self, pages, max_reside=8, chunk=16, page=4, window=None):
        from return_b200.cache.manager import CacheManager, GroupSpec
        self.manager = CacheManager([GroupSpec("full", page, pages)] + ([GroupSpec("win", page, pages, window=window)] if window else []), max_reside)
        self.vocab_size, self.max_positions = 11, 200
        self.config = types.SimpleNamespace(max_reside=max_reside, prefill_chunk=chunk)
        self.env = types.SimpleNamespace(device="cpu")
        self.tokens, self.steps = {}, 0

    def add_request(self, rid):
        self.manager.add(rid)
        self.tokens[rid] = []

    def free_request(self, rid):
        self.manager.free(rid)
        del self.tokens[rid]

    def reserve(self, rid, tokens, want):
        from return_b200.engine.batch import StepEntry
        return StepEntry(rid, tokens, want, self.manager.append(rid, len(tokens)))

    def fork_requests(self, pairs):
        self.manager.fork_all(pairs)
        for src, dst in pairs:
            self.tokens[dst] = list(self.tokens[src])

    def step(self, entries):
        self.manager.check()
        self.steps += 1
        out = []
        for e in entries:
            known = self.tokens[e.rid]
            assert e.start == len(known) and self.manager.length(e.rid) == len(known) + len(e.tokens)
            known += e.tokens
            if e.want:
                seed = 7
                for t in known:
                    seed = (seed * 31 + t + 1) % 1000003
                out.append(torch.randn(self.vocab_size, generator=torch.Generator().manual_seed(seed)))
        return torch.stack(out) if out else torch.empty((0, self.vocab_size))


def host_beams(runner, prompts, monkeypatch, beams=3, new=9, eos=None):
    import contextlib
    from plain import branch_plain
    from return_b200.engine.beams import BeamSearch
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    search = BeamSearch(runner, beams, new, 1.0, eos)
    monkeypatch.setattr(search, "_select", lambda live, logits, n: branch_plain.beam_select(
        logits, torch.tensor([x for s in live for x in s.scores]), n, min(search.keep, n * logits.shape[1])))
    return [[(r.output_ids, r.score, r.finish_reason) for r in results] for results in search.run(prompts)]


@pytest.mark.parametrize("window", [None, 6])
@pytest.mark.parametrize("eos", [None, 5])
def test_beam_search_puts_prompts_off_that_find_no_pages(monkeypatch, eos, window):
    """Down to a pool that holds the beams of one prompt alone, the results are those of a pool that holds all; below it the search raises."""
    from return_b200.cache.manager import KVCapacityError
    rs = np.random.RandomState(4)
    prompts = [[int(x) for x in rs.randint(0, 11, n)] for n in (13, 30, 2, 1, 22, 17, 9)]
    most = BeamRunner(500, window=window)
    want = host_beams(most, prompts, monkeypatch, eos=eos)
    refused, steps = 0, []
    for pages in range(8, 60):
        runner = BeamRunner(pages, window=window)
        try:
            assert host_beams(runner, prompts, monkeypatch, eos=eos) == want
            assert not refused or pages > refused
            steps.append(runner.steps)
        except KVCapacityError:
            assert not steps, "a larger pool holds what a smaller one held"
            refused = pages
        runner.manager.check()
        assert runner.manager.num_requests == 0 and not runner.tokens
    assert 8 <= refused < 20 and max(steps) > min(steps) == most.steps
    # a prompt that does not fit alone
    with pytest.raises(KVCapacityError):
        host_beams(BeamRunner(refused, window=window), prompts, monkeypatch, eos=eos)
