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


def test_tree_shares_cover_the_keys(monkeypatch):
    """Every share is within the launch's splits, the shares cover the longest walk, and CTAs fill the device once at most."""
    monkeypatch.setattr(ops, "num_sms", lambda: 148)
    for nodes, cached, window in (([8], [500], 0), ([16] * 8, [2040] * 8, 0), ([64] * 32, [250 * i for i in range(32)], 0), ([5, 1], [9000, 3], 700),
                                  ([1], [0], 0), ([256], [130000], 0)):
        ends = [c + k for c, k in zip(cached, nodes)]
        splits, share = ops.tree_shares(nodes, ends, window, 4, 8, sum(nodes) * 32, 128, 128, 1)
        tiles = [(e - 1) // 64 - (max(0, e - k - window + 1) if window else 0) // 64 + 1 for e, k in zip(ends, nodes)]
        assert 1 <= splits <= ops.TREE_MAX_SPLITS
        if splits == 1:
            assert share == 0
            continue
        assert share >= ops.TREE_MIN_SHARE and splits * share >= max(tiles) > (splits - 1) * share
        blocks = sum(-(-k * 4 // 128) * 8 * -(-t // share) for k, t in zip(nodes, tiles))
        assert blocks <= 148
