"""Drafted trees and beam search through the engine."""
import math
import os
import json
import subprocess
import sys

import pytest
import torch

import helpers
from helpers import plain

pytestmark = pytest.mark.gpu


def engine_of(model_dir, dtype="float32", **kw):
    from return_b200.engine.config import EngineConfig
    from return_b200.engine.engine import Engine
    base = dict(max_token=1024, max_reside=8, page_size=16, prefill_chunk=64, dtype=dtype)
    base.update(kw)
    return Engine(model_dir, EngineConfig(**base))


class Knows:
    """Drafts what the requests are known to say, behind a wrong first branch, ``depth`` tokens of it; every third step nothing."""

    def __init__(self, outputs, vocab, depth):
        self.outputs, self.vocab, self.depth, self.calls = outputs, vocab, depth, 0

    def propose(self, req, room):
        self.calls += 1
        tokens, parents = [req.all_ids[-1]], [-1]
        rest = self.outputs[req.id][len(req.output):][:self.depth]
        if self.calls % 3 == 0 or room < 2 * len(rest) + 1 or not rest:
            return tokens, parents
        tokens += [(rest[0] + 1) % self.vocab, rest[0]] + [(t + 1) % self.vocab for t in rest[1:]] + rest[1:]
        parents += [0, 0] + [2] * (len(rest) - 1)
        last = 2
        for i in range(len(rest) - 1):
            parents.append(last)
            last = 3 + len(rest) - 1 + i
        return tokens, parents


@pytest.mark.parametrize("case", ["A", "B", "C"])
def test_logits_of_drafted_trees(tmp_path, case):
    """A tree's logits are those of its lines, whatever the windows; the accepted line's rows then serve later steps."""
    from return_b200.engine.batch import StepEntry
    d = helpers.make_model_dir(tmp_path, case)
    vocab = helpers.CASES[case][0]["vocab_size"]
    r = engine_of(d, page_size=helpers.CASES[case][2]).runner
    prompts = [helpers.random_ids(vocab, n, 5 + n) for n in (33, 70, 1)]
    trees = [(helpers.random_ids(vocab, 9, 2), [-1, 0, 0, 1, 2, 2, 4, 6, 7]), (helpers.random_ids(vocab, 4, 3), [-1, 0, 1, 2]), (helpers.random_ids(vocab, 1, 4), None)]
    entries = []
    for i, (prompt, (tokens, parents)) in enumerate(zip(prompts, trees)):
        r.add_request(i)
        r.step([r.reserve(i, prompt)])
    for i, (tokens, parents) in enumerate(trees):
        entries.append(StepEntry(i, tokens, (), r.manager.append(i, len(tokens)), parents))
    logits, batch = r.step_trees(entries)
    lines, row, nxt = [], 0, []
    for prompt, (tokens, parents) in zip(prompts, trees):
        for x in range(len(tokens)):
            line, y = [], x
            while y >= 0:
                line.insert(0, y)
                y = -1 if parents is None else parents[y]
            want = helpers.plain_logits(d, prompt + [tokens[y] for y in line])[-1]
            assert (logits[row].cpu() - want).abs().max() < 2e-4, (x, line)
            row += 1
        lines.append(line)
        for a, b in zip(line, line[1:] + [None]):
            lines[-1] = line
        follow = {a: tokens[b] for a, b in zip(line, line[1:])}
        nxt += [follow.get(x, (tokens[x] + 1) % vocab if parents is None or all(tokens[c] != (tokens[x] + 1) % vocab for c in range(len(tokens))) else vocab - 1)
                for x in range(len(tokens))]
    path, count, emitted = r.commit_trees(batch, torch.tensor(nxt, dtype=torch.int32, device="cuda:0"))
    assert count.tolist() == [len(x) for x in lines] and [p[:c] for p, c in zip(path.tolist(), count.tolist())] == lines
    for i, line in enumerate(lines):
        r.manager.truncate(i, len(prompts[i]) + len(line))
        more = helpers.random_ids(vocab, 2, 9)
        got = r.step([r.reserve(i, more, [0, 1])])
        want = helpers.plain_logits(d, prompts[i] + [trees[i][0][x] for x in line] + more)[-2:]
        assert (got.cpu() - want).abs().max() < 2e-4
    r.manager.check()


@pytest.mark.parametrize("case,chunk", [("A", 64), ("B", 13), ("C", 32)])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_drafted_generation_says_the_same(tmp_path, case, chunk, temperature):
    d = helpers.make_model_dir(tmp_path, case)
    vocab = helpers.CASES[case][0]["vocab_size"]
    prompts = [helpers.random_ids(vocab, n, 1 + i) * 2 for i, n in enumerate((5, 17, 30))]
    kw = dict(page_size=helpers.CASES[case][2], prefill_chunk=chunk)
    ask = dict(max_new_tokens=24, temperature=temperature, top_p=0.95, seed=11)
    want = engine_of(d, **kw).generate(prompts, **ask)
    for depth in (1, 4, 9):
        eng = engine_of(d, draft_tokens=20, **kw)
        eng.drafter = Knows({f"gen-{i}": w.output_ids for i, w in enumerate(want)}, vocab, depth)
        got = eng.generate(prompts, **ask)
        assert [g.output_ids for g in got] == [w.output_ids for w in want]
        assert all(abs(a - b) < 1e-3 for g, w in zip(got, want) for a, b in zip(g.output_logprobs, w.output_logprobs))
        st = eng.stats()
        if chunk > 50:                  # a small budget leaves no room for the deep trees
            assert st["drafts_held"] > 0 and st["drafted"] > st["drafts_held"]
        assert st["page_used"] == 0
        eng.runner.manager.check()
    eng = engine_of(d, draft_tokens=8, **kw)                # the engine's own drafts
    got = eng.generate(prompts, **ask)
    assert [g.output_ids for g in got] == [w.output_ids for w in want]
    eng.runner.manager.check()


def test_drafts_end_where_the_request_ends(tmp_path):
    """Stop sequences and lengths inside an accepted line, a sequence limit, sessions kept behind it."""
    d = helpers.make_model_dir(tmp_path, "A")
    prompts = [helpers.random_ids(256, 9, 3), helpers.random_ids(256, 20, 4)]
    want = engine_of(d).generate(prompts, max_new_tokens=20, temperature=0.0)
    for stop_at in (3, 7, 12):
        stop = [want[0].output_ids[stop_at - 1:stop_at + 1]]
        ref = engine_of(d).generate(prompts, max_new_tokens=20, temperature=0.0, stop_ids=stop)
        eng = engine_of(d, draft_tokens=20)
        eng.drafter = Knows({f"gen-{i}": w.output_ids for i, w in enumerate(want)}, 256, 6)
        got = eng.generate(prompts, max_new_tokens=20, temperature=0.0, stop_ids=stop, keep=True)
        assert [(g.output_ids, g.finish_reason) for g in got] == [(w.output_ids, w.finish_reason) for w in ref]
        eng.runner.manager.check()
        # a kept session goes on from what was committed
        more = prompts[0] + got[0].output_ids + [5]
        again = eng.generate([more], max_new_tokens=4, temperature=0.0, ids=["gen-0"])
        assert again[0].output_ids == plain.greedy_generate(plain.read_config(d), plain.read_weights(d), more, 4)
    eng = engine_of(d, draft_tokens=20, max_model_len=32)
    eng.drafter = Knows({f"gen-{i}": w.output_ids for i, w in enumerate(want)}, 256, 6)
    got = eng.generate(prompts, max_new_tokens=20, temperature=0.0)
    ref = engine_of(d, max_model_len=32).generate(prompts, max_new_tokens=20, temperature=0.0)
    assert [(g.output_ids, g.finish_reason) for g in got] == [(w.output_ids, w.finish_reason) for w in ref]


def test_drafts_where_pages_run_short(tmp_path):
    """Trees that find no pages are left out; requests give way and come back as without drafts."""
    d = helpers.make_model_dir(tmp_path, "B")
    prompts = [helpers.random_ids(384, 24, 20 + i) for i in range(4)]
    want = engine_of(d, page_size=8).generate(prompts, max_new_tokens=30, temperature=0.0)
    for pool in (120, 152, 184):
        eng = engine_of(d, page_size=8, max_token=pool, draft_tokens=20)
        eng.drafter = Knows({f"gen-{i}": w.output_ids for i, w in enumerate(want)}, 384, 5)
        got = eng.generate(prompts, max_new_tokens=30, temperature=0.0)
        assert [g.output_ids for g in got] == [w.output_ids for w in want]
        eng.runner.manager.check()
        assert eng.stats()["page_used"] == 0


def test_drafted_generation_in_bfloat16(tmp_path):
    d = helpers.make_model_dir(tmp_path, "B")
    prompts = [helpers.random_ids(384, n, 5 + i) for i, n in enumerate((9, 40, 71))]
    want = engine_of(d, "bfloat16").generate(prompts, max_new_tokens=16, temperature=0.0)
    eng = engine_of(d, "bfloat16", draft_tokens=16)
    eng.drafter = Knows({f"gen-{i}": w.output_ids for i, w in enumerate(want)}, 384, 4)
    got = eng.generate(prompts, max_new_tokens=16, temperature=0.0)
    same = sum(a == b for g, w in zip(got, want) for a, b in zip(g.output_ids, w.output_ids))
    assert same >= 0.8 * 48 and [g.output_ids[0] for g in got] == [w.output_ids[0] for w in want]
    assert eng.stats()["drafts_held"] > 0


def pisatar_dir(tmp_path):
    from return_b200.benchmark import pisatar_raw_config
    from return_b200.config.pisatar_config import PisatarConfig
    from return_b200.weights import loader
    d = os.path.join(str(tmp_path), "pisatar")
    loader.write_random_model(d, PisatarConfig(pisatar_raw_config(64, 128, 2, 1, 4, 100)), 3, torch.float32)
    return d


def test_models_with_states_take_no_trees(tmp_path):
    d = pisatar_dir(tmp_path)
    with pytest.raises(ValueError, match="draft_tokens"):
        engine_of(d, draft_tokens=4)
    r = engine_of(d).runner
    assert not r.takes_trees()
    from return_b200.engine.batch import StepEntry
    r.add_request("a")
    with pytest.raises(ValueError, match="per-request state"):
        r.step_trees([StepEntry("a", [1, 2], (), r.manager.append("a", 2), [-1, 0])])
    q = engine_of(helpers.make_model_dir(tmp_path, "A")).runner
    q.add_request("a")
    with pytest.raises(ValueError, match="step_trees"):
        q.step([StepEntry("a", [1, 2], [0], q.manager.append("a", 2), [-1, 0])])


# ---------------------------------------------------------------------------------------- beams

def plain_beams(logits_of, prompt, beams, new, penalty, eos):
    """The search written out, whole sequences at every step: (tokens, score, reason), best first."""
    live, left = [([], 0.0)], []
    for _ in range(new):
        found = []
        for b, (tokens, score) in enumerate(live):
            lp = torch.log_softmax(logits_of(prompt + tokens)[-1].double(), -1)
            found += [(score + float(x), b, t) for t, x in enumerate(lp.tolist())]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        nxt = []
        for rank, (score, b, t) in enumerate(found[:2 * beams if eos is not None else beams]):
            tokens = live[b][0] + [t]
            if t == eos:
                if rank < beams:
                    left.append((tokens, score / len(tokens) ** penalty, "stop"))
            elif len(nxt) < beams:
                nxt.append((tokens, score))
        left = sorted(left, key=lambda h: -h[1])[:beams]
        live = nxt
        if len(left) == beams and live[0][1] / len(live[0][0]) ** penalty <= left[-1][1]:
            live = []
            break
    left += [(t, s / len(t) ** penalty, "length") for t, s in live]
    return sorted(left, key=lambda h: -h[1])[:beams]


@pytest.mark.parametrize("case,beams,penalty,graph", [("A", 3, 1.0, True), ("B", 4, 0.0, False), ("C", 2, 2.0, True), ("A", 1, 1.0, False)])
def test_beam_search_equals_plain(tmp_path, case, beams, penalty, graph):
    d = helpers.make_model_dir(tmp_path, case)
    vocab = helpers.CASES[case][0]["vocab_size"]
    prompts = [helpers.random_ids(vocab, n, 30 + n) for n in (4, 31, 16)]
    eng = engine_of(d, page_size=helpers.CASES[case][2], max_reside=7, prefill_chunk=20, use_cuda_graph=graph)
    logits_of = lambda ids: helpers.plain_logits(d, ids)  # noqa: E731
    free = plain_beams(logits_of, prompts[0], beams, 6, penalty, None)
    for eos in (None, free[0][0][2]):              # a word that the best line has in it
        got = eng.beam_search(prompts, beams=beams, max_new_tokens=6, length_penalty=penalty, eos_token_id=eos)
        for prompt, results in zip(prompts, got):
            want = plain_beams(logits_of, prompt, beams, 6, penalty, eos)
            assert [(r.output_ids, r.finish_reason) for r in results] == [(t, why) for t, _, why in want]
            assert all(abs(r.score - s) < 1e-3 for r, (_, s, _) in zip(results, want))
        eng.runner.manager.check()
        assert eng.runner.manager.num_requests == 0


@pytest.mark.parametrize("chunk,lengths", [(1, (3, 1)), (2, (1, 1, 1, 1, 1)), (4, (5, 1, 2, 6))])
def test_beam_search_of_prompts_in_single_tokens(tmp_path, chunk, lengths):
    """Prompts that end in captured steps of single tokens, several steps after each other."""
    d = helpers.make_model_dir(tmp_path, "A")
    prompts = [helpers.random_ids(256, n, 60 + i) for i, n in enumerate(lengths)]
    eng = engine_of(d, max_reside=10, prefill_chunk=chunk, use_cuda_graph=True)
    for _ in range(2):                             # graphs captured, and replayed
        for prompt, results in zip(prompts, eng.beam_search(prompts, beams=2, max_new_tokens=3)):
            want = plain_beams(lambda ids: helpers.plain_logits(d, ids), prompt, 2, 3, 1.0, None)
            assert [r.output_ids for r in results] == [t for t, _, _ in want]
            assert all(abs(r.score - s) < 1e-3 for r, (_, s, _) in zip(results, want))


@pytest.mark.parametrize("kind", ["window", "states"])
def test_beams_hold_what_their_tokens_say(tmp_path, kind):
    """A long search over pages, windows and states that part ways again and again: every result's score is that of its tokens run afresh."""
    d = pisatar_dir(tmp_path) if kind == "states" else helpers.make_model_dir(tmp_path, "C")
    eng = engine_of(d, page_size=8, max_reside=10)
    vocab = eng.runner.vocab_size
    prompts = [helpers.random_ids(vocab, n, 50 + n) for n in (37, 3)]
    got = eng.beam_search(prompts, beams=5, max_new_tokens=40, length_penalty=0.0)
    assert eng.runner.manager.num_requests == 0
    for prompt, results in zip(prompts, got):
        assert len(results) == 5 and len({tuple(r.output_ids) for r in results}) == 5
        assert [r.score for r in results] == sorted((r.score for r in results), reverse=True)
        for r in results:
            ids = prompt + r.output_ids
            runner = eng.runner
            runner.add_request("check")
            logits = torch.cat([runner.step([runner.reserve("check", ids[i:i + 50], range(min(50, len(ids) - i)))]) for i in range(0, len(ids), 50)])
            runner.free_request("check")
            lp = torch.log_softmax(logits[len(prompt) - 1:-1].double(), -1)
            total = float(lp.gather(1, torch.tensor(r.output_ids, device=lp.device)[:, None]).sum())
            assert math.isclose(total, r.logprob, abs_tol=2e-3) and math.isclose(r.score, r.logprob, abs_tol=1e-9)
    # generation goes on as before
    assert eng.generate(prompts, max_new_tokens=3, temperature=0.0)[0].num_tokens == 3


def test_beam_search_where_pages_run_short(tmp_path):
    """Prompts that find no pages beside the others wait; the results are those of a pool that holds all."""
    d = helpers.make_model_dir(tmp_path, "A")
    prompts = [helpers.random_ids(256, n, 70 + n) for n in (40, 25, 60, 5)]
    ask = dict(beams=2, max_new_tokens=20)
    want = engine_of(d, page_size=8).beam_search(prompts, **ask)
    for pool in (136, 176, 240):
        eng = engine_of(d, page_size=8, max_token=pool)
        got = eng.beam_search(prompts, **ask)
        assert [[r.output_ids for r in x] for x in got] == [[r.output_ids for r in x] for x in want]
        assert all(abs(a.score - b.score) < 1e-3 for x, y in zip(got, want) for a, b in zip(x, y))
        eng.runner.manager.check()
        assert eng.runner.manager.num_requests == 0 and eng.stats()["page_used"] == 0


def test_beam_search_refuses_and_gives_back(tmp_path):
    from return_b200.cache.manager import KVCapacityError
    from return_b200.engine.request import Request
    d = helpers.make_model_dir(tmp_path, "A")
    eng = engine_of(d, max_token=128, page_size=8, max_reside=4)
    for kw, error in ((dict(beams=0), ValueError), (dict(beams=5), ValueError), (dict(max_new_tokens=0), ValueError), (dict(eos_token_id=256), ValueError),
                      (dict(max_new_tokens=200), KVCapacityError)):
        with pytest.raises(error):
            eng.beam_search([[1, 2, 3]], **{**dict(beams=2, max_new_tokens=4), **kw})
    with pytest.raises(ValueError):
        eng.beam_search([[]])
    with pytest.raises(KVCapacityError):           # the pool does not hold four beams of this length
        eng.beam_search([helpers.random_ids(256, 60, 1)], beams=4, max_new_tokens=60)
    eng.runner.manager.check()
    assert eng.runner.manager.num_requests == 0 and eng.stats()["page_used"] == 0
    eng.add_request(Request("a", [1, 2, 3]))
    with pytest.raises(RuntimeError):
        eng.beam_search([[1, 2, 3]], beams=2)


def test_command_line(tmp_path):
    d = helpers.make_model_dir(tmp_path, "A")
    base = [sys.executable, "-m", "return_b200", "generate", "--model", d, "--dtype", "float32", "--max-token", "512", "--new", "6", "--temperature", "0",
            "--prompt-ids", "5,17,3,5,17,3"]
    run = lambda *more: [json.loads(x) for x in subprocess.run(base + list(more), capture_output=True, text=True, check=True, cwd=helpers.ROOT).stdout.splitlines()]  # noqa: E731
    want = run()
    assert run("--draft-tokens", "6") == want or run("--draft-tokens", "6")[0]["output_ids"] == want[0]["output_ids"]
    beams = run("--beams", "3", "--length-penalty", "0.5")[0]["beams"]
    assert len(beams) == 3 and all(len(b["output_ids"]) == 6 for b in beams)
