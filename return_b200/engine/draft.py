"""Drafted tokens from the request's own text: what followed the last tokens where they stood before.

The reference drafts nothing.  A request's next tokens are looked up by its last ``longest`` tokens, or fewer down to ``shortest``, in its
prompt and output: each earlier place of the same tokens offers what came behind it.  Several places make a tree, in which common
beginnings are one line.  Host code only; a request's places are kept up token by token, so a step costs a few look-ups.
"""
from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

from .request import Request


class PromptLookup:
    def __init__(self, max_tokens: int, longest: int = 4, shortest: int = 2, places: int = 4):
        """``max_tokens``: most drafted tokens of a tree, beside its root.  ``places``: the latest places of the same tokens that are
        looked at."""
        if max_tokens < 0 or not 1 <= shortest <= longest or places < 1:
            raise ValueError("max_tokens: not negative; 1 <= shortest <= longest; at least one place")
        self.max_tokens, self.longest, self.shortest, self.places = max_tokens, longest, shortest, places

    def _index(self, req: Request) -> Dict[Tuple[int, ...], List[int]]:
        """Where each run of ``shortest`` to ``longest`` tokens ends (the index behind it), oldest first, for all tokens but the last."""
        state = req.draft_state
        if state is None:
            state = req.draft_state = {"tokens": list(req.prompt_ids), "done": 0, "ends": {}}
        known = state["tokens"]
        known += req.output[len(known) - len(req.prompt_ids):]
        ends = state["ends"]
        for end in range(max(1, state["done"]), len(known)):          # the run that ends at the last token is what is looked up
            for n in range(self.shortest, min(self.longest, end) + 1):
                ends.setdefault(tuple(known[end - n:end]), []).append(end)
        state["done"] = max(1, len(known))
        return ends

    def propose(self, req: Request, room: int) -> Tuple[List[int], List[int]]:
        """(tokens, parents) of a tree whose root is the request's last token, with up to ``room`` nodes beside it."""
        room = min(room, self.max_tokens)
        ends = self._index(req)
        known: Sequence[int] = req.draft_state["tokens"]
        tokens, parents = [known[-1]], [-1]
        if room <= 0:
            return tokens, parents
        children: Dict[Tuple[int, int], int] = {}                     # (node, token) -> the child
        for n in range(min(self.longest, len(known)), self.shortest - 1, -1):
            found = ends.get(tuple(known[len(known) - n:]), [])
            for end in found[:-self.places - 1:-1]:                   # the latest first
                node = 0
                for tok in known[end:end + room]:
                    child = children.get((node, tok))
                    if child is None:
                        if len(tokens) > room:
                            break
                        child = children[(node, tok)] = len(tokens)
                        tokens.append(tok)
                        parents.append(node)
                    node = child
            if len(tokens) > 1:                                       # a longer run's places say more than a shorter one's
                break
        return tokens, parents
