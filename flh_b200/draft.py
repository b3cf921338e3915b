"""Trees of drafted tokens for speculative decoding: what Decoder.draft and Decoder.accept (flh_b200.model) take.

A step of a server: draft a tree behind the last token that the model chose, run it through Decoder.draft, keep the longest branch
that the model agrees with, go on behind it.

    tree = DraftTree([-1, 0, 0, 1], device)                       # token 0: the last chosen one; 1 and 2 its children, 3 a child of 1
    logits = model.draft(ids, cache, lengths, tree)               # ids [B, 4]
    path, accepted, chosen = tree.accept_greedy(ids, logits)
    lengths = model.accept(cache, lengths, path, accepted, tree.size)
    # chosen [B]: token 0 of the next tree
"""
from __future__ import annotations

import torch

MAX_TOKENS = 64


class DraftTree:
    """parents[i] < i is the token that token i follows; token 0 is the root and has parent -1.

    bits   int64 [S], on the device: bit j of bits[i] is set where j is i or an ancestor of it (tree_attention's `tree`)
    depth  int32 [S], on the device: ancestors of each token
    """

    def __init__(self, parents, device=None):
        parents = [int(x) for x in parents]
        if not 1 <= len(parents) <= MAX_TOKENS:
            raise ValueError(f"a tree has 1 .. {MAX_TOKENS} tokens")
        if parents[0] != -1 or any(not 0 <= up < i for i, up in enumerate(parents) if i):
            raise ValueError("parents[0] must be -1 and every other parent an earlier token")
        branches = []
        for i, up in enumerate(parents):
            branches.append((branches[up] if i else []) + [i])
        bits = [sum(1 << j for j in b) for b in branches]
        deepest = max(len(b) for b in branches)
        self.parents, self.size = parents, len(parents)
        self.bits = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device=device)
        self.depth = torch.tensor([len(b) - 1 for b in branches], dtype=torch.int32, device=device)
        self._branches = torch.tensor([b + [0] * (deepest - len(b)) for b in branches], dtype=torch.int32, device=device)
        self._above = torch.tensor([[j in b for j in range(len(parents))] for b in branches], device=device)
        self._up = torch.tensor([max(up, 0) for up in parents], device=device)

    @torch.no_grad()
    def accept_greedy(self, ids, logits):
        """The longest branch all of whose tokens (below the root) are what the model would have chosen after their parents; of
        branches that are as long the first.  Tokens below the root whose logits have a NaN (they did not fit the cache), or their
        parent's, are not accepted; what follows a root with NaN logits is not chosen by the model.  ids [B, S], logits [B, S, vocab] -> path int32 [B, depth of the tree + 1] (indices
        behind the branch's end are not used), accepted int32 [B], chosen [B]: what the model chooses after the branch's last token."""
        choice = logits.argmax(dim=-1)                                                    # [B, S]
        lost = logits.gather(2, choice[:, :, None])[:, :, 0].isnan()                      # argmax takes a NaN for the largest
        agreed = (ids == choice[:, self._up]) & ~lost & ~lost[:, self._up]
        agreed[:, 0] = True
        whole = (agreed[:, None, :] | ~self._above).all(dim=-1)                           # every token from the root down to i
        best = torch.where(whole, self.depth + 1, 0).argmax(dim=-1)                       # the first of the deepest
        return self._branches[best], self.depth[best] + 1, choice.gather(1, best[:, None])[:, 0]
