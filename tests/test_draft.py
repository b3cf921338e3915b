"""Trees of drafted tokens on the host: ancestor bits, depths, the branch that greedy decoding accepts."""
import pytest
import torch

from flh_b200.draft import DraftTree


def test_bits_and_depth():
    t = DraftTree([-1, 0, 0, 1, 3, 2])
    assert t.bits.tolist() == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100101] and t.depth.tolist() == [0, 1, 1, 2, 3, 2] and t.size == 6
    assert t.bits.dtype == torch.int64 and t.depth.dtype == torch.int32
    chain = DraftTree(range(-1, 63))
    assert chain.size == 64 and chain.bits[63].item() == -1 and chain.bits[62].item() == (1 << 63) - 1 and chain.depth[63].item() == 63
    star = DraftTree([-1] + [0] * 63)
    assert star.bits[63].item() == 1 - (1 << 63)


@pytest.mark.parametrize("parents", [[], [0], [-1, 1], [-1, -1], [-1, 0, 2], [-1] + [0] * 64])
def test_what_is_no_tree(parents):
    with pytest.raises(ValueError):
        DraftTree(parents)


def test_accept_greedy():
    t = DraftTree([-1, 0, 0, 1, 1, 2])
    want = torch.tensor([[3, 7, 1, 9, 9, 9],        # after the root 3, after token 1 7, after token 2 1
                         [5, 5, 5, 5, 5, 5],
                         [2, 4, 4, 4, 4, 0]])
    logits = torch.nn.functional.one_hot(want, 10).float()
    ids = torch.tensor([[0, 3, 3, 7, 7, 1],         # both children agree: of the branches as long the first, 0 1 3
                        [5, 1, 2, 5, 5, 5],         # no child of the root agrees; what lies below them does not count
                        [8, 2, 2, 0, 0, 4]])        # 0 2 5
    path, accepted, chosen = t.accept_greedy(ids, logits)
    assert path.dtype == torch.int32 and accepted.dtype == torch.int32
    assert [p[:n] for p, n in zip(path.tolist(), accepted.tolist())] == [[0, 1, 3], [0], [0, 2, 5]]
    assert chosen.tolist() == [9, 5, 0]
    one = DraftTree([-1])
    path, accepted, chosen = one.accept_greedy(torch.zeros(2, 1, dtype=torch.int64), logits[:2, :1])
    assert path.tolist() == [[0], [0]] and accepted.tolist() == [1, 1] and chosen.tolist() == [3, 5]


def test_the_configuration_takes_its_fields_in_the_order_they_had():
    from flh_b200.model import DecoderConfig
    c = DecoderConfig(4096, 32, 8, 14336, 4, 32000, 500000.0, 1e-6, "token_asym", 2)
    assert (c.rope_theta, c.eps, c.act_mode, c.tp) == (500000.0, 1e-6, "token_asym", 2) and c.max_positions == 32768


def test_tokens_without_logits_are_not_accepted():
    t = DraftTree([-1, 0, 0, 1])
    logits = torch.nn.functional.one_hot(torch.tensor([[4, 0, 5, 2], [0, 3, 3, 3], [4, 2, 5, 2]]), 6).float()
    logits[0, 1, 3] = float("nan")                  # token 1, which agrees
    logits[1, 0] = float("nan")                     # the root: its children would agree with what argmax makes of it
    logits[2, 3] = float("nan")
    path, accepted, chosen = t.accept_greedy(torch.tensor([[1, 4, 4, 0], [1, 0, 0, 3], [1, 4, 1, 2]]), logits)
    assert [p[:n] for p, n in zip(path.tolist(), accepted.tolist())] == [[0, 2], [0], [0, 1]] and chosen[0] == 5 and chosen[2] == 2
