"""Decoder.draft / accept / evict: drafted tokens through the whole decoder against the plain forward of each branch."""
import pytest
import torch

from flh_b200.draft import DraftTree

pytestmark = pytest.mark.gpu


def _model(mode="group_sym", **other):
    from flh_b200.model import Decoder, DecoderConfig
    cfg = dict(hidden=256, n_heads=4, n_kv_heads=2, ffn=512, n_layers=2, vocab=128, act_mode=mode, max_positions=512)
    return Decoder(DecoderConfig(**{**cfg, **other}), torch.device("cuda"), seed=5)


def _ids(seed, *shape):
    return torch.randint(0, 128, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _near(a, b):
    # a code of the second layer that flips by one step with the last bit of the first layer's attention moves the logits by a
    # percent or two of their range (tests/test_gpu_model.py)
    err = (a.float() - b.float()).abs().max() / b.float().abs().max()
    assert err < 3e-2, err


@pytest.mark.parametrize("mode,hidden", [("group_sym", 256), ("token_asym", 256), ("group_sym", 512)])
def test_tree_equals_every_branch(cuda, mode, hidden):
    m = _model(mode, hidden=hidden)
    prompt, tree = _ids(2, 2, 20), DraftTree([-1, 0, 0, 1, 1, 2, 4], "cuda")
    ids = _ids(3, 2, tree.size)
    cache = m.new_cache(2, 64)
    m(prompt, cache=cache, start=0)
    lengths = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    logits = m.draft(ids, cache, lengths, tree)
    assert logits.shape == (2, tree.size, 128)
    for i in range(tree.size):
        branch = [j for j in range(tree.size) if (int(tree.bits[i]) >> j) & 1]
        _near(logits[:, i:i + 1], m(torch.cat((prompt, ids[:, branch]), dim=1)))


def test_sequences_of_their_own_lengths_and_the_next_step(cuda):
    """Two sequences accept different branches; the step behind them sees what they accepted."""
    m = _model()
    prompt, tree = _ids(4, 2, 12), DraftTree([-1, 0, 0, 2, 3], "cuda")
    ids, nxt = _ids(5, 2, 5), _ids(6, 2, 3)
    cache = m.new_cache(2, 40)
    m(prompt, cache=cache, start=0)
    lengths = torch.tensor([12, 9], dtype=torch.int32, device="cuda")          # the second sequence is shorter
    m.draft(ids, cache, lengths, tree)
    path = torch.tensor([[0, 2, 3, 4], [0, 1, 0, 0]], dtype=torch.int32, device="cuda")
    now = m.accept(cache, lengths, path, torch.tensor([4, 2], dtype=torch.int32, device="cuda"), tree.size)
    assert now.tolist() == [16, 11]
    logits = m.draft(nxt, cache, now)                                          # a chain
    for b, (n, branch) in enumerate(((12, [0, 2, 3, 4]), (9, [0, 1]))):
        whole = torch.cat((prompt[b, :n], ids[b, branch], nxt[b]))[None]
        for i in range(3):
            _near(logits[b:b + 1, i:i + 1], m(whole[:, :n + len(branch) + 1 + i]))


def test_a_recorded_draft_follows_the_lengths(cuda):
    m = _model()
    prompt, tree = _ids(7, 2, 24), DraftTree([-1, 0, 0], "cuda")
    cache = m.new_cache(2, 64)
    m(prompt, cache=cache, start=0)
    ids, lengths = _ids(8, 2, 3), torch.tensor([24, 24], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.draft(ids, cache, lengths, tree)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m.draft(ids, cache, lengths, tree)
    for n in ([10, 17], [24, 1]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        ids.copy_(_ids(sum(n), 2, 3))
        kv = [[c[0].clone(), c[1].clone()] for c in cache]
        g.replay()
        got = out.clone()
        for c, (k, v) in zip(cache, kv):
            c[0].copy_(k), c[1].copy_(v)
        assert torch.equal(got, m.draft(ids, cache, lengths, tree))
        for c, (k, v) in zip(cache, kv):
            c[0].copy_(k), c[1].copy_(v)


def test_the_first_draft_may_be_a_recorded_one(cuda):
    """What a decoder keeps from its first drafted pass on holds its values when that pass was only recorded."""
    m, other = _model(), _model()
    prompt, tree = _ids(7, 2, 24), DraftTree([-1, 0, 0], "cuda")
    ids, lengths = _ids(8, 2, 3), torch.tensor([24, 20], dtype=torch.int32, device="cuda")
    want = None
    for d in (other, m):
        cache = d.new_cache(2, 64)
        d(prompt, cache=cache, start=0)
        if d is other:
            want = d.draft(ids, cache, lengths, tree)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m.draft(ids, cache, lengths, tree)
    assert torch.equal(m.draft(ids, cache, lengths, tree), want)
    g.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("S", [1, 30, 100])
def test_observed_weights(cuda, S):
    """They sum to the tokens and heads that were counted, and the logits are those of a cache without them."""
    m = _model(n_heads=4, n_kv_heads=2)
    first, then = _ids(9, 2, 40), _ids(10, 2, S)
    plain, cache = m.new_cache(2, 160), m.new_cache(2, 160, observe=True)
    m(first, cache=plain, start=0), m(first, cache=cache, start=0)
    _near(m(then, cache=cache, start=40), m(then, cache=plain, start=40))
    for c in cache:
        total = 2.0 * (40 + min(S, 64))                                        # two query heads a kv head; 40 tokens, then the last 64
        assert torch.allclose(c[3].sum(-1), torch.full((2, 2), total, device="cuda"), rtol=1e-4)
        assert not c[3][:, :, 40 + S:].any() and bool((c[3][:, :, :40 + S] > 0).all())


def test_evict_and_go_on(cuda):
    """What was evicted is not seen any more, tokens keep their positions, and evicting nothing changes nothing."""
    m = _model()
    prompt = _ids(11, 2, 60)
    cache, same = m.new_cache(2, 100, observe=True), m.new_cache(2, 100, observe=True)
    m(prompt, cache=cache, start=0), m(prompt, cache=same, start=0)
    lengths = torch.tensor([60, 60], dtype=torch.int32, device="cuda")
    assert m.evict(same, lengths, 60, 10).tolist() == [60, 60]
    for a, b in zip(cache, same):
        assert all(torch.equal(x, y) for x, y in zip((a[0], a[1], a[3]), (b[0], b[1], b[3])))
    before = [[c[0].clone(), c[1].clone(), c[3].clone()] for c in cache]
    now = m.evict(cache, lengths, 24, 8)
    assert now.tolist() == [24, 24]
    step, positions = _ids(12, 2, 1), torch.tensor([60, 60], dtype=torch.int32, device="cuda")
    for c, (k, v, w) in zip(cache, before):
        assert torch.equal(c[0][:, :, 16:24], k[:, :, 52:60]) and not c[3][:, :, 24:].any()
        # the 16 heaviest of the first 52
        heavy = w[:, :, :52].topk(16, dim=-1).indices.sort(dim=-1).values
        assert torch.equal(c[1][:, :, :16], v.gather(2, heavy[..., None].expand(2, 2, 16, v.shape[-1])))
    got = m.draft(step, cache, now, positions=positions)
    # the same step on a cache where the others were never there
    clean = m.new_cache(2, 100, observe=True)
    for c, d in zip(cache, clean):
        d[0][:, :, :24], d[1][:, :, :24] = c[0][:, :, :24], c[1][:, :, :24]
    assert torch.equal(got, m.draft(step, clean, now, positions=positions))
    with pytest.raises(RuntimeError, match="observe"):
        m.evict(m.new_cache(2, 10), lengths, 5, 1)


def test_speculative_run_equals_one_token_at_a_time(cuda):
    """Greedy decoding with trees that hold the right token now and then gives the tokens of greedy decoding without them."""
    m = _model()
    prompt = _ids(13, 1, 16)
    lengths = torch.tensor([16], dtype=torch.int32, device="cuda")
    one, cache = m.new_cache(1, 128), m.new_cache(1, 128)
    first = m(prompt, cache=one, start=0)[:, -1].argmax(-1)
    m(prompt, cache=cache, start=0)
    # greedy, a token at a time, through draft() with one token: the same kernels and row order of the quantisers
    want, tok, at = [], first, lengths.clone()
    for _ in range(24):
        logits = m.draft(tok[:, None], one, at)
        want.append((int(tok), logits[0, 0].float().topk(2).values))
        tok, at = logits[:, 0].argmax(-1), at + 1
    tree, got, tok, step = DraftTree([-1, 0, 0, 1, 2], "cuda"), [], first, 0
    while len(got) < 20:
        guess = [w[0] for w in want[len(got) + 1:len(got) + 3]]
        wrong = [(g + 1) % 128 for g in guess]
        ids = [int(tok)] + ([guess[0], wrong[0], guess[1] if step % 2 else wrong[1], guess[1]] if step % 3 else [wrong[0], wrong[0], guess[1], guess[1]])
        ids = torch.tensor([ids], device="cuda")
        logits = m.draft(ids, cache, lengths, tree)
        path, accepted, tok = tree.accept_greedy(ids, logits)
        n = int(accepted)
        assert n == (1 if step % 3 == 0 else 3 if step % 2 else 2)
        got += [int(ids[0, int(i)]) for i in path[0, :n]]
        lengths = m.accept(cache, lengths, path, accepted, tree.size)
        step += 1
        assert got == [w[0] for w in want[:len(got)]]


def test_what_draft_refuses_leaves_the_cache_as_it_was(cuda):
    m = _model()
    cache, lengths = m.new_cache(2, 100), torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    for ids, tree in ((_ids(1, 2, 65), None), (_ids(1, 2, 0), None), (_ids(1, 2, 4), DraftTree([-1, 0, 0], "cuda"))):
        with pytest.raises(RuntimeError, match="1 .. 64 tokens"):
            m.draft(ids, cache, lengths, tree)
    small = _model(hidden=256, n_heads=8, n_kv_heads=8)                        # heads of 32
    other = small.new_cache(2, 100)
    with pytest.raises(RuntimeError, match="64 or 128"):
        small.draft(_ids(1, 2, 4), other, lengths)
    with pytest.raises(RuntimeError, match="64 or 128"):
        small.new_cache(2, 100, observe=True)
    assert not any(bool(c[i].any()) for c in (*cache, *other) for i in (0, 1))


def test_a_cache_longer_than_max_positions(cuda):
    """What forward() takes draft() goes on with: the tables reach to the cache's end."""
    m, other = _model(max_positions=16), _model()
    prompt, ids, lengths = _ids(21, 2, 40), _ids(22, 2, 3), torch.tensor([40, 37], dtype=torch.int32, device="cuda")
    got = []
    for d in (m, other):
        small, cache = d.new_cache(2, 10), d.new_cache(2, 70)
        first = d.draft(ids, small, torch.tensor([0, 0], dtype=torch.int32, device="cuda"))       # (the tables of a short cache come first)
        d(prompt, cache=cache, start=0)
        got.append((first, d.draft(ids, cache, lengths)))
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(a.isfinite().all())


@pytest.mark.parametrize("mode", ["group_sym", "token_asym"])
def test_tokens_behind_the_end_of_the_cache(cuda, mode):
    """They have no logits, and are not accepted; the others have those that they have in a longer cache."""
    m = _model(mode)
    prompt, tree = _ids(23, 4, 22), DraftTree([-1, 0, 1, 1, 2], "cuda")
    lengths = torch.tensor([20, 22, 17, 18], dtype=torch.int32, device="cuda")
    short, roomy = m.new_cache(4, 22), m.new_cache(4, 30)
    for c in (short, roomy):
        m(prompt, cache=c, start=0)
    ids = _ids(24, 4, 5)
    full = m.draft(ids, roomy, lengths, tree)
    for i in range(1, 5):                                                      # every token below the root is what the model would choose
        ids[:, i] = full[:, tree.parents[i]].argmax(-1)
        full = m.draft(ids, roomy, lengths, tree)
    got = m.draft(ids, short, lengths, tree)
    fits = (lengths[:, None] + torch.arange(5, device="cuda") < 22)
    assert fits.sum(1).tolist() == [2, 0, 5, 4]
    assert bool(got[~fits].isnan().all()) and torch.equal(got[fits], full[fits])
    path, accepted, chosen = tree.accept_greedy(ids, got)
    assert accepted.tolist() == [2, 1, 4, 3] and [p[:n] for p, n in zip(path.tolist(), accepted.tolist())] == [[0, 1], [0], [0, 1, 2, 4], [0, 1, 2]]
    assert m.accept(short, lengths, path, accepted, 5).tolist() == [22, 22, 21, 21]


def _observed(m, prompt, room=40):
    cache = m.new_cache(prompt.shape[0], prompt.shape[1] + room, observe=True)
    m(prompt, cache=cache, start=0)
    return cache


@pytest.mark.parametrize("n_heads,n_kv_heads", [(4, 2), (4, 1)])
def test_what_is_not_accepted_leaves_no_weights(cuda, n_heads, n_kv_heads):
    """Accepted tokens add what they would have added one at a time; whatever else was drafted makes no difference."""
    m = _model(n_heads=n_heads, n_kv_heads=n_kv_heads)
    prompt = _ids(31, 2, 30)
    # 8 tokens of which 0 2 3 6 and 0 1 are accepted; 40 of which the same are: more rows than one kernel takes
    for size in (8, 40):
        tree = DraftTree([-1, 0, 0, 2, 2, 1, 3, 4] + [7] * (size - 8), "cuda")
        path, accepted = torch.tensor([[0, 2, 3, 6], [0, 1, 0, 0]], dtype=torch.int32, device="cuda"), torch.tensor([4, 2], dtype=torch.int32, device="cuda")
        runs = []
        for seed in (33, 34):                                                  # other tokens where nothing is accepted
            ids = _ids(seed, 2, size)
            right = _ids(32, 2, 8)
            ids[0, [0, 2, 3, 6]], ids[1, [0, 1]] = right[0, [0, 2, 3, 6]], right[1, [0, 1]]
            cache, lengths = _observed(m, prompt, 50), torch.tensor([30, 30], dtype=torch.int32, device="cuda")
            before = [c[3].clone() for c in cache]
            m.draft(ids, cache, lengths, tree)
            assert all(torch.equal(c[3], w) for c, w in zip(cache, before))
            now = m.accept(cache, lengths, path, accepted, size)
            runs.append((cache, ids))
            assert now.tolist() == [34, 32]
            for c in cache:
                for b, n in enumerate((4, 2)):
                    total = (30 + n) * n_heads / n_kv_heads
                    assert torch.allclose(c[3][b].sum(-1), torch.full((n_kv_heads,), total, device="cuda"), rtol=1e-4)
                    assert not c[3][b, :, 30 + n:].any() and bool((c[3][b, :, 30:30 + n] > 0).all())
        for a, b in zip(runs[0][0], runs[1][0]):
            assert torch.equal(a[3], b[3])
        # the same, one token at a time
        cache, ids = runs[0]
        for b, branch in enumerate(([0, 2, 3, 6], [0, 1])):
            one = _observed(m, prompt[b:b + 1], 50)
            for i, t in enumerate(branch):
                m.draft(ids[b:b + 1, t:t + 1], one, torch.tensor([30 + i], dtype=torch.int32, device="cuda"))
            # the first layer sees the same q and k up to a rounding of the products before them; in the second a quantised code may flip
            assert torch.allclose(cache[0][3][b], one[0][3][0], rtol=2e-2, atol=1e-3)
            assert (cache[1][3][b] - one[1][3][0]).abs().sum() < 0.05 * one[1][3][0].sum()


def test_entries_that_are_drafted_over_have_no_weights_of_before(cuda):
    """The second sequence is shorter than the prompt that was run: what lies behind its length counts for nothing."""
    m = _model()
    prompt = _ids(41, 2, 30)
    lengths = torch.tensor([30, 22], dtype=torch.int32, device="cuda")
    for S, accepted in ((1, None), (5, 3)):
        cache = _observed(m, prompt)
        kept = [c[3].clone() for c in cache]
        m.draft(_ids(42, 2, S), cache, lengths)
        if accepted:
            m.accept(cache, lengths, torch.arange(S, dtype=torch.int32, device="cuda").repeat(2, 1), torch.full_like(lengths, accepted), S)
        for c, w in zip(cache, kept):
            n = accepted or 1
            assert bool(((c[3] - w)[1, :, :22] >= 0).all()) and torch.allclose((c[3][1, :, :22 + n].sum(-1) - w[1, :, :22].sum(-1)), torch.tensor(2.0 * n, device="cuda"), rtol=1e-3)


def test_recorded_drafts_of_an_observed_cache(cuda):
    """Two recorded steps, of one tree and of another, replayed in turn: accept counts those of the last replay."""
    m = _model()
    prompt, trees = _ids(51, 2, 24), [DraftTree([-1, 0, 0, 1], "cuda"), DraftTree([-1, 0, 1, 0, 3, 4], "cuda")]
    lengths, ids = torch.tensor([24, 20], dtype=torch.int32, device="cuda"), [_ids(52, 2, 4), _ids(53, 2, 6)]
    paths = [torch.tensor([[0, 1, 3], [0, 2, 0]], dtype=torch.int32, device="cuda"), torch.tensor([[0, 3, 4, 5], [0, 1, 2, 0]], dtype=torch.int32, device="cuda")]
    counts = [torch.tensor([3, 2], dtype=torch.int32, device="cuda"), torch.tensor([4, 0], dtype=torch.int32, device="cuda")]
    cache, eager = _observed(m, prompt, 60), _observed(m, prompt, 60)
    other, at = _observed(m, prompt, 60), lengths.clone()
    for t, i in zip(trees, ids):
        m.draft(i, other, at, t)                                               # (what is made at the first call)
    torch.cuda.synchronize()
    drafts, accepts = [], []
    for k in range(2):
        g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m.draft(ids[k], cache, at, trees[k])
        with torch.cuda.graph(h):
            now = m.accept(cache, at, paths[k], counts[k], trees[k].size)
        drafts.append(g), accepts.append((h, now))
    n = lengths.clone()
    for k, recorded in ((0, True), (1, False), (0, False), (1, True)):
        drafts[k].replay()
        if recorded:
            accepts[k][0].replay()
            at.copy_(accepts[k][1])
        else:
            at.copy_(m.accept(cache, at, paths[k], counts[k], trees[k].size))
        m.draft(ids[k], eager, n, trees[k])
        n = m.accept(eager, n, paths[k], counts[k], trees[k].size)
        assert torch.equal(at, n)
        for a, b in zip(cache, eager):
            assert torch.equal(a[3], b[3])
            for s, e in enumerate(n.tolist()):
                assert torch.equal(a[0][s, :, :e], b[0][s, :, :e]) and torch.equal(a[1][s, :, :e], b[1][s, :, :e])


def test_evicting_by_what_was_accepted(cuda):
    """Draft, accept and evict on an observed cache: the same entries stay whatever was guessed beside the accepted tokens."""
    m = _model()
    prompt, tree = _ids(61, 1, 40), DraftTree([-1, 0, 0, 1, 2, 4], "cuda")
    path, accepted, kept = torch.tensor([[0, 2, 4]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"), []
    for seed in (62, 63):
        cache, lengths, positions = _observed(m, prompt), torch.tensor([40], dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")
        for step in range(4):
            ids, right = _ids(seed + 10 * step, 1, 6), _ids(70 + step, 1, 6)
            ids[:, [0, 2, 4]] = right[:, [0, 2, 4]]
            m.draft(ids, cache, lengths, tree, positions=positions)
            lengths, positions = m.accept(cache, lengths, path, accepted, 6), positions + accepted
            if step % 2:
                lengths = m.evict(cache, lengths, 24, 6)
        kept.append([(c[0][:, :, :24].clone(), c[3].clone()) for c in cache])
    for (ka, wa), (kb, wb) in zip(*kept):
        assert torch.equal(ka, kb) and torch.equal(wa, wb)
    with pytest.raises(RuntimeError, match="observe=True"):
        m.draft(_ids(1, 1, 3), [list(c) for c in cache], lengths)


def test_attention_is_timed_as_attention(cuda, monkeypatch):
    import contextlib
    from flh_b200 import model
    m, inside, seen = _model(), [], []

    @contextlib.contextmanager
    def region(name):
        inside.append(name)
        yield
        inside.pop()

    monkeypatch.setattr(model.timing, "region", region)
    for name in ("tree_attention", "rope_kv", "rope_kv_at"):
        monkeypatch.setattr(cuda, name, lambda *a, _f=getattr(cuda, name), _n=name, **k: (seen.append((_n, list(inside))), _f(*a, **k))[1])
    cache = m.new_cache(2, 200, observe=True)
    m(_ids(1, 2, 80), cache=cache, start=0), m(_ids(2, 2, 5), cache=cache, start=80)
    m.draft(_ids(3, 2, 4), cache, torch.tensor([85, 85], dtype=torch.int32, device="cuda"))
    assert {(n, *at) for n, at in seen} == {("tree_attention", "attention"), ("rope_kv", "glue"), ("rope_kv_at", "glue")} and len(seen) == 12
