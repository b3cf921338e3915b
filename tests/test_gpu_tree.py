"""Attention of a drafted tree over a ragged KV cache, its accumulated weights, and what happens to the cache around it, against
64-bit restatements (tree_reference.py).  The wiring either side is flh/quantized_model/modeling_llama.py:389-440."""
import numpy as np
import pytest
import torch

import tree_reference as R
from helpers import rs

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _normal(seed, *shape, dtype=torch.float16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _check_attention(C, q, k, v, lengths, tree, observe=True, scale=None):
    want, tol, w, wtol = R.attention(q, k, v, lengths.tolist(), tree, scale)
    out = C.tree_attention(q, k, v, lengths, tree=tree, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    R.assert_close(out, want, tol)
    if observe:
        start = torch.rand(w.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
        weights = start.clone()
        again = C.tree_attention(q, k, v, lengths, tree=tree, weights=weights, scale=scale)
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))
        total = start.double() + w
        R.assert_close(weights, total, wtol + 2.0 ** -24 * total.abs())
        assert torch.equal(weights[w == 0], start[w == 0])
        twice = start.clone()
        C.tree_attention(q, k, v, lengths, tree=tree, weights=twice, scale=scale)
        assert torch.equal(twice, weights)
    assert C.tree_attention_status()[0] == 0


# (query heads, kv heads, head size, tokens, lengths, room behind the last drafted entry)
SHAPES = [
    (4, 4, 64, 1, [1], 0), (4, 2, 64, 1, [0], 3), (8, 1, 128, 1, [31, 32, 33], 5), (32, 32, 128, 1, [500], 64), (4, 4, 128, 2, [127, 128, 129, 1], 1),
    (6, 2, 128, 3, [95, 700], 0), (7, 1, 64, 5, [1000, 3, 64], 40), (8, 8, 128, 16, [257], 0), (64, 8, 128, 13, [2047, 100], 9), (16, 2, 128, 2, [4099], 100),
    (2, 2, 64, 17, [63, 640], 2), (4, 1, 64, 64, [513, 0], 0), (8, 1, 128, 64, [1531, 64], 31), (5, 5, 128, 64, [1, 2, 3], 70), (8, 4, 128, 33, [900, 20, 333], 5),
    (3, 1, 128, 43, [260], 0), (40, 1, 128, 64, [300], 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,D,S,lengths,room", SHAPES)
def test_attention_and_weights(cuda, nh, nkv, D, S, lengths, room, dtype):
    B, T = len(lengths), max(lengths) + S + room
    q, k, v = _normal(1, B, S, nh, D, dtype=dtype, scale=1.5), _normal(2, B, nkv, T, D, dtype=dtype), _normal(3, B, nkv, T, D, dtype=dtype)
    r = rs(S + nh)
    trees = torch.stack([R.random_tree(r, S)[0] for _ in range(B)]).cuda()
    _check_attention(cuda, q, k, v, _ints(lengths), trees)
    _check_attention(cuda, q, k, v, _ints(lengths), trees[0].contiguous(), observe=False)
    _check_attention(cuda, q, k, v, _ints(lengths), None, observe=False)


@pytest.mark.parametrize("S,nh,nkv", [(1, 2, 2), (64, 8, 1)])
def test_many_sequences_of_uneven_lengths(cuda, S, nh, nkv):
    r = rs(5)
    lengths = [int(x) for x in r.randint(0, 90, size=70)] + [3000]
    T = 3000 + S
    q, k, v = _normal(1, 71, S, nh, 64), _normal(2, 71, nkv, T, 64), _normal(3, 71, nkv, T, 64)
    _check_attention(cuda, q, k, v, _ints(lengths), None)


@pytest.mark.parametrize("S,nh", [(3, 4), (9, 4), (20, 4), (33, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_shares(cuda, S, nh, D):
    """Hundreds of thousands of entries: every ring, barrier and tile of scores is gone around many times, with rows that change their maximum."""
    lengths = [150001, 90007, 33]
    T = lengths[0] + S
    q, k, v = _normal(1, 3, S, nh, D, scale=1.5), _normal(2, 3, 1, T, D), _normal(3, 3, 1, T, D)
    k[0, 0, :lengths[0]] *= torch.linspace(0.2, 3.0, lengths[0], device="cuda")[:, None].half()
    _check_attention(cuda, q, k, v, _ints(lengths), None)


def test_one_long_sequence(cuda):
    q, k, v = _normal(1, 1, 2, 8, 128, dtype=torch.bfloat16), _normal(2, 1, 1, 70003, 128, dtype=torch.bfloat16), _normal(3, 1, 1, 70003, 128, dtype=torch.bfloat16)
    _check_attention(cuda, q, k, v, _ints([70001]), None)


@pytest.mark.parametrize("S", [3, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_single_entries_out(cuda, S, dtype):
    """Scores in the hundreds: every maximum is replaced on the way, most weights are zero."""
    q, k, v = _normal(1, 2, S, 4, 128, dtype=dtype, scale=12.0), _normal(2, 2, 2, 900, 128, dtype=dtype, scale=4.0), _normal(3, 2, 2, 900, 128, dtype=dtype)
    k[:, :, :400] = k[:, :, :400].sort(dim=2).values                          # rising scores in some directions
    _check_attention(cuda, q, k, v, _ints([800, 333]), None, scale=0.5)


@pytest.mark.parametrize("S,g,nkv", [(2, 4, 296), (8, 4, 148), (64, 3, 148)])
@pytest.mark.parametrize("dtype", TYPES)
def test_light_entries_beside_heavy_ones(cuda, S, g, nkv, dtype):
    """Four entries with value 0 whose weights are e^18 = 2^26 times those of all the others, which have value 1: together these give the
    result, and each by itself is below float16's smallest number where the heaviest weight is 1."""
    n, D = 16384, 64
    k, v = torch.zeros(1, nkv, n + S, D, device="cuda", dtype=dtype), torch.ones(1, nkv, n + S, D, device="cuda", dtype=dtype)
    k[:, :, 0:128:32, 0], v[:, :, 0:128:32] = 18.0, 0.0                       # in a tile of every warp, and of both streams of many rows
    q = torch.zeros(1, S, nkv * g, D, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    out = cuda.tree_attention(q, k, v, _ints([n]), scale=1.0).double()
    light = (n - 4 + torch.arange(1, S + 1, device="cuda")).double() * np.exp(-18.0)
    want = (light / (4 + light))[None, :, None, None].expand(out.shape)
    # a weight and the result are off by half a step each, the exponentials by less than 2^-18 (a score of 18 of exact products, its scaling
    # and the power of two: 26 * 2^-23 + 2^-21); a weight under 2^-14 absolutely by half of float16's smallest number: 2^-25 relative to a
    # heaviest weight that is raised to 2^7 at least, 2^-32; a result under 2^-14 by 2^-25.  Sums of up to 16,384 weights in binary32: 2^-10
    # at most if one after the other, and equal ones are summed in tiles
    u = R.HALF_STEP[dtype]
    tol = want * (2.02 * u + 2.0 ** -17 + 2.0 ** -10) + (light[None, :, None, None].expand(out.shape) * np.exp(18.0) * 2.0 ** -32 / 4 + 2.0 ** -25 if dtype == torch.float16 else 0.0)
    R.assert_close(out, want, tol)


@pytest.mark.parametrize("S,nh,nkv,D", [(4, 2, 1, 64), (9, 8, 4, 128), (64, 4, 1, 128), (64, 8, 1, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_that_see_nothing(cuda, S, nh, nkv, D, dtype):
    lengths = [0, 40, 0]
    tree = torch.stack([R.chain(S)] * 3)
    tree[0, 0] = tree[0, S - 1] = 0
    tree[1, 1] = 0                                                             # sees the committed entries
    tree[2] = 0
    q, k, v = _normal(1, 3, S, nh, D, dtype=dtype), _normal(2, 3, nkv, 130, D, dtype=dtype), _normal(3, 3, nkv, 130, D, dtype=dtype)
    _check_attention(cuda, q, k, v, _ints(lengths), tree.cuda())
    out = cuda.tree_attention(q, k, v, _ints(lengths), tree=tree.cuda())
    assert not out[0, 0].any() and not out[0, S - 1].any() and not out[2].any() and out[1, 1].any()


@pytest.mark.parametrize("S,nh,nkv,D", [(6, 2, 1, 64), (2, 4, 4, 128), (8, 16, 4, 128), (64, 2, 1, 128), (48, 8, 1, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_seen_may_hold_anything(cuda, S, nh, nkv, D, dtype):
    """NaN and infinities behind the drafted entries change nothing; in a drafted entry only for the tokens that see it."""
    lengths, T = [37, 130], 300
    q, k, v = _normal(1, 2, S, nh, D, dtype=dtype), _normal(2, 2, nkv, T, D, dtype=dtype), _normal(3, 2, nkv, T, D, dtype=dtype)
    r = rs(9)
    tree = torch.stack([R.random_tree(r, S)[0] for _ in lengths])
    tree[:, S - 1] = 1 | (-(1 << 63) if S == 64 else 1 << (S - 1))             # only the last token sees the last one
    for i in range(S - 1):
        assert not (int(tree[0, i]) >> (S - 1)) & 1
    for b, n in enumerate(lengths):
        k[b, :, n + S:], v[b, :, n + S:] = float("nan"), float("inf")
    _check_attention(cuda, q, k, v, _ints(lengths), tree.cuda())
    for fill_k, fill_v in ((None, float("inf")), (None, float("nan")), (float("nan"), None), (float("inf"), float("-inf"))):
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lengths):
            if fill_k is not None:
                k2[b, :, n + S - 1] = fill_k
            if fill_v is not None:
                v2[b, :, n + S - 1, ::3] = fill_v
        out = cuda.tree_attention(q, k2, v2, _ints(lengths), tree=tree.cuda())
        plain = cuda.tree_attention(q, k, v, _ints(lengths), tree=tree.cuda())
        assert torch.equal(out[:, :S - 1], plain[:, :S - 1]) and bool(out[:, :S - 1].isfinite().all())
        if fill_k is None:
            bad = torch.zeros(D, dtype=torch.bool, device="cuda")
            bad[::3] = True
            assert torch.equal(out[:, S - 1][..., bad].isnan(), torch.full_like(out[:, S - 1][..., bad], fill_v).isnan())
            assert not out[:, S - 1][..., bad].isfinite().any()
            want, tol, _, _ = R.attention(q, k2, v2, lengths, tree)
            R.assert_close(out, want, tol)
        else:
            assert out[:, S - 1].isnan().all()
        w = torch.zeros(2, nkv, T, device="cuda")
        cuda.tree_attention(q, k2, v2, _ints(lengths), tree=tree.cuda(), weights=w)
        if fill_k is None:
            assert w.isfinite().all()
        for b, n in enumerate(lengths):
            assert not w[b, :, n + S:].any()


@pytest.mark.parametrize("S,nh", [(2, 4), (40, 4)])
def test_scores_that_are_all_minus_infinity_are_not_empty(cuda, S, nh):
    q, k, v = torch.full((1, S, nh, 64), 1.0, device="cuda").half(), torch.full((1, 1, 80, 64), float("-inf"), device="cuda").half(), _normal(3, 1, 1, 80, 64)
    assert cuda.tree_attention(q, k, v, _ints([30])).isnan().all()


@pytest.mark.parametrize("S,nh,nkv", [(3, 8, 2), (20, 8, 2)])
def test_lengths_at_and_over_the_end_of_the_cache(cuda, S, nh, nkv):
    """Entries T and up do not exist: drafted tokens there are not seen; lengths outside 0 .. T are the nearer end."""
    T, D = 70, 128
    q, k, v = _normal(1, 5, S, nh, D), _normal(2, 5, nkv, T, D), _normal(3, 5, nkv, T, D)
    given = [T, T - 1, T - S, 1000, -5]
    _check_attention(cuda, q, k, v, _ints(given), None)
    assert torch.equal(cuda.tree_attention(q, k, v, _ints(given)), cuda.tree_attention(q, k, v, _ints([T, T - 1, T - S, T, 0])))


def test_strides_of_q(cuda):
    k, v, lengths = _normal(2, 2, 2, 90, 64), _normal(3, 2, 2, 90, 64), _ints([50, 70])
    by_head = _normal(1, 2, 4, 6, 64)                                          # [B, heads, S, D]
    want = cuda.tree_attention(by_head.transpose(1, 2).contiguous(), k, v, lengths)
    assert torch.equal(cuda.tree_attention(by_head.transpose(1, 2), k, v, lengths), want)
    wide = torch.zeros(2, 6, 4, 72, device="cuda", dtype=torch.float16)
    wide[..., :64] = by_head.transpose(1, 2)
    assert torch.equal(cuda.tree_attention(wide[..., :64], k, v, lengths), want)
    one = by_head[:1, :, :1].transpose(1, 2)
    assert torch.equal(cuda.tree_attention(one.expand(2, 1, 4, 64), k, v, lengths)[0], cuda.tree_attention(one.contiguous(), k[:1], v[:1], lengths[:1])[0])


@pytest.mark.parametrize("S", [1, 40])
def test_offsets_over_32_bits(cuda, S):
    """A cache of 2.7 billion values, 5.4 GB each of K and V: the last sequence lies behind 2^31 values and 2^32 bytes."""
    T = 1 << 21
    k, v = (torch.empty(5, 2, T, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    q = _normal(1, 5, S, 4, 128)
    n = 150
    for b in range(5):
        k[b, :, :n + S], v[b, :, :n + S] = _normal(10 + b, 2, n + S, 128), _normal(20 + b, 2, n + S, 128)
    lengths = _ints([n] * 5)
    w = torch.zeros(5, 2, T, device="cuda")
    out = cuda.tree_attention(q, k, v, lengths, weights=w)
    want, tol, ww, wtol = R.attention(q, k[:, :, :n + S], v[:, :, :n + S], [n] * 5)
    R.assert_close(out, want, tol)
    R.assert_close(w[:, :, :n + S], ww, wtol + 2.0 ** -24 * ww)
    # the far end of the last sequence
    k[4, :, T - n - S:], v[4, :, T - n - S:] = k[4, :, :n + S].clone(), v[4, :, :n + S].clone()
    now = cuda.cache_accept([k], [v], _ints([n, n, n, n, T - S - n]), _ints([[0, S - 1]] * 5 if S > 1 else [[0]] * 5), _ints([2 if S > 1 else 1] * 5), S)
    assert now.tolist()[4] == T - S - n + (2 if S > 1 else 1)
    del k, v


def test_a_recorded_step_follows_the_lengths(cuda):
    """Two graphs over the same caches, replayed with other lengths, beside eager calls on another stream."""
    B, S, nh, nkv, D, T = 3, 5, 8, 2, 128, 600
    k, v = _normal(2, B, nkv, T, D), _normal(3, B, nkv, T, D)
    qs = [_normal(4 + i, B, S, nh, D) for i in range(2)]
    lengths, w = [_ints([10, 20, 30]) for _ in range(2)], [torch.zeros(B, nkv, T, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        cuda.tree_attention(qs[0], k, v, lengths[0], weights=w[0])
    torch.cuda.current_stream().wait_stream(side)
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cuda.tree_attention(qs[i], k, v, lengths[i], weights=w[i]))
        graphs.append(g)
    w[0].zero_(), w[1].zero_()
    lengths[0].copy_(_ints([500, 0, 77]))
    lengths[1].copy_(_ints([1, 595, 300]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = None
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    with torch.cuda.stream(streams[2]):
        eager = cuda.tree_attention(qs[0], k, v, _ints([333, 4, 5]))
    torch.cuda.synchronize()
    for i in range(2):
        want, tol, ww, wtol = R.attention(qs[i], k, v, lengths[i].tolist())
        R.assert_close(outs[i], want, tol)
        R.assert_close(w[i], ww, wtol + 2.0 ** -24 * ww)
    want, tol, _, _ = R.attention(qs[0], k, v, [333, 4, 5])
    R.assert_close(eager, want, tol)


# ------------------------------------------------------------------------------------------------------------ rope_kv_at
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,nh,nkv,D", [(1, 1, 4, 4, 64), (3, 5, 8, 2, 128), (2, 64, 4, 1, 128), (70, 9, 2, 1, 96)])
def test_rope_kv_at_equals_the_tensor_operations(cuda, B, S, nh, nkv, D, dtype):
    from flh_b200.model import rope, rope_tables
    r = rs(B + S)
    T = 100
    qkv = _normal(1, B * S, (nh + 2 * nkv) * D, dtype=dtype)
    lengths = [int(x) for x in r.randint(0, T - S + 1, size=B)]
    positions = _ints(r.randint(0, 5000, size=(B, S)).tolist())
    cos, sin = rope_tables(torch.arange(5000, device="cuda"), D, 10000.0)
    k, v = _normal(2, B, nkv, T, D, dtype=dtype), _normal(3, B, nkv, T, D, dtype=dtype)
    want_k, want_v = k.clone(), v.clone()
    q = cuda.rope_kv_at(qkv, cos, sin, positions, _ints(lengths), k, v, nh)
    parts = qkv.view(B, S, nh + 2 * nkv, D)
    for b, n in enumerate(lengths):
        assert torch.equal(q[b:b + 1], rope(parts[b:b + 1, :, :nh], positions[b], 10000.0))
        want_k[b, :, n:n + S] = rope(parts[b:b + 1, :, nh:nh + nkv], positions[b], 10000.0)[0].transpose(0, 1)
        want_v[b, :, n:n + S] = parts[b, :, nh + nkv:].transpose(0, 1)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_rope_kv_at_outside_the_cache_and_the_tables(cuda):
    from flh_b200.model import rope_tables
    B, S, nh, nkv, D, T = 3, 4, 2, 1, 64, 10
    qkv = _normal(1, B * S, (nh + 2 * nkv) * D)
    cos, sin = rope_tables(torch.arange(16, device="cuda"), D, 10000.0)
    k, v = _normal(2, B, nkv, T, D), _normal(3, B, nkv, T, D)
    k0, v0 = k.clone(), v.clone()
    positions = _ints([[0, 1, 2, 3], [15, 16, -1, 0], [1, 1, 1, 1]])
    q = cuda.rope_kv_at(qkv, cos, sin, positions, _ints([8, 0, -2]), k, v, nh)
    assert torch.equal(q.isnan().any(-1).any(-1).cpu(), torch.tensor([[False] * 4, [False, True, True, False], [False] * 4]))
    assert torch.equal(k[0, :, :8], k0[0, :, :8]) and not torch.equal(k[0, :, 8:], k0[0, :, 8:])      # two of four tokens fit
    assert k[1, :, 1:3].isnan().all() and not k[1, :, 0].isnan().any() and torch.equal(k[1, :, 4:], k0[1, :, 4:])
    assert torch.equal(v[1, 0, :4], qkv.view(B, S, -1)[1, :, (nh + nkv) * D:])
    assert torch.equal(k[2, :, 2:], k0[2, :, 2:]) and torch.equal(v[2, :, 2:], v0[2, :, 2:])           # tokens 2 and 3 lie at entries 0 and 1


# ----------------------------------------------------------------------------------------------------- accept and evict
def _layers(seed, L, B, nkv, T, D, dtype):
    k, v = _normal(seed, L, B, nkv, T, D, dtype=dtype), _normal(seed + 1, L, B, nkv, T, D, dtype=dtype)
    w = torch.rand(L, B, nkv, T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return k, v, w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,B,nkv,D,S,A", [(1, 1, 1, 64, 1, 1), (3, 2, 4, 128, 16, 5), (2, 5, 1, 128, 64, 64), (128, 1, 2, 64, 33, 7), (2, 3, 2, 8, 7, 7), (1, 2, 3, 256, 64, 40)])
@pytest.mark.parametrize("weighted", [False, True])
def test_cache_accept(cuda, L, B, nkv, D, S, A, dtype, weighted):
    r = rs(A + S)
    T = 200
    lengths = [int(x) for x in r.randint(0, T - S + 1, size=B)]
    counts = [int(x) for x in r.randint(0, A + 1, size=B)]
    counts[0] = A
    paths = np.stack([np.sort(r.choice(S, A, replace=False)) for _ in range(B)])
    k, v, w = _layers(4, L, B, nkv, T, D, dtype)
    want = [x.clone() for x in (k, v, w)]
    for b, (n, a) in enumerate(zip(lengths, counts)):
        at = [n + int(x) for x in paths[b, :a]]
        for x, y in zip(want, (k, v, w)):
            x[:, b, :, n:n + a] = y[:, b][:, :, at]
        want[2][:, b, :, n + a:n + S] = 0
    now = cuda.cache_accept(list(k), list(v), _ints(lengths), _ints(paths.tolist()), _ints(counts), S, weights=list(w) if weighted else None)
    assert now.tolist() == [n + a for n, a in zip(lengths, counts)]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    if weighted:
        assert torch.equal(w, want[2])


def test_cache_accept_in_any_order_and_outside(cuda):
    """A path that goes down, names an entry twice, has indices that are no drafted token, a count over the path's length, and entries
    behind the end of the cache."""
    k, v, w = _layers(8, 1, 3, 2, 20, 64, torch.float16)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    path = _ints([[5, 3, 3, 0], [-1, 6, 2, 1 << 20], [2, 3, 1, 0]])
    now = cuda.cache_accept([k[0]], [v[0]], _ints([10, 4, 18]), path, _ints([4, 99, 3]), 6, weights=[w[0]])
    assert now.tolist() == [14, 8, 20]
    for x, x0 in ((k, k0), (v, v0), (w, w0)):
        assert torch.equal(x[0, 0, :, 10:14], x0[0, 0][:, [15, 13, 13, 10]])
        assert torch.equal(x[0, 1, :, 4:8], x0[0, 1][:, [4, 5, 6, 7]])
        assert torch.equal(x[0, 2, :, 18:20], x0[0, 2][:, [18, 19]])
        assert torch.equal(x[0, :, :, :4], x0[0, :, :, :4])
    assert torch.equal(k[0, 0, :, 14:], k0[0, 0, :, 14:]) and not w[0, 0, :, 14:16].any() and not w[0, 1, :, 8:10].any()
    assert torch.equal(w[0, 0, :, 16:], w0[0, 0, :, 16:])


def _check_evict(C, k, v, w, lengths, keep, recent):
    L, B, nkv, T, _ = k.shape
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    kept, left, now = C.cache_evict(list(k), list(v), list(w), _ints(lengths), keep, recent)
    wn = w0.cpu().numpy()
    assert torch.equal(w.view(torch.int32), w0.view(torch.int32))
    assert now.tolist() == [min(max(n, 0), T, keep) for n in lengths]
    for y in range(L):
        for b in range(B):
            n = min(max(lengths[b], 0), T)
            for h in range(nkv):
                rows = R.evict(wn[y, b, h], n, keep, recent)
                m = len(rows)
                assert m == min(n, keep)
                assert kept[y, b, h].tolist() == rows.tolist() + [-1] * (keep - m)
                at = torch.from_numpy(rows).cuda()
                assert torch.equal(left[y, b, h, :m].view(torch.int32), w0[y, b, h, at].view(torch.int32)) and not left[y, b, h, m:].any()
                assert torch.equal(k[y, b, h, :m], k0[y, b, h, at]) and torch.equal(v[y, b, h, :m], v0[y, b, h, at])
                assert torch.equal(k[y, b, h, m:], k0[y, b, h, m:]) and torch.equal(v[y, b, h, m:], v0[y, b, h, m:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,B,nkv,D,T,lengths,keep,recent", [
    (1, 1, 1, 64, 5, [4], 2, 1), (1, 1, 1, 64, 5, [5], 1, 0), (1, 1, 2, 128, 33, [33], 33, 5), (2, 3, 2, 128, 700, [700, 650, 20], 64, 17), (3, 2, 1, 64, 2100, [2100, 1025], 1024, 0),
    (1, 2, 2, 128, 300, [300, 299], 298, 298), (1, 1, 1, 128, 40000, [39999], 9001, 100), (2, 1, 3, 80, 500, [480], 100, 50), (1, 2, 1, 8, 4096, [4096, 4000], 4000, 1), (1, 1, 1, 64, 60000, [60000], 30000, 10),
])
def test_cache_evict(cuda, L, B, nkv, D, T, lengths, keep, recent, dtype):
    k, v, w = _layers(6, L, B, nkv, T, D, dtype)
    _check_evict(cuda, k, v, w, lengths, keep, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "odd", "zero"])
@pytest.mark.parametrize("keep,recent", [(300, 40), (128, 128), (999, 3)])
def test_cache_evict_ties_and_odd_weights(cuda, kind, keep, recent):
    """Ties go to the lower index; NaN is the largest; -0 and 0 are the same."""
    k, v, w = _layers(6, 1, 2, 2, 1200, 64, torch.float16)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_((w * 4).floor())
    elif kind == "signs":
        w.sub_(0.5)
        w[..., ::5] = -0.0
        w[..., 1::5] = 0.0
    elif kind == "zero":
        w.zero_()
        w[..., 777] = 1e-45
    else:
        w[..., ::7] = float("nan")
        w[..., 1::7] = float("inf")
        w[..., 2::7] = float("-inf")
        w[..., 3::7] = -float("nan")
    _check_evict(cuda, k, v, w, [1200, 1001], keep, recent)


@pytest.mark.parametrize("B,T", [(1, 3000), (80, 4500), (2, 40000)])
def test_cache_evict_ties_in_longer_rows(cuda, B, T):
    """Three values in all weights, in every form of the selection: rows of a few thousand entries, longer ones, those of several blocks."""
    k, v, w = _layers(6, 1, B, 1, T, 8, torch.float16)
    w.copy_((w * 3).floor() / 4)
    _check_evict(cuda, k, v, w, [T - b % 7 for b in range(B)], T // 3, 50)


def test_cache_evict_of_sequences_that_fit(cuda):
    k, v, w = _layers(6, 2, 4, 1, 50, 128, torch.bfloat16)
    _check_evict(cuda, k, v, w, [0, 1, 50, -3], 50, 10)
    _check_evict(cuda, k, v, w, [0, 1, 10, 77], 10, 10)


def test_a_run_of_steps(cuda):
    """Append, attend, accept and evict as a server does, over ragged sequences, against the same steps as tensor operations."""
    from flh_b200.model import rope, rope_tables
    B, nh, nkv, D, T, S = 3, 4, 2, 64, 96, 6
    r = rs(21)
    cos, sin = rope_tables(torch.arange(512, device="cuda"), D, 10000.0)
    k, v = torch.full((B, nkv, T, D), float("nan"), device="cuda").half(), torch.full((B, nkv, T, D), float("nan"), device="cuda").half()
    w = torch.zeros(B, nkv, T, device="cuda")
    lengths, at = _ints([0] * B), _ints([0] * B)                              # entries, and how many tokens the sequences are long
    held = [[[] for _ in range(nkv)] for _ in range(B)]                       # (k row, v row, weight) of every entry
    for step in range(14):
        tree, depth = R.random_tree(r, S)
        tree, depth = tree.cuda(), depth.cuda()
        qkv = _normal(100 + step, B * S, (nh + 2 * nkv) * D)
        positions = (at[:, None] + depth).contiguous()
        q = cuda.rope_kv_at(qkv, cos, sin, positions, lengths, k, v, nh)
        out = cuda.tree_attention(q, k, v, lengths, tree=tree, weights=w)
        parts = qkv.view(B, S, nh + 2 * nkv, D)
        turned = torch.cat([rope(parts[b:b + 1, :, :nh + nkv], positions[b], 10000.0) for b in range(B)])
        full = max(len(held[b][0]) for b in range(B)) + S
        kk, vv = torch.zeros(B, nkv, full, D, device="cuda").half(), torch.zeros(B, nkv, full, D, device="cuda").half()
        for b in range(B):
            for h in range(nkv):
                rows = held[b][h]
                for i, e in enumerate(rows):
                    kk[b, h, i], vv[b, h, i] = e[0], e[1]
                kk[b, h, len(rows):len(rows) + S] = turned[b, :, nh + h]
                vv[b, h, len(rows):len(rows) + S] = parts[b, :, nh + nkv + h]
        want, tol, ww, _ = R.attention(turned[:, :, :nh], kk, vv, [len(held[b][0]) for b in range(B)], tree)
        R.assert_close(out, want, tol)
        # one branch of every tree: a token and its ancestors
        pick = [int(x) for x in r.randint(0, S, size=B)]
        branch = [[j for j in range(S) if (int(tree[i]) >> j) & 1] for i in pick]
        path = _ints([x + [0] * (S - len(x)) for x in branch])
        for b in range(B):
            for h in range(nkv):
                n = len(held[b][h])
                held[b][h] = [[e[0], e[1], e[2] + ww[b, h, i]] for i, e in enumerate(held[b][h])] + [[kk[b, h, n + j], vv[b, h, n + j], ww[b, h, n + j]] for j in branch[b]]
        accepted = _ints([len(x) for x in branch])
        lengths = cuda.cache_accept([k], [v], lengths, path, accepted, S, weights=[w])
        at = at + accepted
        if step % 4 == 3:
            kept, left, lengths = cuda.cache_evict([k], [v], [w], lengths, 16, 5)
            w = left[0].clone()
            for b in range(B):
                for h in range(nkv):
                    stay = [i for i in kept[0, b, h].tolist() if i >= 0]
                    weight = np.array([float(e[2]) for e in held[b][h]])
                    n = len(weight)
                    if n > 16:          # what stayed is as heavy as what went, up to rounding
                        gone = [i for i in range(n - 5) if i not in stay]
                        assert set(range(n - 5, n)) <= set(stay) and len(stay) == 16
                        assert min(weight[i] for i in stay if i < n - 5) >= max(weight[i] for i in gone) * (1 - 1e-5)
                    else:
                        assert stay == list(range(n))
                    held[b][h] = [held[b][h][i] for i in stay]
        assert lengths.tolist() == [len(held[b][0]) for b in range(B)]
        for b in range(B):
            for h in range(nkv):
                n = len(held[b][h])
                assert torch.equal(k[b, h, :n], torch.stack([e[0] for e in held[b][h]])) and torch.equal(v[b, h, :n], torch.stack([e[1] for e in held[b][h]]))
                got = w[b, h, :n].double()
                assert torch.allclose(got, torch.stack([e[2] for e in held[b][h]]), rtol=1e-4, atol=1e-6)
                assert not w[b, h, n:].any()


def test_recorded_append_accept_and_evict(cuda):
    """The other calls in one graph, replayed with other lengths and paths, against the same calls made eagerly."""
    from flh_b200.model import rope_tables
    L, B, nkv, T, D, S, nh = 2, 3, 2, 120, 64, 6, 4
    cos, sin = rope_tables(torch.arange(300, device="cuda"), D, 10000.0)
    k, v, w = _layers(31, L, B, nkv, T, D, torch.float16)
    qkv, lengths, path, accepted = _normal(32, B * S, (nh + 2 * nkv) * D), _ints([5, 6, 7]), _ints([[0, 2, 4]] * B), _ints([1, 2, 3])
    positions = (lengths[:, None] + torch.arange(S, dtype=torch.int32, device="cuda")).contiguous()

    def calls(k, v, w):
        q = [cuda.rope_kv_at(qkv, cos, sin, positions, lengths, k[y], v[y], nh) for y in range(L)]
        now = cuda.cache_accept(list(k), list(v), lengths, path, accepted, S, weights=list(w))
        kept, left, after = cuda.cache_evict(list(k), list(v), list(w), now, 20, 4)
        return [*q, now, kept, left, after]

    calls(*(x.clone() for x in (k, v, w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        outs = calls(k, v, w)
    for n, paths, counts in (([100, 0, 50], [[1, 2, 5], [0, 1, 2], [3, 4, 5]], [3, 1, 0]), ([114, 20, 30], [[0, 1, 2]] * 3, [3, 3, 3])):
        lengths.copy_(_ints(n)), path.copy_(_ints(paths)), accepted.copy_(_ints(counts))
        positions.copy_(lengths[:, None] + torch.arange(S, dtype=torch.int32, device="cuda"))
        copies = [x.clone() for x in (k, v, w)]
        g.replay()
        want = calls(*copies)
        for a, b in zip([*outs, k, v, w], [*want, *copies]):
            assert torch.equal(a, b)


def test_calls_on_a_stream_of_their_own_and_without_the_native_ones(cuda, monkeypatch):
    k, v, w = _layers(41, 2, 2, 2, 90, 128, torch.bfloat16)
    q, lengths = _normal(42, 2, 3, 4, 128, dtype=torch.bfloat16), _ints([60, 33])
    path, accepted = _ints([[0, 2], [1, 2]]), _ints([2, 2])

    def calls(k, v, w):
        out = cuda.tree_attention(q, k[0], v[0], lengths, weights=w[0])
        now = cuda.cache_accept(list(k), list(v), lengths, path, accepted, 3, weights=list(w))
        return [out, now, *cuda.cache_evict(list(k), list(v), list(w), now, 30, 5), k, v, w]

    want = calls(*(x.clone() for x in (k, v, w)))
    copies = [x.clone() for x in (k, v, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls(*copies)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.setattr(cuda, "_host", None)
    got = calls(*(x.clone() for x in (k, v, w)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batches(cuda):
    k, n = torch.zeros(0, 2, 10, 64, dtype=torch.float16, device="cuda"), _ints([])
    assert cuda.tree_attention(torch.zeros(0, 3, 4, 64, dtype=torch.float16, device="cuda"), k, k.clone(), n).shape == (0, 3, 4, 64)
    assert cuda.cache_accept([k], [k.clone()], n, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), n.clone(), 3).shape == (0,)
    kept, left, now = cuda.cache_evict([k], [k.clone()], [torch.zeros(0, 2, 10, device="cuda")], n, 4, 1)
    assert kept.shape == (1, 0, 2, 4) and left.shape == (1, 0, 2, 10) and now.shape == (0,)
    one = _layers(1, 1, 2, 2, 10, 64, torch.float16)
    assert cuda.cache_accept([one[0][0]], [one[1][0]], _ints([3, 4]), torch.zeros(2, 0, dtype=torch.int32, device="cuda"), _ints([5, 5]), 3).tolist() == [3, 4]


@pytest.mark.parametrize("B,S,nh,nkv", [(40, 2, 8, 2), (40, 20, 8, 2), (3, 40, 64, 8), (300, 1, 2, 2), (33, 64, 16, 2)])
def test_every_division_of_the_work(cuda, B, S, nh, nkv):
    """More jobs than CTAs, more sequences than a warp has lanes, jobs that are cut and jobs that are not, in a cache with room to spare."""
    r = rs(B)
    for T, top in ((4000, 700), (150, 80)):
        lengths = [int(x) for x in r.randint(0, top, size=B)]
        q, k, v = _normal(1, B, S, nh, 64), _normal(2, B, nkv, T, 64), _normal(3, B, nkv, T, 64)
        w = torch.zeros(B, nkv, T, device="cuda")
        out = cuda.tree_attention(q, k, v, _ints(lengths), weights=w)
        some = sorted(set([0, 1, B // 2, B - 1, *r.randint(0, B, size=4).tolist()]))
        want, tol, ww, wtol = R.attention(q[some], k[some, :, :top + S], v[some, :, :top + S], [lengths[b] for b in some])
        R.assert_close(out[some], want, tol)
        R.assert_close(w[some][:, :, :top + S], ww, wtol + 2.0 ** -24 * ww)
        assert torch.allclose(w.sum(-1), torch.full((B, nkv), float(S * nh // nkv), device="cuda"), rtol=1e-4)
    assert cuda.tree_attention_status()[0] == 0


def _graph_time(f):
    """Device time of a call, replayed in a graph: the best of several."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f()
    best = float("inf")
    for _ in range(12):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.parametrize("S,nh,nkv,long,short,others,observe", [
    (5, 64, 8, 60000, 1000, 15, False), (1, 64, 8, 60000, 500, 31, False), (1, 64, 8, 60000, 500, 31, True), (1, 64, 8, 40000, 2000, 20, False), (64, 32, 8, 30000, 300, 4, False),
    (5, 64, 8, 60000, 1000, 15, True), (5, 64, 8, 16000, 500, 73, True), (64, 32, 8, 30000, 300, 4, True),
    (1, 64, 8, 60000, 500, 36, False), (1, 32, 32, 28000, 500, 8, False), (5, 64, 8, 16000, 500, 17, False), (5, 64, 8, 16000, 500, 73, False), (1, 64, 8, 60000, 500, 36, True),
])
def test_one_long_sequence_among_short_ones(cuda, S, nh, nkv, long, short, others, observe):
    """The work goes by what the sequences hold: one long one costs about what the same entries cost in sequences that are alike."""
    B, T, D = 1 + others, long + S, 64
    lengths, total = [short] * others, long + others * short
    lengths.insert(others // 3, long)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = _normal(4, B, S, nh, D)
    k, v = (torch.randn(B, nkv, T, D, dtype=torch.float16, device="cuda", generator=g) for _ in range(2))
    w = torch.zeros(B, nkv, T, device="cuda") if observe else None
    n, even = _ints(lengths), _ints([total // B] * B)
    out = cuda.tree_attention(q, k, v, n, weights=w)
    for b in (0, others // 3, B - 1):
        want, tol, ww, wtol = R.attention(q[b:b + 1], k[b:b + 1, :, :lengths[b] + S], v[b:b + 1, :, :lengths[b] + S], lengths[b:b + 1])
        R.assert_close(out[b:b + 1], want, tol)
        if observe:
            R.assert_close(w[b:b + 1, :, :lengths[b] + S], ww, wtol + 2.0 ** -24 * ww)
            assert not w[b, :, lengths[b] + S:].any()
    uneven, even = (_graph_time(lambda: cuda.tree_attention(q, k, v, x, weights=w)) for x in (n, even))
    print(f"\nuneven {uneven:.1f} us, even {even:.1f} us")
    assert uneven < 2.5 * even, (uneven, even)
    assert cuda.tree_attention_status()[0] == 0


@pytest.mark.parametrize("g,D", [(8, 128), (4, 128), (3, 64), (8, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_odd_values_where_two_blocks_of_rows_share_a_tile(cuda, g, D, dtype):
    """Stale and drafted values that are not finite, in tiles that two streams of rows read: as without them for the rows that do not see them,
    the same every time."""
    S, B, T = 64, 40, 400
    r = rs(g + D)
    lengths = [int(x) for x in r.randint(0, T - S, size=B)]
    q, k, v = _normal(1, B, S, 2 * g, D, dtype=dtype), _normal(2, B, 2, T, D, dtype=dtype), _normal(3, B, 2, T, D, dtype=dtype)
    tree = torch.stack([R.random_tree(r, S)[0] for _ in lengths]).cuda()
    tree[:, S - 1] = 1 | -(1 << 63)                                            # only the last token sees the last one
    clean = v.clone()
    for b, n in enumerate(lengths):
        clean[b, :, n + S:] = 0
        v[b, :, n + S:] = float("nan")
        v[b, :, n + S - 1, b % 8::8] = float("inf")
    want = cuda.tree_attention(q, k, clean, _ints(lengths), tree=tree)
    for _ in range(20):
        got = cuda.tree_attention(q, k, v, _ints(lengths), tree=tree)
        assert torch.equal(got[:, :S - 1], want[:, :S - 1])
        for b in (0, 1, 17, B - 1):
            odd = torch.arange(D, device="cuda") % 8 == b % 8
            assert torch.equal(got[b, S - 1][:, ~odd], want[b, S - 1][:, ~odd]) and bool((got[b, S - 1][:, odd] == float("inf")).all())
    assert cuda.tree_attention_status()[0] == 0


@pytest.mark.parametrize("B,S,nh,nkv,D,T", [(3, 4, 8, 2, 128, 200), (3, 4, 8, 2, 64, 9000), (40, 5, 6, 3, 64, 700), (3, 33, 8, 2, 128, 500), (4, 64, 12, 2, 64, 300), (2, 64, 16, 2, 128, 5000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_the_first_tokens_only(cuda, B, S, nh, nkv, D, T, dtype):
    """counted tokens of each sequence add to the weights, none to all of them; the output is that of all tokens."""
    r = rs(B + S)
    lengths, counted = [int(x) for x in r.randint(0, T - S, size=B)], [int(x) for x in r.randint(0, S + 1, size=B)]
    lengths[0], counted[-1], counted[0], counted[1] = T - S, 1, 0, S
    q, k, v = _normal(1, B, S, nh, D, dtype=dtype), _normal(2, B, nkv, T, D, dtype=dtype), _normal(3, B, nkv, T, D, dtype=dtype)
    tree = torch.stack([R.random_tree(r, S)[0] for _ in lengths]).cuda()
    start = torch.rand(B, nkv, T, device="cuda")
    w, every, given = start.clone(), start.clone(), list(counted)
    given[1], given[0] = S + 100, -3                                           # the nearer end
    out = cuda.tree_attention(q, k, v, _ints(lengths), tree=tree, weights=w, counted=_ints(given))
    assert torch.equal(out.view(torch.int16), cuda.tree_attention(q, k, v, _ints(lengths), tree=tree).view(torch.int16))
    for b, c in enumerate(counted):
        if c == 0:
            assert torch.equal(w[b], start[b])
            continue
        _, _, ww, wtol = R.attention(q[b:b + 1, :c], k[b:b + 1], v[b:b + 1], lengths[b:b + 1], tree[b:b + 1, :c])
        total = start[b:b + 1].double() + ww
        R.assert_close(w[b:b + 1], total, wtol + 2.0 ** -24 * total.abs())
    cuda.tree_attention(q, k, v, _ints(lengths), tree=tree, weights=every, counted=_ints([S] * B))
    again = start.clone()
    cuda.tree_attention(q, k, v, _ints(lengths), tree=tree, weights=again)
    assert torch.equal(every, again) and cuda.tree_attention_status()[0] == 0


def test_counted_without_the_native_call(cuda, monkeypatch):
    q, k, v, lengths, counted = _normal(1, 2, 3, 4, 64), _normal(2, 2, 2, 90, 64), _normal(3, 2, 2, 90, 64), _ints([60, 33]), _ints([1, 2])
    got = []
    for host in (cuda._host, None):
        monkeypatch.setattr(cuda, "_host", host)
        w = torch.zeros(2, 2, 90, device="cuda")
        got.append((cuda.tree_attention(q, k, v, lengths, weights=w, counted=counted), w))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and torch.allclose(w.sum((1, 2)), torch.tensor([4.0, 8.0], device="cuda"), rtol=1e-4)


@pytest.mark.parametrize("L,B,nkv,T,lengths", [(4, 4, 5, 50001, [50001, 45056, 45057, 49000]), (1, 1, 1, 400003, [400001]), (1, 1, 2, 364600, [364571])])
def test_cache_evict_of_rows_longer_than_a_block_keeps(cuda, L, B, nkv, T, lengths):
    """More keys in a block's stretch than its shared memory holds: those behind are read again, with ties on both sides."""
    k, v, w = _layers(6, L, B, nkv, T, 8, torch.float16)
    w.copy_((w * 5).floor() / 4)
    _check_evict(cuda, k, v, w, lengths, T // 2, 1000)
    k, v, w = _layers(7, L, B, nkv, T, 8, torch.float16)
    _check_evict(cuda, k, v, w, lengths, T - 6000, 3)


@pytest.mark.parametrize("S,nh,nkv", [(2, 4, 2), (8, 8, 2), (64, 8, 1)])
@pytest.mark.parametrize("k0", [512.0, 2048.0, 4096.0, 8192.0, 16384.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_millions(cuda, S, nh, nkv, k0, dtype):
    """Scores whose last place is 2^-2 .. 8 in powers of two: the entries of the largest one share the weight evenly."""
    n, D = 700, 64
    k, v = torch.zeros(1, nkv, n + S, D, device="cuda", dtype=dtype), _normal(3, 1, nkv, n + S, D, dtype=dtype)
    k[..., 0] = k0
    k[:, :, ::3, 0] = k0 * 0.75                                                # lower by hundreds of thousands and more: no weight
    q = torch.zeros(1, S, nh, D, device="cuda", dtype=dtype)
    q[..., 0] = 4096.0                                                         # products of powers of two: exact
    out = cuda.tree_attention(q, k, v, _ints([n]), scale=1.0)
    for s in range(S):
        at = [t for t in range(n + s + 1) if t % 3]
        for h in range(nh):
            x = v[0, h * nkv // nh, at].double()
            # equal weights, whatever they are rounded to: only the result's rounding and sums of 32 bits
            R.assert_close(out[0, s, h], x.mean(0), R.HALF_STEP[dtype] * 1.01 * x.mean(0).abs() + (2.02 * R.HALF_STEP[dtype] + 2.0 ** -14) * x.abs().mean(0))
