"""The operators around a KV cache that is drafted into and evicted from, as measurable cases.

Speculative decoding puts a tree of drafted tokens behind what a sequence has committed, attends with all of them in one pass,
keeps the branch that the model agrees with and goes on; a long-running conversation keeps the cache entries that its queries
looked at most and drops the others.  Five calls, on caches [B, kv heads, T, D] whose sequences have lengths of their own:

  append   rotary embedding of the drafted q and k at their depth in the tree, k and v written behind each sequence's length
  attend   attention of S = 1 .. 64 drafted tokens over what is committed and, by a bit mask for each token, over its ancestors;
           S = 1 is ordinary decode
  observe  the same, and the attention weights of all query heads of a kv head added up for every cache entry
  accept   the accepted branch moved together behind the committed entries, in all layers at once
  evict    the entries with the largest accumulated weights and the most recent ones kept, moved together in order, in all layers

Sizes are the attention of the 7B- and 70B-shaped decoders of flh_b200.model and of shards of them over 2 .. 8 ranks, head sizes 64
and 128, batches of 1 .. 64 sequences, contexts from one token to 65,536.
"""
import math

import torch

own = False

# (query heads, kv heads, head size) of a layer: 7B, 70B, their shards over 2, 4 and 8 ranks, the small decoder of the tests
HEADS = ((32, 32, 128), (64, 8, 128), (16, 16, 128), (8, 1, 128), (16, 2, 128), (4, 4, 128), (4, 2, 64), (4, 4, 64))
MAX_ATTEND = 1_000_000                 # largest B * kv heads * context of an attention
MAX_ATTEND_FLOPS = 7.5e10
MAX_MOVED = 32 * 8 * 8192              # largest layers * B * kv heads * context of an eviction


def attend(name, dtype, nh, nkv, d, batch, drafted, ctx, room, weights=False, shared=True):
    return dict(name=name, kind="attend", dtype=dtype, nh=nh, nkv=nkv, d=d, batch=batch, drafted=drafted, ctx=ctx, room=room, weights=weights, shared=shared)


def append(name, dtype, nh, nkv, d, batch, drafted, ctx, room):
    return dict(name=name, kind="append", dtype=dtype, nh=nh, nkv=nkv, d=d, batch=batch, drafted=drafted, ctx=ctx, room=room)


def accept(name, dtype, layers, nkv, d, batch, drafted, path, ctx, weights):
    return dict(name=name, kind="accept", dtype=dtype, layers=layers, nkv=nkv, d=d, batch=batch, drafted=drafted, path=path, ctx=ctx, weights=weights)


def evict(name, dtype, layers, nkv, d, batch, ctx, keep, recent, room):
    return dict(name=name, kind="evict", dtype=dtype, layers=layers, nkv=nkv, d=d, batch=batch, ctx=ctx, keep=keep, recent=recent, room=room)


def listed():
    return [
        # one token of one short conversation, 7B: the smallest attention
        attend("decode1_7b", "float16", 32, 32, 128, 1, 1, 500, 64),
        # a decode batch whose cache is to be evicted from: every step adds up its attention weights
        attend("decode16_7b_observe", "float16", 32, 32, 128, 16, 1, 1531, 64, weights=True),
        # trees of 13 drafted tokens, one for each of four conversations, grouped heads, ragged contexts
        attend("tree13_70b", "bfloat16", 64, 8, 128, 4, 13, 8190, 77, shared=False),
        # the largest tree on a long context: 512 query rows share every key, the largest amount of arithmetic
        attend("tree64_70b_long", "float16", 64, 8, 128, 1, 64, 32768, 64),
        # one rank's share of a 70B layer, many long ragged conversations, a short chain of drafts: the largest read
        attend("tree5_shard_long", "bfloat16", 8, 1, 128, 16, 5, 65536, 99),
        # the last 64 tokens of four prompts looking at what was prefilled: what an eviction behind a prefill goes by
        attend("window64_7b_observe", "float16", 32, 32, 128, 4, 64, 1984, 64, weights=True),
        # one drafted token (ordinary decode) of a small batch
        append("append1_7b", "float16", 32, 32, 128, 4, 1, 1000, 64),
        # trees of 32 tokens for a batch
        append("append32_70b", "bfloat16", 64, 8, 128, 32, 32, 2048, 64),
        # one conversation, a few accepted tokens, all layers of 7B
        accept("accept_7b", "float16", 32, 32, 128, 1, 16, 5, 700, False),
        # one rank's share of 70B, a batch, the accumulated weights move along
        accept("accept_shard", "bfloat16", 80, 1, 128, 16, 64, 12, 2000, True),
        # one layer of one conversation down to half
        evict("evict_layer", "float16", 1, 32, 128, 1, 2047, 1024, 256, 64),
        # every layer of a shard after a long prompt: the largest move
        evict("evict_shard_long", "bfloat16", 32, 8, 128, 1, 8192, 2048, 333, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choices(("attend", "observe", "append", "accept", "evict"), (4, 2, 1, 1, 2))[0]
    nh, nkv, d = rng.choice(HEADS)
    dtype = rng.choice(("float16", "bfloat16"))
    batch = _log_int(rng, 1, 64)
    if kind in ("attend", "observe"):
        weights = kind == "observe"
        drafted = 1 if rng.random() < 0.3 else _log_int(rng, 2, 64)
        ctx = min(65536, MAX_ATTEND // (batch * nkv), int(MAX_ATTEND_FLOPS / (4 * batch * drafted * nh * d)))
        case = attend("", dtype, nh, nkv, d, batch, drafted, _log_int(rng, 1, ctx), rng.randint(64, 200), weights, rng.random() < 0.5)
    elif kind == "append":
        case = append("", dtype, nh, nkv, d, batch, _log_int(rng, 1, min(64, 1024 // batch)), _log_int(rng, 1, 4096), rng.randint(64, 200))
    elif kind == "accept":
        layers = _log_int(rng, 1, 80)
        batch = min(batch, max(1, 1024 // (layers * nkv)))
        drafted = _log_int(rng, 4, 64)
        case = accept("", dtype, layers, nkv, d, batch, drafted, rng.randint(2, min(12, drafted - 1)), _log_int(rng, 1, 1500), rng.random() < 0.5)
    else:
        layers = _log_int(rng, 1, 32)
        batch = min(batch, 8)
        ctx = _log_int(rng, 64, max(64, min(32768, MAX_MOVED // (layers * nkv * batch))))
        keep = rng.randint(max(1, ctx // 8), ctx)
        case = evict("", dtype, layers, nkv, d, batch, ctx, keep, rng.randint(0, keep // 2), rng.randint(1, 200))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------------- preparation
def _lengths(case):
    """Contexts of a batch: from ctx down to about half of it, of odd sizes; which sequence has which goes by the seed."""
    ctx, batch = case["ctx"], case["batch"]
    return [max(1, ctx - b * ctx // (2 * batch) - (17 * b) % 29) for b in range(batch)]


def _counts(case):
    """Accepted tokens of a batch: between two and the whole path."""
    return [max(2, case["path"] - b % 4) for b in range(case["batch"])]


def _tree(g, batch, drafted):
    """Random trees: (ancestor bits int64, depth int32), both [batch, drafted]; token 0 is the root."""
    pick = torch.rand(batch, drafted, device="cuda", generator=g)
    parent = (pick * torch.arange(drafted, device="cuda").clamp(min=1)).long()      # of token i: one of 0 .. i - 1
    bits = torch.ones(batch, drafted, dtype=torch.int64, device="cuda")
    depth = torch.zeros(batch, drafted, dtype=torch.int32, device="cuda")
    for i in range(1, drafted):
        up = parent[:, i:i + 1]
        bits[:, i] = bits.gather(1, up)[:, 0] | (-(1 << 63) if i == 63 else 1 << i)
        depth[:, i] = depth.gather(1, up)[:, 0] + 1
    return bits, depth


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, kind, batch, nkv, d = getattr(torch, case["dtype"]), case["kind"], case["batch"], case["nkv"], case["d"]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32 if math.prod(shape) < 1 << 26 else t).to(t)

    order = torch.randperm(batch, device="cuda", generator=g)
    state = dict(kind=kind, lengths=torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order])
    if kind in ("attend", "append"):
        s, nh, cap = case["drafted"], case["nh"], case["ctx"] + case["drafted"] + case["room"]
        state.update(k=normal(batch, nkv, cap, d), v=normal(batch, nkv, cap, d))
        bits, depth = _tree(g, batch, s)
        if kind == "append":
            angle = torch.arange(cap, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
            state.update(qkv=normal(batch * s, (nh + 2 * nkv) * d), cos=angle.cos().float(), sin=angle.sin().float(), nh=nh,
                         positions=state["lengths"][:, None] + depth)
            return state
        # a head that singles some entries out: scores spread by 1.5 and more
        state.update(q=(normal(batch, s, nh, d) * 1.5), tree=bits[0].contiguous() if case["shared"] else bits)
        state["weights"] = torch.rand(batch, nkv, cap, device="cuda", generator=g) if case["weights"] else None
        return state
    cap = case["ctx"] + (case["drafted"] if kind == "accept" else case["room"])
    layers = case["layers"]
    state.update(k=normal(layers, batch, nkv, cap, d), v=normal(layers, batch, nkv, cap, d), weights=None)
    if kind == "evict" or case["weights"]:
        # few entries hold most of the weight
        state["weights"] = torch.rand(layers, batch, nkv, cap, device="cuda", generator=g).log().neg().square()
    state.update(ks=list(state["k"].unbind(0)), vs=list(state["v"].unbind(0)), ws=None if state["weights"] is None else list(state["weights"].unbind(0)))
    if kind == "evict":
        state.update(keep=case["keep"], recent=case["recent"])
        return state
    s, a = case["drafted"], case["path"]
    # the root, then a branch through the tree: drafted tokens of rising index, none where it already lies
    branch = 2 + torch.rand(batch, s - 2, device="cuda", generator=g).argsort(dim=1)[:, :a - 1].sort(dim=1).values
    path = torch.cat((torch.zeros(batch, 1, dtype=torch.int64, device="cuda"), branch), dim=1).int().contiguous()
    state.update(path=path, accepted=torch.tensor(_counts(case), dtype=torch.int32, device="cuda")[order], drafted=s)
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def _calls():
    from flh_b200 import _CUDA
    return _CUDA


def run(state):
    return {"attend": _attend, "append": _append, "accept": _accept, "evict": _evict}[state["kind"]](state)


def _attend(state):
    q, k, v, lengths, tree, weights = (state[n] for n in ("q", "k", "v", "lengths", "tree", "weights"))
    if own:
        out = _calls().tree_attention(q, k, v, lengths, tree=tree, weights=weights)
        return [out] if weights is None else [out, weights]
    b, s, nh, d = q.shape
    nkv, cap = k.shape[1:3]
    rows = q.float().view(b, s, nkv, nh // nkv, d).permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, d)
    scores = (rows @ k.float().transpose(-1, -2) / math.sqrt(d)).view(b, nkv, s, nh // nkv, cap)
    ahead = torch.arange(cap, device=q.device) - lengths[:, None]                                     # [b, cap]; 0 is the first drafted entry
    drafted = (tree.expand(b, s)[:, :, None] >> ahead.clamp(0, s - 1)[:, None, :]) & 1                 # [b, s, cap]
    seen = (ahead < 0)[:, None, :] | ((ahead < s)[:, None, :] & (drafted != 0))
    scores = scores.masked_fill(~seen[:, None, :, None, :], -torch.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p.view(b, nkv, -1, cap) @ v.float()).view(b, nkv, s, nh // nkv, d).permute(0, 2, 1, 3, 4).reshape(b, s, nh, d).to(q.dtype)
    return [out] if weights is None else [out, weights.add_(p.sum((2, 3)))]


def _append(state):
    qkv, cos, sin, positions, lengths, k, v, nh = (state[n] for n in ("qkv", "cos", "sin", "positions", "lengths", "k", "v", "nh"))
    if own:
        return [_calls().rope_kv_at(qkv, cos, sin, positions, lengths, k, v, nh), k, v]
    b, s = positions.shape
    nkv, d = k.shape[1], k.shape[3]
    x = qkv.view(b, s, nh + 2 * nkv, d)
    c, n = cos[positions.long()][:, :, None], sin[positions.long()][:, :, None]
    x1, x2 = x[:, :, :nh + nkv, :d // 2].float(), x[:, :, :nh + nkv, d // 2:].float()
    turned = torch.cat((x1 * c - x2 * n, x2 * c + x1 * n), dim=-1).to(qkv.dtype)
    at = (lengths[:, None] + torch.arange(s, device=k.device)).long()[:, None, :, None].expand(b, nkv, s, d)
    k.scatter_(2, at, turned[:, :, nh:].transpose(1, 2))
    v.scatter_(2, at, x[:, :, nh + nkv:].transpose(1, 2))
    return [turned[:, :, :nh].contiguous(), k, v]


def _accept(state):
    k, v, weights, lengths, path, accepted, s = (state[n] for n in ("k", "v", "weights", "lengths", "path", "accepted", "drafted"))
    if own:
        now = _calls().cache_accept(state["ks"], state["vs"], lengths, path, accepted, s, weights=state["ws"])
        return [now, k, v] if weights is None else [now, k, v, weights]
    b, a = path.shape
    i = torch.arange(s, device=k.device)
    taken = i < accepted[:, None]                                                                      # [b, s]
    source = torch.where(taken, torch.nn.functional.pad(path, (0, s - a)), i)                          # where drafted entry i comes from
    here, there = lengths[:, None] + i, lengths[:, None] + source

    def moved(x, fill):
        tail = (1,) * (x.dim() - 4)
        at = [t.long().view(1, b, 1, s, *tail).expand(x.shape[:3] + (s,) + x.shape[4:]) for t in (here, there)]
        rows = x.gather(3, at[1])
        x.scatter_(3, at[0], rows if fill is None else torch.where(taken.view(1, b, 1, s), rows, fill))

    moved(k, None), moved(v, None)
    now = lengths + accepted
    if weights is None:
        return [now, k, v]
    moved(weights, 0.0)
    return [now, k, v, weights]


def _evict(state):
    k, v, weights, lengths, keep, recent = (state[n] for n in ("k", "v", "weights", "lengths", "keep", "recent"))
    if own:
        kept, left, now = _calls().cache_evict(state["ks"], state["vs"], state["ws"], lengths, keep, recent)
        return [kept, left, now, k, v]
    cap, d = k.shape[3:]
    j = torch.arange(cap, device=k.device)
    now = lengths.clamp(max=keep)
    n = lengths[:, None, None]                                                                         # [b, 1, 1] against [layers, b, heads, cap]
    rank = weights.masked_fill(j >= n - recent, torch.inf).masked_fill(j >= n, -torch.inf)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    valid = torch.arange(keep, device=k.device) < now[:, None, None]
    kept = best.masked_fill(~valid, cap).sort(dim=-1).values
    at = kept.clamp(max=cap - 1)
    left = torch.zeros_like(weights)
    left[..., :keep] = weights.gather(3, at).masked_fill(~valid, 0.0)
    wide = at[..., None].expand(at.shape + (d,))
    k[..., :keep, :] = torch.where(valid[..., None], k.gather(3, wide), k[..., :keep, :])
    v[..., :keep, :] = torch.where(valid[..., None], v.gather(3, wide), v[..., :keep, :])
    return [kept.masked_fill(~valid, -1).int(), left, now, k, v]


# ---------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "accept": _exact_accept, "evict": _exact_evict}[state["kind"]](state)


def _exact_attend(state):
    q, k, v, tree, weights = (state[n] for n in ("q", "k", "v", "tree", "weights"))
    b, s, nh, d = q.shape
    nkv = k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    total = None if weights is None else weights.double()
    every = [[(int(w) >> j) & 1 for j in range(s)] for w in tree.reshape(-1).tolist()]
    for i, n in enumerate(state["lengths"].tolist()):
        rows_of = every if tree.dim() == 1 else every[i * s:(i + 1) * s]
        mask = torch.ones(s, n + s, dtype=torch.bool, device=q.device)
        mask[:, n:] = torch.tensor(rows_of, device=q.device) != 0
        for h in range(nkv):
            heads = slice(h * (nh // nkv), (h + 1) * (nh // nkv))
            x = torch.einsum("shd,td->hst", q[i, :, heads].double(), k[i, h, :n + s].double()) * d ** -0.5
            p = torch.softmax(x.masked_fill(~mask, float("-inf")), dim=-1)
            out[i, :, heads] = torch.einsum("hst,td->shd", p, v[i, h, :n + s].double())
            if total is not None:
                total[i, h, :n + s] += p.sum((0, 1))
    return [out] if total is None else [out, total]


def _exact_append(state):
    qkv, positions, k, v, nh = (state[n] for n in ("qkv", "positions", "k", "v", "nh"))
    b, s = positions.shape
    nkv, d = k.shape[1], k.shape[3]
    q, k, v = torch.empty(b, s, nh, d, dtype=torch.float64, device=k.device), k.double(), v.double()
    for i, n in enumerate(state["lengths"].tolist()):
        x = qkv[i * s:(i + 1) * s].double().view(s, nh + 2 * nkv, d)
        z = torch.complex(x[..., :d // 2], x[..., d // 2:])
        where = positions[i].long()
        z = z[:, :nh + nkv] * torch.complex(state["cos"][where].double(), state["sin"][where].double())[:, None]
        x[:, :nh + nkv] = torch.cat((z.real, z.imag), dim=-1)
        q[i], k[i, :, n:n + s], v[i, :, n:n + s] = x[:, :nh], x[:, nh:nh + nkv].transpose(0, 1), x[:, nh + nkv:].transpose(0, 1)
    return [q, k, v]


def _exact_accept(state):
    k, v, weights, s = (state[n] for n in ("k", "v", "weights", "drafted"))
    ends = []
    for i, (n, a, path) in enumerate(zip(state["lengths"].tolist(), state["accepted"].tolist(), state["path"].tolist())):
        from_ = [n + p for p in path[:a]]
        for x in (k, v) if weights is None else (k, v, weights):
            x[:, i, :, n:n + a] = x[:, i][:, :, from_]
        if weights is not None:
            weights[:, i, :, n + a:n + s] = 0
        ends.append(n + a)
    now = torch.tensor(ends, dtype=torch.int32, device=k.device)
    return [now, k, v] if weights is None else [now, k, v, weights]


def _exact_evict(state):
    k, v, weights, keep, recent = (state[n] for n in ("k", "v", "weights", "keep", "recent"))
    layers, b, nkv, cap, _ = k.shape
    kept = torch.full((layers, b, nkv, keep), -1, dtype=torch.int32, device=k.device)
    left, ends = torch.zeros_like(weights), []
    for i, n in enumerate(state["lengths"].tolist()):
        m = min(n, keep)
        late = list(range(max(0, n - recent), n))[-m:]
        # the heaviest of the others, the lower index first among equals
        by_weight = torch.sort(-weights[:, i, :, :n - len(late)].double(), dim=-1, stable=True).indices[..., :m - len(late)]
        rows = torch.cat((by_weight, torch.tensor(late, dtype=torch.int64, device=k.device).expand(layers, nkv, len(late))), dim=-1).sort(dim=-1).values
        kept[:, i, :, :m] = rows.int()
        for y in range(layers):
            for h in range(nkv):
                left[y, i, h, :m] = weights[y, i, h, rows[y, h]]
                k[y, i, h, :m], v[y, i, h, :m] = k[y, i, h, rows[y, h]], v[y, i, h, rows[y, h]]
        ends.append(m)
    return [kept, left, torch.tensor(ends, dtype=torch.int32, device=k.device), k, v]


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, batch, nkv, d = case["kind"], case["batch"], case["nkv"], case["d"]
    lengths = _lengths(case)
    if kind == "attend":
        rows, entries = case["drafted"] * case["nh"], sum(n + case["drafted"] for n in lengths)
        side = batch * (4 + 8 * case["drafted"]) + (8 * nkv * entries if case["weights"] else 0)
        return {"bytes": 2 * 2 * nkv * d * entries + 2 * 2 * batch * rows * d + side, "flops": 4 * rows * d * entries}
    if kind == "append":
        tokens, heads = batch * case["drafted"], case["nh"] + 2 * nkv
        return {"bytes": 2 * 2 * tokens * heads * d + tokens * (4 * d + 4) + 4 * batch, "flops": 3 * tokens * (case["nh"] + nkv) * d}
    heads = case["layers"] * nkv
    if kind == "accept":
        moved = sum(a - 1 for a in _counts(case))                       # the root lies where it belongs
        side = heads * (8 * moved + 4 * (batch * case["drafted"] - sum(_counts(case)))) if case["weights"] else 0
        return {"bytes": 2 * 2 * 2 * heads * moved * d + side + 4 * batch * (case["path"] + 3), "flops": 0}
    cap, kept = case["ctx"] + case["room"], sum(min(n, case["keep"]) for n in lengths)
    # weights read; what is kept of them, its indices and the rows behind it written; rows that stay where they are counted as moved
    moved = sum(case["keep"] for n in lengths if n > case["keep"])
    return {"bytes": heads * (4 * sum(lengths) + 4 * batch * cap + 4 * batch * case["keep"] + 2 * 2 * 2 * moved * d) + 8 * batch, "flops": heads * (sum(lengths) + kept)}
