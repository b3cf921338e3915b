"""64-bit restatements of the operators on a cache that is drafted into and evicted from, with error bounds by arithmetic."""
import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def chain(s):
    """Ancestor bits of a chain of s tokens."""
    return torch.tensor([((1 << (i + 1)) - 1) - (1 << 64 if i == 63 else 0) for i in range(s)], dtype=torch.int64)


def random_tree(r, s):
    """Ancestor bits (int64 [s]) and depth of a random tree whose token 0 is the root."""
    bits, depth = [1], [0]
    for i in range(1, s):
        parent = r.randint(0, i)
        bits.append(bits[parent] | (1 << i))
        depth.append(depth[parent] + 1)
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64), torch.tensor(depth, dtype=torch.int32)


def seen_mask(tree, b, s, n, total):
    """bool [s, total]: what the tokens of sequence b with n committed entries see of its first `total` entries."""
    row = chain(s) if tree is None else (tree if tree.dim() == 1 else tree[b]).cpu()
    seen = torch.zeros(s, total, dtype=torch.bool)
    seen[:, :min(n, total)] = True
    for i in range(s):
        for j in range(s):
            if n + j < total and (int(row[i]) >> j) & 1:
                seen[i, n + j] = True
    return seen


def attention(q, k, v, lengths, tree=None, scale=None):
    """-> out f64, its bound, the weights f64 [B, nkv, T], their bound (to which the rounding of the sum with what was there adds).

    p is off by a relative 2 d: d = 2^-24 for each of the D + 1 products and sums of a score and its scaling, in units of the sum of
    magnitudes, twice (once in the exponent, once in the sum that divides; exp2 itself 2^-21).  The weighted sum takes p rounded to the
    tensors' type: half a step u of each, absolutely at least that of the smallest float16 (2^-25, against a sum of 1 or more).  The
    result is rounded once more."""
    B, S, nh, D = q.shape
    nkv, T = k.shape[1:3]
    g, u = nh // nkv, HALF_STEP[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    w, wtol = (torch.zeros(B, nkv, T, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T)
        total = min(n + S, T)
        seen = seen_mask(tree, b, S, n, total).to(q.device)
        for h in range(nkv):
            qh, kh, vh = q[b, :, h * g:(h + 1) * g].double(), k[b, h, :total].double(), v[b, h, :total].double()
            x = torch.einsum("sgd,td->sgt", qh, kh) * scale
            size = torch.einsum("sgd,td->sgt", qh.abs(), kh.abs()) * scale
            some = seen.any(-1)[:, None, None]
            x = torch.where(seen[:, None], x, -torch.inf)
            p = torch.where(some, torch.softmax(torch.where(some, x, 0.0), -1), 0.0)
            d = torch.where(seen[:, None] & size.isfinite(), size, 0.0).amax(-1, keepdim=True) * (D + 1) * 2.0 ** -24 + 2.0 ** -21
            # a weight of zero on an entry that is not seen adds nothing, whatever lies there
            o, size_o, size_v = (torch.empty(S, g, D, dtype=torch.float64, device=q.device) for _ in range(3))
            for s in range(S):
                at = seen[s].nonzero()[:, 0]
                pv = p[s][:, at, None] * vh[at]
                o[s], size_o[s], size_v[s] = pv.sum(1), pv.abs().sum(1), vh[at].abs().sum(0)
            out[b, :, h * g:(h + 1) * g] = o
            tol[b, :, h * g:(h + 1) * g] = u * o.abs() * 1.01 + (u + 2 * d) * size_o * 1.01 + (2.0 ** -25 * (size_v + 1) if q.dtype == torch.float16 else 0.0) + 1e-30
            w[b, h, :total] = torch.where(seen[:, None], p, 0.0).sum((0, 1))
            wtol[b, h, :total] = (torch.where(seen[:, None], p, 0.0) * (2 * d + (S * g + 2) * 2.0 ** -24)).sum((0, 1)) + 1e-30
    return out, tol, w, wtol


def assert_close(got, want, tol):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan().sum(), want.isnan().sum())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or bool((off <= 0).all()), (float(off.max()), int((off > 0).sum()), off.numel())


def evict(weights, n, keep, recent):
    """Entries of one head (weights float32 numpy [T], n of them) that stay."""
    if n <= keep:
        return np.arange(n)
    w = weights[:n - recent].astype(np.float64)
    w = np.where(np.isnan(w), np.inf, w)
    nan_first = np.lexsort((np.arange(len(w)), ~np.isnan(weights[:n - recent]), -w))     # heaviest first, NaN above +inf, the lower index first
    return np.sort(np.concatenate((nan_first[:keep - recent], np.arange(n - recent, n))))
