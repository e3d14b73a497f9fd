"""A 64-bit restatement of prompt_attention and its gradients, with the errors that the arithmetic allows."""
import torch

from attention_ref import half_step


def visible(nq, nk, window, sinks, device="cuda"):
    """[nq, nk]: which of nk tokens the last nq of them see."""
    at = nk - nq + torch.arange(nq, device=device)[:, None]
    t = torch.arange(nk, device=device)[None]
    seen = t <= at
    if window:
        seen = seen & ((t > at - window) | (t < sinks))
    return seen


def head(q, k, v, seen, scale, grad=None):
    """One head: out, its bound, and with the output's gradient those of q, k and v with theirs.  float64 [tokens, dim].

    Bounds, h being half a step of the type: a score is a sum of dim products in float32 with the scaling and the exponential's argument, (dim + 16) 2^-24 of the sum of the products'
    magnitudes, which changes a weight by that much relative to itself, and another score in the sum by which it is divided by as much (twice); sums over n tokens err by
    n 2^-24 of their terms.  A weight is rounded once (h of itself, and in float16 no more than 2^-37 of the largest of its row beside that, the largest being 2^12 at least where
    a step is 2^-24), and so is dS; dP is a sum of dim products; delta a sum of dim products with the rounded output."""
    dtype = q.dtype
    h, dim, n = half_step(dtype), q.shape[1], k.shape[0]
    small = 2.0 ** -37 if dtype == torch.float16 else 0.0
    q, k, v = (x.double() for x in (q, k, v))
    scores = torch.where(seen, q @ k.t() * scale, float("-inf"))
    any_seen = seen.any(-1, keepdim=True)
    p = torch.where(any_seen, torch.softmax(torch.where(any_seen, scores, 0.0), -1), 0.0)
    out = p @ v
    reach = torch.where(seen, (q.abs() @ k.abs().t()) * abs(scale), 0.0).amax(-1, keepdim=True)
    loose = 2 * (dim + 16) * 2.0 ** -24 * reach + 2 * n * 2.0 ** -24          # of a weight, relative
    most = p.amax(-1, keepdim=True)
    seen_v = seen.double() @ v.abs()
    off = h * out.abs() + (h + loose) * (p @ v.abs()) + small * most * seen_v + 2.0 ** -25
    if grad is None:
        return [(out, off)]
    g = grad.double()
    dp = g @ v.t()
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # (2^-36: the smallest step of P, whose exponent begins at 2^12)
    dv, dv_off = p.t() @ g, ((p * (h + loose) + seen.double() * (2.0 ** -36 if small else 0.0)).t() @ g.abs())
    ds_off = h * ds.abs() + p * (loose * (dp - delta).abs() + (dim + 2) * 2.0 ** -23 * (g.abs() @ v.abs().t()) + (g.abs() * off).sum(-1, keepdim=True) + dim * 2.0 ** -23 * (g * out).abs().sum(-1, keepdim=True))
    # (float16: a step of dS's type below the largest of its row or column, 2^12 at least)
    row, column = small * ds.abs().amax(-1, keepdim=True), small * ds.abs().amax(0, keepdim=True)
    dq, dk = scale * (ds @ k), scale * (ds.t() @ q)
    # dQ = scale dS (K - c), c a mean of keys that the row sees (no value of it is larger than the largest of theirs): in 64 bits sum(dS) c is nothing, as a row's dS add up to
    # zero; what they are off by adds up to sum(dS's bounds) at most, and meets c in dQ.
    wrong = (ds_off + row) * seen
    largest = torch.stack([torch.where(s[:, None], k.abs(), 0.0).amax(0) for s in seen]) if n else torch.zeros_like(q)
    dq_off = abs(scale) * (wrong @ k.abs() + wrong.sum(-1, keepdim=True) * largest)
    dk_off = abs(scale) * ((ds_off + column * seen).t() @ q.abs())
    rows = [(out, off)]
    for want, o in ((dq, dq_off), (dk, dk_off), (dv, dv_off)):
        rows.append((want, o + h * want.abs() + 2 * n * 2.0 ** -24 * o + 2.0 ** -25))
    return rows


def reference(q, k, v, spans, window, sinks, scale, grad=None):
    """(value, bound) of out, and of the gradients of q, k and v: tokens packed one behind the other, `spans` (q from, q to, k from, k to) of each sequence."""
    heads, kv = q.shape[1], k.shape[1]
    share = heads // kv
    like = [q] + ([q, k, v] if grad is not None else [])
    total = [(torch.zeros(t.shape, dtype=torch.float64, device=t.device), torch.full(t.shape, 2.0 ** -25, dtype=torch.float64, device=t.device)) for t in like]
    for q0, q1, k0, k1 in spans:
        if q1 == q0:
            continue
        seen = visible(q1 - q0, k1 - k0, window, sinks, q.device)
        for n in range(heads):
            got = head(q[q0:q1, n], k[k0:k1, n // share], v[k0:k1, n // share], seen, scale, None if grad is None else grad[q0:q1, n]) if k1 > k0 else []
            places = ((slice(q0, q1), n), (slice(q0, q1), n), (slice(k0, k1), n // share), (slice(k0, k1), n // share))
            for (value, bound), (want, off), at in zip(total, got, places):
                value[at] += want
                bound[at] += off
    return total


def close(got, want, bound, what):
    worst = ((got.double() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.3f} times the bound"
    return worst
