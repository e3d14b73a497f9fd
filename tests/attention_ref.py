"""64-bit restatements of rotate_heads, the cache's format and cache_attention for the tests, and inputs for them."""
import numpy as np
import torch


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def rotate(x, cos, sin, positions, weight, eps):
    """x [tokens, heads, dim] float64; a position outside the table gives zeros."""
    half, rows = cos.shape[1], cos.shape[0]
    y = x
    if weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight
    inside = (positions >= 0) & (positions < rows)
    at = positions.clamp(0, rows - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
    out = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    return torch.where(inside[:, None, None], out, torch.zeros_like(out))


def quantize(x, bits, group):
    """x float array [..., dim] -> (codes, scale float16, zero point), the format's definition in numpy; the difference and the quotient of the
    range are float32 operations there, the codes those of exact quotients (a float64 quotient of 11-bit numbers rounds to the same whole number)."""
    top = (1 << bits) - 1
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    with np.errstate(over="ignore"):
        step = np.minimum((hi.astype(np.float32) - lo.astype(np.float32)) / np.float32(top), np.float32(65504))
    near = step.astype(np.float16)
    with np.errstate(over="ignore"):                             # (of the branch not taken)
        scale = np.where(near.astype(np.float32) < step, np.nextafter(near, np.float16(np.inf)), near)
    scale = np.maximum(scale, np.float16(2.0 ** -24))
    s = scale.astype(np.float64)
    zero = np.minimum(np.rint(-lo / s), top)
    codes = np.clip(np.rint(g / s[..., None]) + zero[..., None], 0, top)
    scale = np.where(bad, np.float16(np.nan), scale)
    return codes.reshape(x.shape).astype(np.int64), scale, zero


def unpack(words, bits, dim):
    """int32 array [..., dim * bits / 32] -> codes [..., dim]"""
    u = words.astype(np.int64) & 0xFFFFFFFF
    return np.stack([(u >> (i * bits)) & ((1 << bits) - 1) for i in range(32 // bits)], -1).reshape(*words.shape[:-1], dim)


def rows(words, meta, slots, bits, group):
    """float64 [slots, kv_heads, dim] of the cache's rows, on the cache's device."""
    page, row = slots // words.shape[2], slots % words.shape[2]
    w = words[page, :, row]
    if bits == 16:
        return w.double()
    u = w.long() & 0xFFFFFFFF
    codes = torch.stack([(u >> (i * bits)) & ((1 << bits) - 1) for i in range(32 // bits)], -1).flatten(-2)
    pairs = meta[page, :, :, row].double()
    return ((codes.double().unflatten(-1, (-1, group)) - pairs[..., 1:]) * pairs[..., :1]).flatten(-2)


class Batch:
    """A filled cache, page table, lengths and queries.  Unwritten rows hold NaN (16 bits) or random bits with NaN pairs, unused table
    entries a number far outside."""

    def __init__(self, lengths, heads, kv_heads, dim, page, bits, group, dtype, seed=0, spare=2, width=None, spread=1.0, device="cuda"):
        import bitween_amd as bw
        gen = torch.Generator(device=device).manual_seed(seed)
        self.dtype, self.bits, self.group = dtype, bits, group
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        self.cache = bw.PagedCache(pages, kv_heads, dim, page, bits, group, dtype, device)
        c = self.cache
        for t in (c.keys, c.values):
            if bits == 16:
                t.fill_(float("nan"))
            else:
                t.random_(-2 ** 31, 2 ** 31 - 1, generator=gen)
        if bits != 16:
            c.key_meta.fill_(float("nan"))
            c.value_meta.fill_(float("nan"))
        order = torch.randperm(pages, device=device, generator=gen)
        width = width or max(1, max(counts))
        self.table = torch.full((len(lengths), width), 2 ** 30, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.slots, at = [], 0
        for b, (n, m) in enumerate(zip(lengths, counts)):
            self.table[b, :m] = order[at:at + m]
            t = torch.arange(n, device=device)
            self.slots.append(order[at:at + m][t // page] * page + t % page)
            at += m
        total = sum(lengths)
        self.k = (spread * torch.randn(total, kv_heads, dim, device=device, generator=gen)).to(dtype)
        self.v = (0.5 + torch.randn(total, kv_heads, dim, device=device, generator=gen)).to(dtype)
        self.q = torch.randn(len(lengths), heads, dim, device=device, generator=gen).to(dtype)
        if total:
            c.write(self.k, self.v, torch.cat(self.slots))

    def attend(self, scale=None):
        return self.cache.attend(self.q, self.table, self.lengths, scale)

    def check(self, out, scale=None, lengths=None):
        """out against 64 bits.  One rounding of the result; weights of the softmax held to 16 bits or better (2^-16 of their sum times the largest
        value); scores in float32: a sum of dim products, the scaling and the exponential's argument, together at most (dim + 16) 2^-24 of the sum of
        the products' magnitudes, which changes a weight by that much relative to itself.  Over codes a value is the difference scale * code -
        scale * zero point, and it is these two that the weights multiply: an error of 2^-20 of a weight (two float16 numbers, each cut to 11 bits) is
        2^-20 of a group's whole range (2^bits - 1) scale, however near to each other code and zero point are, and sums of 32 products of codes
        are cut by at most 32 * 2^-16 of a unit of 8 bits or 32 * 2^-20 of a unit of 4 bits, 2^-18.9 and 2^-18.9 of the range.  So the largest
        value is the group's largest range there."""
        c = self.cache
        dim, kv = self.q.shape[2], c.keys.shape[1]
        share = self.q.shape[1] // kv
        scale = dim ** -0.5 if scale is None else scale
        for b in range(self.q.shape[0]):
            n = len(self.slots[b]) if lengths is None else lengths[b]
            got = out[b].double()
            if n <= 0:
                assert torch.equal(out[b], torch.zeros_like(out[b])), f"sequence {b} is empty"
                continue
            k, v = (rows(w, m, self.slots[b][:n], self.bits, self.group).transpose(0, 1) for w, m in ((c.keys, c.key_meta), (c.values, c.value_meta)))
            q = self.q[b].double().view(kv, share, dim)
            scores = torch.matmul(k, q.transpose(1, 2).contiguous()) * scale
            weights = torch.softmax(scores, 1).transpose(1, 2).contiguous()
            want = torch.matmul(weights, v.contiguous()).reshape(-1, dim)
            reach = (torch.matmul(k.abs(), q.abs().transpose(1, 2).contiguous()) * abs(scale)).amax(1).reshape(-1, 1)      # of a query head
            top = v.abs().amax(1)
            if self.bits != 16:
                at = self.slots[b][:n]
                pairs = c.value_meta[at // c.page_size, :, :, at % c.page_size].double()
                top = (pairs[..., 0].amax(0) * (2 ** self.bits - 1)).repeat_interleave(self.group, -1)
            top = top.repeat_interleave(share, 0)
            bound = half_step(self.dtype) * want.abs() + (2.0 ** -16 + 2 * (dim + 16) * 2.0 ** -24 * reach) * top + 2.0 ** -25
            worst = ((got - want).abs() / bound).max().item()
            assert worst <= 1, f"sequence {b} of {n} tokens: {worst:.3f} times the bound"
