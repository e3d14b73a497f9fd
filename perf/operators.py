"""Performance cases of what stands between the quantized linears of a decoder layer: the rotation of queries and keys, the key-value
cache with its 4- and 8-bit forms, and the attention of one new token over it.

A case is a plain dict; `path` says which work it is:

  rotate   queries and keys of `tokens` tokens: each head divided by its root mean square and weighted (`norm`), then rotated by the angle of
           the token's position; `backward` adds the gradients of both inputs (and of the weights)
  cache    keys and values of `tokens` tokens written into a paged cache and read back
  read     keys and values of `tokens` tokens read back from a cache that holds them
  attend   one new token of each of `batch` sequences against the cache, up to `length` cached tokens each (`ragged`: most have fewer, some none)
  step     rotate, write and attend of one new token of each sequence, as a decode step calls them

`bits` 16 is a cache in `dtype` itself; 8 and 4 are asymmetric codes with a float16 scale and zero point for every `group` values of a head.
"""
import functools

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # One token of a Llama-2-7B layer into an 8-bit cache and back: latency of two calls is all there is.
        {"name": "cache-one-token-w8", "path": "cache", "tokens": 1, "kv_heads": 32, "dim": 128, "bits": 8, "group": 64, "page": 16, "dtype": "float16"},
        # A prompt of an odd length, 8 key-value heads (Llama-3-8B), 4 bits in small groups, small pages.
        {"name": "cache-prompt-w4", "path": "cache", "tokens": 2047, "kv_heads": 8, "dim": 128, "bits": 4, "group": 32, "page": 16, "dtype": "bfloat16"},
        # A long document written in one go.
        {"name": "cache-document-w8", "path": "cache", "tokens": 32768, "kv_heads": 8, "dim": 128, "bits": 8, "group": 128, "page": 64, "dtype": "float16"},
        # A shared prefix read back for a prompt's own attention: 12 heads of 64 (OPT-125m).
        {"name": "read-prefix-w4", "path": "read", "tokens": 12289, "kv_heads": 12, "dim": 64, "bits": 4, "group": 64, "page": 32, "dtype": "float16"},
        # The attention of the repository's decoder benchmark: one sequence, 32 heads, just over 512 cached tokens.
        {"name": "attend-one-513", "path": "attend", "batch": 1, "length": 513, "heads": 32, "kv_heads": 32, "dim": 128, "bits": 16, "group": 0, "page": 64, "dtype": "float16"},
        # One sequence with a very long 4-bit cache.
        {"name": "attend-one-65537-w4", "path": "attend", "batch": 1, "length": 65537, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 4, "group": 128, "page": 64, "dtype": "float16"},
        # A serving batch of mixed lengths over an 8-bit cache.
        {"name": "attend-48-ragged-w8", "path": "attend", "batch": 48, "length": 4001, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "group": 64, "page": 16, "dtype": "bfloat16"},
        # Many short sequences on a small model.
        {"name": "attend-128-short", "path": "attend", "batch": 128, "length": 300, "ragged": True, "heads": 12, "kv_heads": 12, "dim": 64, "bits": 16, "group": 0, "page": 16, "dtype": "float16"},
        # The largest: 64 sequences of up to 8192 tokens, 16-bit cache.
        {"name": "attend-64-ragged-8192", "path": "attend", "batch": 64, "length": 8192, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 16, "group": 0, "page": 32, "dtype": "bfloat16"},
        # One token's queries and keys, no norm (Llama-2-7B).
        {"name": "rotate-one-token", "path": "rotate", "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 128, "rotary": 128, "norm": False, "dtype": "float16"},
        # A training sequence with head norms, forward and backward.
        {"name": "rotate-train-2048", "path": "rotate", "tokens": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "norm": True, "backward": True, "dtype": "bfloat16"},
        # A decode step of 16 sequences: rotation, cache write and attention, one after the other.
        {"name": "step-16", "path": "step", "batch": 16, "length": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "norm": False, "bits": 16, "group": 0, "page": 32, "dtype": "float16"},
    ]


#: Values of keys (or of values) that the largest listed case attends to: no drawn case has more.
_ROOM = 30 * 8192 * 8 * 128


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    path = rng.choice(["attend"] * 5 + ["cache"] * 2 + ["read"] + ["rotate"] * 2 + ["step"] * 2)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 12, 32])
    case = {"path": path, "dim": dim, "kv_heads": kv, "dtype": rng.choice(["float16", "bfloat16"])}
    if path != "rotate":
        bits = 16 if path == "step" or dim == 80 else rng.choice([16, 8, 8, 4, 4])
        group = 0 if bits == 16 else rng.choice([g for g in (32, 64, 128) if dim % g == 0])
        case.update(bits=bits, group=group, page=rng.choice([16, 32, 64, 128]))
    if path in ("attend", "step", "rotate"):
        case["heads"] = kv * rng.choice([g for g in (1, 2, 4, 5, 8, 16) if kv * g <= 64])
    if path in ("attend", "step"):
        length = _log(rng, 1, min(65536, _ROOM // (kv * dim)) if path == "attend" else 4096)
        batch = min(_log(rng, 1, 128), max(1, min((30 if path == "attend" else 8) * 8192, _ROOM // (kv * dim)) // length))
        case.update(batch=batch, length=length, ragged=batch > 1 and rng.random() < 0.7)
    else:
        case["tokens"] = _log(rng, 1, min(32768, _ROOM // 8 // (kv * dim)) if path != "rotate" else 8192)
    if path in ("rotate", "step"):
        case.update(norm=rng.random() < 0.5, rotary=rng.choice([dim, dim, dim // 2]))
    if path == "rotate":
        case["backward"] = rng.random() < 0.5
    return case


def _lengths(case):
    """Cached tokens of each sequence: `length` each, or spread over 1 ... length with every sixteenth sequence idle (a padded batch)."""
    n, most = case["batch"], case["length"]
    if not case.get("ragged"):
        return [most] * n
    spread = [1 + int((most - 1) * ((0.37 + 0.6180339887 * b) % 1.0)) for b in range(n)]
    spread[0] = most
    return [0 if case["path"] == "attend" and b % 16 == 15 else spread[b] for b in range(n)]


# ---- plain forms -------------------------------------------------------------------------------------------------------------


def _codes(x, bits, group):
    """Codes (int32) and (scale, zero point) of every group: scale = the range of the group's values and zero over 2^bits - 1, the difference
    and the quotient rounded to float32, then up to float16; zero point and codes the nearest whole numbers, ties to even.  In 64 bits next to
    those borders."""
    top = 2 ** bits - 1
    g = x.double().unflatten(-1, (x.shape[-1] // group, group))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    step = ((hi - lo).float().double() / torch.full_like(lo, top)).float().clamp(max=65504.0)
    scale = step.half()
    scale = torch.where(scale.float() < step, (scale.view(torch.int16) + 1).view(torch.float16), scale)
    scale = torch.where(scale == 0, torch.full_like(scale, 2.0 ** -24), scale)
    zero = torch.round(-lo / scale.double()).clamp(0, top)
    codes = (torch.round(g / scale.double()[..., None]) + zero[..., None]).clamp(0, top)
    return codes.flatten(-2).to(torch.int32), torch.stack([scale, zero.half()], -1)


def _pack(codes, bits):
    shifts = torch.arange(0, 32, bits, device=codes.device, dtype=torch.int32)
    return (codes.unflatten(-1, (-1, 32 // bits)) << shifts).sum(-1, dtype=torch.int64).to(torch.int32)


def _unpack(words, bits):
    shifts = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shifts) & (2 ** bits - 1)).flatten(-2)


def _write(state, x, words, meta):
    page, row = state["slots"] // state["page"], state["slots"] % state["page"]
    if state["bits"] == 16:
        words[page, :, row] = x
        return
    codes, pairs = _codes(x, state["bits"], state["group"])
    words[page, :, row] = _pack(codes, state["bits"])
    meta[page, :, :, row] = pairs


def _values(words, pairs, bits, group):
    """scale (q - zero) in float32 of packed rows [..., words] with pairs [..., groups, 2]."""
    if bits == 16:
        return words.float()
    q = _unpack(words, bits).float().unflatten(-1, (-1, group))
    return ((q - pairs[..., 1:].float()) * pairs[..., :1].float()).flatten(-2)


def _read(state, words, meta):
    page, row = state["slots"] // state["page"], state["slots"] % state["page"]
    return _values(words[page, :, row], None if meta is None else meta[page, :, :, row], state["bits"], state["group"]).to(state["dtype"])


def _cached(state, words, meta):
    """Every sequence's cached rows as float32 [batch, kv_heads, rows, dim], by its page table."""
    table = state["table"].clamp(min=0)
    rows = words[table]                                                             # [batch, pages, kv_heads, page, words]
    pairs = None if meta is None else meta[table].transpose(3, 4)                   # [batch, pages, kv_heads, page, groups, 2]
    return _values(rows, pairs, state["bits"], state["group"]).transpose(1, 2).flatten(2, 3)


def _attend(state, q):
    k, v = (_cached(state, state[n], state[n[:-1] + "_meta"]) for n in ("keys", "values"))
    batch, heads, dim = q.shape
    kv = k.shape[1]
    seen = (torch.arange(k.shape[2], device=q.device) < state["lengths"][:, None])[:, None, None, :]
    scores = torch.matmul(q.float().view(batch, kv, heads // kv, dim), k.transpose(2, 3).contiguous()) * dim ** -0.5
    scores = torch.where(seen, scores, torch.full_like(scores, float("-inf")))
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - top), torch.zeros_like(scores))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(seen.transpose(2, 3), v, torch.zeros_like(v))) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(batch, heads, dim).to(q.dtype)


def _rotated(x, cos, sin, weight, eps):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.float()
    half = cos.shape[-1]
    a, b = y[..., :half], y[..., half:2 * half]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1).to(x.dtype)


def _rotated_grad(g, x, cos, sin, weight, eps):
    """Gradients of x and of the weight: the rotation turned back, then the norm's."""
    half = cos.shape[-1]
    g = g.float()
    a, b = g[..., :half], g[..., half:2 * half]
    c, s = cos[:, None], sin[:, None]
    g = torch.cat([a * c + b * s, b * c - a * s, g[..., 2 * half:]], -1)
    if weight is None:
        return g.to(x.dtype), None
    y = x.float()
    r = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    n = y * r
    gw = g * weight.float()
    return (r * (gw - n * (gw * n).mean(-1, keepdim=True))).to(x.dtype), (g * n).sum((0, 1)).to(weight.dtype)


def _rotate(state):
    cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
    pairs = [(state["q"], state["q_weight"]), (state["k"], state["k_weight"])]
    out = [_rotated(x, cos, sin, w, state["eps"]) for x, w in pairs]
    if "grads" in state:
        back = [_rotated_grad(g, x, cos, sin, w, state["eps"]) for g, (x, w) in zip(state["grads"], pairs)]
        out += [b[0] for b in back] + [b[1] for b in back if b[1] is not None]
    return out


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _keys(gen, rows, kv_heads, dim, dtype):
    """Keys as a layer projects them: a few channels of every head lie far from zero."""
    x = torch.randn(rows, kv_heads, dim, device="cuda", generator=gen)
    offset = torch.randn(kv_heads, dim, device="cuda", generator=gen)
    return (x + torch.where(offset.abs() > 1.8, 2 * offset, torch.zeros_like(offset))).to(dtype)


def _table(gen, rows, rotary, top):
    """cos and sin of the positions below `top` (float32, formed in 64 bits), and a position for each of `rows` tokens."""
    half = rotary // 2
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(half, device="cuda", dtype=torch.float64) / half)
    return angle.cos().float(), angle.sin().float(), torch.randint(0, top, (rows,), device="cuda", generator=gen)


def _empty_cache(state, case, pages):
    kv, page, dim, bits = case["kv_heads"], case["page"], case["dim"], case["bits"]
    for name in ("key", "value"):
        if bits == 16:
            state[name + "s"], state[name + "_meta"] = torch.zeros(pages, kv, page, dim, device="cuda", dtype=state["dtype"]), None
        else:
            state[name + "s"] = torch.zeros(pages, kv, page, dim * bits // 32, device="cuda", dtype=torch.int32)
            state[name + "_meta"] = torch.zeros(pages, kv, dim // case["group"], page, 2, device="cuda", dtype=torch.float16)


def _filled(state, case, gen, rows):
    """New keys and values into the state's slots, some at a time."""
    slots, chunk = state["slots"], max(1, (1 << 24) // (case["kv_heads"] * case["dim"]))
    for at in range(0, rows, chunk):
        state["slots"] = slots[at:at + chunk]
        n = state["slots"].shape[0]
        _write(state, _keys(gen, n, case["kv_heads"], case["dim"], state["dtype"]), state["keys"], state["key_meta"])
        _write(state, torch.randn(n, case["kv_heads"], case["dim"], device="cuda", generator=gen).to(state["dtype"]), state["values"], state["value_meta"])
    state["slots"] = slots


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, path, kv, dim = DTYPES[case["dtype"]], case["path"], case["kv_heads"], case["dim"]
    state = {"path": path, "dtype": dtype, "bits": case.get("bits"), "group": case.get("group"), "page": case.get("page")}
    if path in ("cache", "read"):
        rows = case["tokens"]
        pages = -(-rows // case["page"])
        pages += pages // 4 + 1
        _empty_cache(state, case, pages)
        # whole pages in an order of their own
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(rows, device="cuda")
        state["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        if path == "read":
            _filled(state, case, gen, rows)
        else:
            # keys and values are parts of one projection's rows
            fused = torch.empty(rows, 2 * kv, dim, device="cuda", dtype=dtype)
            fused[:, :kv] = _keys(gen, rows, kv, dim, dtype)
            fused[:, kv:] = torch.randn(rows, kv, dim, device="cuda", generator=gen).to(dtype)
            state["k"], state["v"] = fused[:, :kv], fused[:, kv:]
    if path in ("attend", "step"):
        lengths = _lengths(case)
        counts = [-(-n // case["page"]) for n in lengths]
        pages = sum(counts) + 1
        _empty_cache(state, case, pages)
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        table = torch.full((len(lengths), max(1, max(counts))), -1, device="cuda", dtype=torch.int32)
        at, slots = 0, []
        for b, (n, c) in enumerate(zip(lengths, counts)):
            table[b, :c] = order[at:at + c]
            rows = torch.arange(n, device="cuda")
            slots.append(order[at:at + c].long()[rows // case["page"]] * case["page"] + rows % case["page"])
            at += c
        state["table"], state["lengths"] = table, torch.tensor(lengths, device="cuda", dtype=torch.int32)
        state["slots"] = torch.cat(slots)
        _filled(state, case, gen, int(state["slots"].shape[0]))
        state["q"] = torch.randn(len(lengths), case["heads"], dim, device="cuda", generator=gen).to(dtype)
    if path in ("rotate", "step"):
        rows = case["tokens"] if path == "rotate" else case["batch"]
        state["cos"], state["sin"], state["positions"] = _table(gen, rows, case["rotary"], 8192)
        state["q"] = torch.randn(rows, case["heads"], dim, device="cuda", generator=gen).to(dtype)
        state["k"] = _keys(gen, rows, kv, dim, dtype)
        state["eps"] = 1e-6
        for name in ("q_weight", "k_weight"):
            state[name] = (1 + 0.2 * torch.randn(dim, device="cuda", generator=gen)).to(dtype) if case["norm"] else None
        if case.get("backward"):
            state["grads"] = [torch.randn(x.shape, device="cuda", generator=gen).to(dtype) for x in (state["q"], state["k"])]
            state["leaves"] = [state["q"], state["k"]] + ([state["q_weight"], state["k_weight"]] if case["norm"] else [])
            for x in state["leaves"]:
                x.requires_grad_(True)
    if path == "step":
        # the new token is the last of its sequence
        state["positions"] = (state["lengths"] - 1).long()
        state["slots"] = torch.stack([s[-1] for s in slots])
        state["v"] = torch.randn(case["batch"], kv, dim, device="cuda", generator=gen).to(dtype)
    return state


@functools.cache
def _package():
    import bitween_amd
    return bitween_amd


def _own(state):
    bw, path = _package(), state["path"]
    if path in ("rotate", "step"):
        q, k = bw.rotate_heads(state["q"], state["k"], state["cos"], state["sin"], state["positions"], state["q_weight"], state["k_weight"], state["eps"])
        if path == "rotate":
            if "grads" not in state:
                return [q, k]
            return [q.detach(), k.detach(), *torch.autograd.grad([q, k], state["leaves"], state["grads"])]
    cache = (state["keys"], state["values"], state["key_meta"], state["value_meta"], state["bits"], state["group"])
    if path == "attend":
        return bw.cache_attention(state["q"], state["table"], state["lengths"], *cache)
    if path == "step":
        bw.write_cache(k, state["v"], state["slots"], *cache)
        return [bw.cache_attention(q, state["table"], state["lengths"], *cache), state["keys"], state["values"]]
    if path == "cache":
        bw.write_cache(state["k"], state["v"], state["slots"], *cache)
    return bw.read_cache(state["slots"], *cache, state["dtype"])


def run(state):
    if own:
        return _own(state)
    path = state["path"]
    with torch.no_grad():
        if path == "rotate":
            return _rotate(state)
        if path == "attend":
            return _attend(state, state["q"])
        if path == "step":
            q, k = _rotate(state)
            _write(state, k, state["keys"], None)
            _write(state, state["v"], state["values"], None)
            return [_attend(state, q), state["keys"], state["values"]]
        if path == "cache":
            _write(state, state["k"], state["keys"], state["key_meta"])
            _write(state, state["v"], state["values"], state["value_meta"])
        return [_read(state, state["keys"], state["key_meta"]), _read(state, state["values"], state["value_meta"])]


def work(case):
    """Each input read once, each output written once; 2 flops for every product and sum of the attention, about 8 (12 with the norm) for every
    rotated value and direction, about 6 for every quantized one."""
    path, dim, kv = case["path"], case["dim"], case["kv_heads"]
    total = flops = 0
    if path != "rotate":
        row = 2 * kv * (dim * case["bits"] // 8 + (4 * (dim // case["group"]) if case["group"] else 0))      # a token's key and value in the cache
    if path in ("rotate", "step"):
        rows = case["tokens"] if path == "rotate" else case["batch"]
        values, passes = rows * (case["heads"] + kv) * dim, 2 if case.get("backward") else 1
        total += 2 * values * 2 + rows * (case["rotary"] * 4 + 8) + (4 * dim if case["norm"] else 0)
        flops += values * (12 if case["norm"] else 8) * passes
        if case.get("backward"):                              # the incoming gradients and the inputs' own; where there is a norm, its inputs are read already
            total += 2 * values * 2 + (4 * dim if case["norm"] else 0)
    if path in ("cache", "read"):
        rows = case["tokens"]
        total += rows * (8 + 4 * kv * dim) + rows * row
        flops += rows * 2 * kv * dim * 2
        if path == "cache":
            total += rows * (4 * kv * dim + 8) + rows * row
            flops += rows * 2 * kv * dim * 6
    if path in ("attend", "step"):
        tokens = sum(_lengths(case))
        total += tokens * row + case["batch"] * (2 * 2 * case["heads"] * dim + 4) + 4 * sum(-(-n // case["page"]) for n in _lengths(case))
        flops += 4 * tokens * case["heads"] * dim
        if path == "step":
            total += case["batch"] * (2 * 2 * kv * dim + row + 8)
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------


def _stored(x, bits, group, dtype):
    """What a cache of `bits` gives back for x, by the definition: numpy on the host, with the roundings that the format has and no others."""
    import numpy as np
    if bits == 16:
        return x
    top = 2 ** bits - 1
    a = x.double().cpu().numpy()
    shape = a.shape
    a = a.reshape(-1, group)
    lo, hi = np.minimum(a.min(1), 0.0), np.maximum(a.max(1), 0.0)
    step = np.minimum(((hi - lo).astype(np.float32) / np.float32(top)), np.float32(65504))
    near = step.astype(np.float16)
    scale = np.where(near.astype(np.float32) < step, np.nextafter(near, np.float16(np.inf)), near)
    scale = np.maximum(scale, np.float16(2.0 ** -24)).astype(np.float64)[:, None]
    zero = np.minimum(np.rint(-lo[:, None] / scale), top)
    q = np.minimum(np.maximum(np.rint(a / scale) + zero, 0), top)
    return torch.from_numpy((scale * (q - zero)).reshape(shape)).to(x.device)


def _turned(x, cos, sin, weight, eps):
    """Pairs (x_i, x_{i + half}) as complex numbers times e^{i angle}, in 64 bits."""
    half = cos.shape[-1]
    y = x.double()
    if weight is not None:
        y = weight.double() * y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    z = torch.complex(y[..., :half], y[..., half:2 * half]) * torch.complex(cos.double(), sin.double())[:, None]
    return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)


def exact(case, seed):
    state = prepare(case, seed)
    path = case["path"]
    if path == "rotate" or path == "step":
        cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
        leaves = [None if state[n] is None else state[n].detach().double().requires_grad_("grads" in state) for n in ("q", "k", "q_weight", "k_weight")]
        out = [_turned(x, cos, sin, w, state["eps"]) for x, w in zip(leaves[:2], leaves[2:])]
        if path == "rotate":
            if "grads" not in state:
                return out
            back = torch.autograd.grad(out, [x for x in leaves if x is not None], [g.double() for g in state["grads"]])
            return [o.detach() for o in out] + list(back)
    if path in ("cache", "read"):
        if path == "cache":
            return [_stored(state[n], case["bits"], case["group"], state["dtype"]).double() for n in ("k", "v")]
        return [_rows(state, case, n, state["slots"]) for n in ("key", "value")]
    if path == "step":                                        # what lies between the operators is held in the inputs' own type
        q, k = (x.to(state["dtype"]) for x in out)
        page, row = state["slots"] // case["page"], state["slots"] % case["page"]
        state["keys"][page, :, row] = k
        state["values"][page, :, row] = state["v"]
    else:
        q = state["q"]
    kv, share = case["kv_heads"], case["heads"] // case["kv_heads"]
    result = torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        at = torch.arange(n, device=q.device)
        slots = state["table"][b].long()[at // case["page"]] * case["page"] + at % case["page"]
        k, v = (_rows(state, case, name, slots).transpose(0, 1) for name in ("key", "value"))      # [kv, n, dim]
        w = torch.softmax((k @ q[b].double().view(kv, share, -1).transpose(1, 2).contiguous()) / case["dim"] ** 0.5, dim=1)
        result[b] = (w.transpose(1, 2).contiguous() @ v.contiguous()).reshape(case["heads"], -1)
    return [result, state["keys"].double(), state["values"].double()] if path == "step" else result


def _rows(state, case, name, slots):
    """Rows of the cache in 64 bits, by arithmetic on whole numbers: [rows, kv_heads, dim]."""
    words, meta, bits = state[name + "s"], state[name + "_meta"], case["bits"]
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    flat = (slots // page)[:, None] * kv * page + torch.arange(kv, device=slots.device) * page + (slots % page)[:, None]
    rows = words.reshape(-1, words.shape[-1])[flat]
    if bits == 16:
        return rows.double()
    unsigned = rows.to(torch.int64) % (1 << 32)
    at = torch.arange(dim, device=slots.device)
    q = unsigned[..., at * bits // 32] // (1 << (at * bits % 32)) % (1 << bits)
    groups = dim // case["group"]
    place = ((slots // page)[:, None, None] * kv + torch.arange(kv, device=slots.device)[:, None]) * groups + torch.arange(groups, device=slots.device)
    pairs = meta.reshape(-1, 2)[place * page + (slots % page)[:, None, None]].double()
    return (q.unflatten(-1, (groups, case["group"])) - pairs[..., 1:]).mul(pairs[..., :1]).flatten(-2)
