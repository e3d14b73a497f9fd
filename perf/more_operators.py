"""Performance cases of what a decoder layer with positions of several axes, a sliding window or a prompt of its own needs beside its
quantized linears.

A case is a plain dict; `path` says which work it is:

  axes     rotation of queries and keys of `tokens` tokens whose position has a number for each of `sections` (time, height, width; pairs of a
           head for each, in order or `interleaved`), with the norm of each head (`norm`); `backward` adds the gradients
  append   queries, keys and values of `tokens` tokens: queries and keys rotated, keys and values into their rows of a paged cache.  What the
           rows hold then is read back where they are codes
  window   one new token of each of `batch` sequences against the last `window` tokens of its cache and the first `sinks`, up to `length` cached
           tokens each (`ragged`: most have fewer, some none).  Pages that neither reaches have been given back
  prompt   causal attention of many tokens of each sequence: `tokens` new ones, each over the `window` tokens up to its own (0: all) and the first
           `sinks`; `prefix` tokens of the sequence come before them; `ragged`: the tokens are those of several sequences, one behind the other;
           `backward` adds the gradients

`bits` 16 is a cache in `dtype` itself; 8 and 4 are asymmetric codes with a float16 scale and zero point for every `group` values of a head.
"""
import functools

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # An image's patches in a prompt, by time, height and width.
        {"name": "axes-image-1024", "path": "axes", "tokens": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "sections": "16,24,24", "interleaved": False, "norm": False, "dtype": "float16"},
        # A training sequence of video frames with head norms, forward and backward.
        {"name": "axes-train-4095", "path": "axes", "tokens": 4095, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "sections": "24,20,20", "interleaved": True, "norm": True, "backward": True, "dtype": "bfloat16"},
        # One token of a Llama-2-7B layer into a 16-bit cache: latency is all there is.
        {"name": "append-one-token", "path": "append", "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 128, "rotary": 128, "sections": "", "norm": False, "bits": 16, "group": 0, "page": 64, "dtype": "float16"},
        # A serving batch's new tokens into an 8-bit cache, with head norms.
        {"name": "append-64-w8", "path": "append", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "sections": "", "norm": True, "bits": 8, "group": 64, "page": 32, "dtype": "bfloat16"},
        # A long prompt with images into a 4-bit cache of small groups.
        {"name": "append-prompt-w4", "path": "append", "tokens": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "sections": "16,24,24", "norm": False, "bits": 4, "group": 32, "page": 16, "dtype": "float16"},
        # One very long sequence that sees its last 4096 tokens and four sinks.
        {"name": "window-one-131072", "path": "window", "batch": 1, "length": 131072, "window": 4096, "sinks": 4, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 16, "group": 0, "page": 64, "dtype": "bfloat16"},
        # A serving batch of mixed lengths over an 8-bit cache; pages end inside the window.
        {"name": "window-48-ragged-w8", "path": "window", "batch": 48, "length": 16001, "ragged": True, "window": 2000, "sinks": 20, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "group": 64, "page": 16, "dtype": "bfloat16"},
        # Many sequences of a small model with a short window over 4 bits.
        {"name": "window-128-short-w4", "path": "window", "batch": 128, "length": 3000, "ragged": True, "window": 500, "sinks": 1, "heads": 12, "kv_heads": 12, "dim": 64, "bits": 4, "group": 64, "page": 32, "dtype": "float16"},
        # The prompt of the repository's decoder benchmark, and one token more.
        {"name": "prompt-513", "path": "prompt", "tokens": 513, "prefix": 0, "window": 0, "sinks": 0, "heads": 32, "kv_heads": 32, "dim": 128, "dtype": "float16"},
        # A long prompt with a window and sinks.
        {"name": "prompt-8192-window", "path": "prompt", "tokens": 8192, "prefix": 0, "window": 1024, "sinks": 4, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bfloat16"},
        # The next few tokens of a long prompt that is fed in pieces: few rows, a long axis.
        {"name": "prompt-chunk-63", "path": "prompt", "tokens": 63, "prefix": 32000, "window": 0, "sinks": 0, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "float16"},
        # The largest: training on documents packed one behind the other, forward and backward.
        {"name": "train-packed-8192", "path": "prompt", "tokens": 8192, "prefix": 0, "ragged": True, "window": 0, "sinks": 0, "heads": 32, "kv_heads": 8, "dim": 128, "backward": True, "dtype": "bfloat16"},
    ]


#: No drawn case has more than the largest listed one: scores that its plain form holds, bytes and operations.
_SCORES, _BYTES, _FLOPS = 32 * 8192 * 8192, 335_000_000, 500_000_000_000


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _sections(rng, half, interleaved=False):
    """Pairs of two, three or four axes, in whatever shares; interleaved ones come from each axis in turn as long as it has some, then from the first."""
    n = rng.choice([2, 3, 3, 4])
    if interleaved:
        rest = [rng.randint(1, half // n) for _ in range(n - 1)]
        return ",".join(map(str, [half - sum(rest)] + rest))
    cuts = sorted(rng.sample(range(1, half), n - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [half]))


def draw(rng):
    path = rng.choice(["axes"] * 2 + ["append"] * 3 + ["window"] * 3 + ["prompt"] * 5)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 12, 32])
    case = {"path": path, "dim": dim, "kv_heads": kv, "heads": kv * rng.choice([g for g in (1, 2, 4, 5, 8, 16) if kv * g <= 64]), "dtype": rng.choice(["float16", "bfloat16"])}
    if path in ("append", "window"):
        bits = 16 if dim == 80 else rng.choice([16, 8, 8, 4, 4])
        group = 0 if bits == 16 else rng.choice([g for g in (32, 64, 128) if dim % g == 0])
        case.update(bits=bits, group=group, page=rng.choice([16, 32, 64, 128]))
    if path in ("axes", "append"):
        rotary = rng.choice([dim, dim, dim // 2])
        case.update(tokens=_log(rng, 1, 4095 if path == "axes" else 8191), rotary=rotary, norm=rng.random() < 0.5)
        case["interleaved"] = path == "axes" and rng.random() < 0.4
        case.update(sections=_sections(rng, rotary // 2, case["interleaved"]) if path == "axes" or rng.random() < 0.5 else "")
    if path == "axes":
        case["backward"] = rng.random() < 0.5
    if path == "window":
        window = _log(rng, 1, 4096)
        batch = min(_log(rng, 1, 128), max(1, 48 * 2000 * 1024 // (window * kv * dim)))
        case.update(batch=batch, length=_log(rng, max(1, window // 2), 16 * window), ragged=batch > 1 and rng.random() < 0.7, window=window, sinks=rng.choice([0, 1, 4, 33]))
    if path == "prompt":
        case.update(tokens=_log(rng, 1, 8192), prefix=0 if rng.random() < 0.6 else _log(rng, 1, 32000), ragged=False,
                    window=_log(rng, 1, 4096) if rng.random() < 0.5 else 0, sinks=rng.choice([0, 0, 1, 4, 33]), backward=rng.random() < 0.5)
        while case["heads"] * case["tokens"] * (case["tokens"] + case["prefix"]) > _SCORES or work(case)["flops"] > _FLOPS:
            case.update(tokens=(case["tokens"] + 1) // 2, prefix=case["prefix"] // 2)
        case["ragged"] = case["prefix"] == 0 and case["tokens"] >= 16 and rng.random() < 0.5
    while work(case)["bytes"] > _BYTES:
        case.update({n: (case[n] + 1) // 2 for n in ("tokens", "prefix", "batch") if n in case})
    return case


def _lengths(case):
    """Cached tokens of each sequence: `length` each, or spread over 1 ... length with every sixteenth sequence idle (a padded batch)."""
    n, most = case["batch"], case["length"]
    if not case.get("ragged"):
        return [most] * n
    spread = [1 + int((most - 1) * ((0.37 + 0.6180339887 * b) % 1.0)) for b in range(n)]
    spread[0] = most
    return [0 if b % 16 == 15 else spread[b] for b in range(n)]


def _seen(case, n):
    """Which of n cached tokens a new one sees: (sinks, the first of the window)."""
    return min(case["sinks"], n), max(0, n - case["window"])


def _documents(case):
    """Lengths of the sequences that the tokens are cut into: a long one, a short one, one of middle length and so on."""
    left, out, share = case["tokens"], [], [0.42, 0.03, 0.2, 0.11, 0.17, 0.01]
    if not case.get("ragged"):
        return [left]
    while left:
        out.append(min(left, 1 + int(case["tokens"] * share[len(out) % len(share)])))
        left -= out[-1]
    return out


def _axis_of(sections, half, interleaved):
    """The axis of each of a head's pairs."""
    counts = [int(s) for s in sections.split(",")] if sections else [half]
    if not interleaved:
        return [a for a, n in enumerate(counts) for _ in range(n)]
    n = len(counts)
    return [i % n if i < n * counts[i % n] else 0 for i in range(half)]


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


def _read(state, slots, words, meta):
    """Rows of the cache in float32, [..., kv_heads, dim]."""
    page, row = slots // state["page"], slots % state["page"]
    return _values(words[page, :, row], None if meta is None else meta[page, :, :, row], state["bits"], state["group"])


def _angles(state):
    """cos and sin of every pair of every token, [tokens, half]: pair i turns by the position on its own axis."""
    if state["axis"] is None:
        return state["cos"][state["positions"]], state["sin"][state["positions"]]
    at = state["positions"][state["axis"]].transpose(0, 1)                          # [tokens, half]
    column = torch.arange(at.shape[1], device=at.device)
    return state["cos"][at, column], state["sin"][at, column]


def _normed(x, weight, eps):
    """Each head over its root mean square, which is formed in 64 bits: what a value is next to a code's border hangs on its last bit."""
    y = x.float()
    if weight is None:
        return y
    return y * torch.rsqrt((x.double() * x.double()).mean(-1, keepdim=True) + eps).float() * weight.float()


def _rotated(x, cos, sin, weight, eps):
    y = _normed(x, weight, eps)
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


def _axes(state):
    cos, sin = _angles(state)
    pairs = [(state["q"], state["q_weight"]), (state["k"], state["k_weight"])]
    out = [_rotated(x, cos, sin, w, state["eps"]) for x, w in pairs]
    if "grads" in state:
        back = [_rotated_grad(g, x, cos, sin, w, state["eps"]) for g, (x, w) in zip(state["grads"], pairs)]
        out += [b[0] for b in back] + [b[1] for b in back if b[1] is not None]
    return out


def _append(state):
    cos, sin = _angles(state)
    q = _rotated(state["q"], cos, sin, state["q_weight"], state["eps"])
    _write(state, _rotated(state["k"], cos, sin, state["k_weight"], state["eps"]), state["keys"], state["key_meta"])
    _write(state, state["v"], state["values"], state["value_meta"])
    if state["bits"] == 16:
        return [q, state["keys"], state["values"]]
    return [q] + [_read(state, state["slots"], state[n + "s"], state[n + "_meta"]).to(q.dtype) for n in ("key", "value")]


def _softmax(scores, seen):
    """Weights of each row's seen scores (none seen: zeros)."""
    top = torch.where(seen, scores, torch.full_like(scores, -3.0e38)).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - top), torch.zeros_like(scores))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _window(state):
    """Only the sinks' and the window's rows are gathered."""
    q, lengths, table = state["q"], state["lengths"].long()[:, None], state["table"]
    batch, heads, dim = q.shape
    first = torch.arange(state["sinks"], device=q.device)[None].expand(batch, -1)
    last = lengths - state["window"] + torch.arange(state["window"], device=q.device)
    at = torch.cat([first, last], 1)                                                # [batch, sinks + window]
    seen = torch.cat([first < lengths, last >= state["sinks"]], 1)
    page = table.gather(1, torch.where(seen, at // state["page"], torch.zeros_like(at))).long()
    slots = torch.where(seen, page * state["page"] + at % state["page"], torch.zeros_like(at))
    k, v = (_read(state, slots, state[n + "s"], state[n + "_meta"]).transpose(1, 2) for n in ("key", "value"))          # [batch, kv_heads, rows, dim]
    kv = k.shape[1]
    scores = torch.matmul(q.float().view(batch, kv, heads // kv, dim), k.transpose(2, 3).contiguous()) * dim ** -0.5
    seen = seen[:, None, None, :]
    p = _softmax(scores, seen)
    out = torch.matmul(p, torch.where(seen.transpose(2, 3), v, torch.zeros_like(v)).contiguous())
    return out.reshape(batch, heads, dim).to(q.dtype)


def _visible(state):
    """[new tokens, tokens]: which a new token sees."""
    at, of, k_at, k_of = state["at"][:, None], state["of"][:, None], state["k_at"][None], state["k_of"][None]
    seen = (of == k_of) & (k_at <= at)
    if state["window"]:
        seen = seen & ((k_at > at - state["window"]) | (k_at < state["sinks"]))
    return seen


def _prompt(state):
    q, k, v = (state[n].float().transpose(0, 1) for n in "qkv")                     # [heads, tokens, dim]
    heads, tokens, dim = q.shape
    kv, scale = k.shape[0], dim ** -0.5
    q = q.reshape(kv, -1, dim)                                                      # a key head's query heads, one behind the other
    k, v = k.contiguous(), v.contiguous()
    seen = _visible(state).repeat(heads // kv, 1)[None]
    p = _softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * scale, seen)
    out = torch.matmul(p, v)

    def rows(x, n, like):
        return x.reshape(n, -1, dim).transpose(0, 1).to(like.dtype).contiguous()
    result = rows(out, heads, state["q"])
    if "grad" not in state:
        return result
    g = state["grad"].float().transpose(0, 1).reshape(kv, -1, dim)
    dv = torch.matmul(p.transpose(1, 2).contiguous(), g)
    ds = p * (torch.matmul(g, v.transpose(1, 2).contiguous()) - (g * out).sum(-1, keepdim=True)) * scale
    return [result, rows(torch.matmul(ds, k), heads, state["q"]), rows(torch.matmul(ds.transpose(1, 2).contiguous(), q), kv, state["k"]), rows(dv, kv, state["v"])]


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _keys(gen, rows, kv_heads, dim, dtype):
    """Keys as a layer projects them: a few channels of every head lie far from zero."""
    x = torch.randn(rows, kv_heads, dim, device="cuda", generator=gen)
    offset = torch.randn(kv_heads, dim, device="cuda", generator=gen)
    return (x + torch.where(offset.abs() > 1.8, 2 * offset, torch.zeros_like(offset))).to(dtype)


def _table(rotary, top):
    """cos and sin of the positions below `top` (float32, formed in 64 bits)."""
    half = rotary // 2
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(half, device="cuda", dtype=torch.float64) / half)
    return angle.cos().float(), angle.sin().float()


def _empty_cache(state, case, pages):
    kv, page, dim, bits = case["kv_heads"], case["page"], case["dim"], case["bits"]
    for name in ("key", "value"):
        if bits == 16:
            state[name + "s"], state[name + "_meta"] = torch.zeros(pages, kv, page, dim, device="cuda", dtype=state["dtype"]), None
        else:
            state[name + "s"] = torch.zeros(pages, kv, page, dim * bits // 32, device="cuda", dtype=torch.int32)
            state[name + "_meta"] = torch.zeros(pages, kv, dim // case["group"], page, 2, device="cuda", dtype=torch.float16)


def _filled(state, case, gen):
    """New keys and values into the state's slots, some at a time."""
    slots, chunk = state["slots"], max(1, (1 << 24) // (case["kv_heads"] * case["dim"]))
    for at in range(0, slots.shape[0], chunk):
        state["slots"] = slots[at:at + chunk]
        n = state["slots"].shape[0]
        _write(state, _keys(gen, n, case["kv_heads"], case["dim"], state["dtype"]), state["keys"], state["key_meta"])
        _write(state, torch.randn(n, case["kv_heads"], case["dim"], device="cuda", generator=gen).to(state["dtype"]), state["values"], state["value_meta"])
    state["slots"] = slots


def _prepare_heads(state, case, gen):
    rows, kv, dim, dtype, sections = case["tokens"], case["kv_heads"], case["dim"], state["dtype"], case["sections"]
    state["cos"], state["sin"] = _table(case["rotary"], 8192)
    state["sections"], state["interleaved"] = tuple(int(s) for s in sections.split(",")) if sections else None, bool(case.get("interleaved"))
    state["axis"] = torch.tensor(_axis_of(sections, case["rotary"] // 2, state["interleaved"]), device="cuda") if sections else None
    shape = (len(state["sections"]), rows) if sections else (rows,)
    state["positions"] = torch.randint(0, 8192, shape, device="cuda", generator=gen)
    # parts of one projection's rows
    fused = torch.empty(rows, case["heads"] + 2 * kv, dim, device="cuda", dtype=dtype)
    fused[:, :case["heads"]] = torch.randn(rows, case["heads"], dim, device="cuda", generator=gen)
    fused[:, case["heads"]:-kv] = _keys(gen, rows, kv, dim, dtype)
    fused[:, -kv:] = torch.randn(rows, kv, dim, device="cuda", generator=gen)
    state["q"], state["k"], state["v"] = fused[:, :case["heads"]], fused[:, case["heads"]:-kv], fused[:, -kv:]
    state["eps"] = 1e-6
    for name in ("q_weight", "k_weight"):
        state[name] = (1 + 0.2 * torch.randn(dim, device="cuda", generator=gen)).to(dtype) if case["norm"] else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, path, kv, dim = DTYPES[case["dtype"]], case["path"], case["kv_heads"], case["dim"]
    state = {"path": path, "dtype": dtype, "bits": case.get("bits"), "group": case.get("group"), "page": case.get("page"), "window": case.get("window"), "sinks": case.get("sinks")}
    if path in ("axes", "append"):
        _prepare_heads(state, case, gen)
    if path == "axes" and case.get("backward"):
        state["q"], state["k"] = state["q"].contiguous(), state["k"].contiguous()
        state["grads"] = [torch.randn(x.shape, device="cuda", generator=gen).to(dtype) for x in (state["q"], state["k"])]
        state["leaves"] = [state["q"], state["k"]] + ([state["q_weight"], state["k_weight"]] if case["norm"] else [])
        for x in state["leaves"]:
            x.requires_grad_(True)
    if path == "append":
        pages = -(-case["tokens"] // case["page"])
        pages += pages // 4 + 1
        _empty_cache(state, case, pages)
        # whole pages in an order of their own
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(case["tokens"], device="cuda")
        state["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
    if path == "window":
        lengths, page = _lengths(case), case["page"]
        columns = []                                             # the pages that a sequence still has, by their place in its table
        for n in lengths:
            sinks, first = _seen(case, n)
            columns.append(sorted(set(range(-(-sinks // page))) | set(range(first // page, -(-n // page)))) if n else [])
        pages = sum(map(len, columns)) + 1
        _empty_cache(state, case, pages)
        order = torch.randperm(pages, device="cuda", generator=gen)
        table = torch.full((len(lengths), max(1, max(-(-n // page) for n in lengths))), -1, device="cuda", dtype=torch.int32)
        used = 0
        for b, c in enumerate(columns):
            if c:
                table[b, torch.tensor(c, device="cuda")] = order[used:used + len(c)].to(torch.int32)
            used += len(c)
        state["slots"] = (order[:used, None] * page + torch.arange(page, device="cuda")).flatten()
        _filled(state, case, gen)
        state["table"], state["lengths"] = table, torch.tensor(lengths, device="cuda", dtype=torch.int32)
        state["q"] = torch.randn(len(lengths), case["heads"], dim, device="cuda", generator=gen).to(dtype)
    if path == "prompt":
        documents, tokens, prefix = _documents(case), case["tokens"], case["prefix"]
        state["q"] = torch.randn(tokens, case["heads"], dim, device="cuda", generator=gen).to(dtype)
        state["k"] = _keys(gen, prefix + tokens, kv, dim, dtype)
        state["v"] = torch.randn(prefix + tokens, kv, dim, device="cuda", generator=gen).to(dtype)
        sizes = torch.tensor(documents, device="cuda")
        starts = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), sizes.cumsum(0)])
        state["starts"] = starts.to(torch.int32) if case.get("ragged") else None
        # what the plain form masks by: every token's sequence and its place there
        of = torch.repeat_interleave(torch.arange(len(documents), device="cuda"), sizes)
        place = torch.arange(tokens, device="cuda") - starts[of]
        state["of"], state["at"] = of, place + prefix
        state["k_of"] = torch.cat([torch.zeros(prefix, device="cuda", dtype=torch.int64), of])
        state["k_at"] = torch.cat([torch.arange(prefix, device="cuda"), place + prefix])
        if case.get("backward"):
            state["grad"] = torch.randn(tokens, case["heads"], dim, device="cuda", generator=gen).to(dtype)
            state["leaves"] = [state[n].requires_grad_(True) for n in "qkv"]
    return state


@functools.cache
def _package():
    import bitween_amd
    return bitween_amd


def _own(state):
    bw, path = _package(), state["path"]
    if path == "axes":
        q, k = bw.rotate_heads(state["q"], state["k"], state["cos"], state["sin"], state["positions"], state["q_weight"], state["k_weight"], state["eps"],
                               sections=state["sections"], interleaved=state["interleaved"])
        if "grads" not in state:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], state["leaves"], state["grads"])]
    if path == "prompt":
        out = bw.prompt_attention(state["q"], state["k"], state["v"], state["starts"], window=state["window"] or None, sinks=state["sinks"])
        if "grad" not in state:
            return out
        return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["grad"])]
    cache = (state["keys"], state["values"], state["key_meta"], state["value_meta"], state["bits"], state["group"])
    if path == "window":
        return bw.cache_attention(state["q"], state["table"], state["lengths"], *cache, window=state["window"], sinks=state["sinks"])
    q = bw.append_cache(state["q"], state["k"], state["v"], state["cos"], state["sin"], state["positions"], state["slots"], *cache,
                        q_weight=state["q_weight"], k_weight=state["k_weight"], eps=state["eps"], sections=state["sections"])
    if state["bits"] == 16:
        return [q, state["keys"], state["values"]]
    return [q, *bw.read_cache(state["slots"], *cache, state["dtype"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"axes": _axes, "append": _append, "window": _window, "prompt": _prompt}[state["path"]](state)


def _pairs(case):
    """Scores of one query head that the prompt needs."""
    total = 0
    for n in _documents(case):
        first, last = case["prefix"], case["prefix"] + n                            # positions of its new tokens
        total += n * (first + last + 1) // 2                                        # ... each with itself and all before it
        window, sinks = case["window"], case["sinks"]
        if window:                                                                  # without those between the sinks and the window
            hidden = [max(0, p - window + 1 - sinks) for p in (first, last - 1)]
            m = min(n, hidden[1])                                                   # tokens that miss some: 1, 2, ... or a run of these
            total -= m * (hidden[1] + hidden[1] - m + 1) // 2
    return total


def work(case):
    """Each input read once, each output written once; 2 flops for every product and sum of the attention (5 products of a training step for the forward's
    2), about 8 (12 with the norm) for every rotated value and direction, about 6 for every quantized one."""
    path, dim, kv = case["path"], case["dim"], case["kv_heads"]
    total = flops = 0
    if path in ("append", "window"):
        row = 2 * kv * (dim * case["bits"] // 8 + (4 * (dim // case["group"]) if case["group"] else 0))      # a token's key and value in the cache
    if path in ("axes", "append"):
        rows, axes = case["tokens"], max(1, len(case["sections"].split(",")))
        values, passes = rows * (case["heads"] + kv) * dim, 2 if case.get("backward") else 1
        total += rows * (case["rotary"] * 4 + 8 * axes) + (4 * dim if case["norm"] else 0)
        flops += values * (12 if case["norm"] else 8) * passes
        if path == "axes":
            total += 2 * values * 2
            if case.get("backward"):                          # the incoming gradients and the inputs' own; where there is a norm, its inputs are read already
                total += 2 * values * 2 + (4 * dim if case["norm"] else 0)
        else:                                                 # queries in and out, keys and values in and into the cache; codes are read back
            total += rows * (2 * 2 * case["heads"] * dim + 2 * 2 * kv * dim + row + 8)
            if case["bits"] != 16:
                total += rows * (row + 2 * 2 * kv * dim + 8)
                flops += rows * 2 * kv * dim * 8
    if path == "window":
        for n in _lengths(case):
            sinks, first = _seen(case, n)
            tokens = n - max(0, first - sinks)
            total += tokens * row + 4 * -(-tokens // case["page"])
            flops += 4 * tokens * case["heads"] * dim
        total += case["batch"] * (2 * 2 * case["heads"] * dim + 4)
    if path == "prompt":
        q, k = case["tokens"] * case["heads"] * dim * 2, (case["tokens"] + case["prefix"]) * kv * dim * 2
        total += 2 * q + 2 * k
        flops += 4 * _pairs(case) * case["heads"] * dim
        if case.get("backward"):                              # the output's gradient comes in, those of q, k and v go out
            total += 2 * q + 2 * k
            flops += 10 * _pairs(case) * case["heads"] * dim
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------


def _stored(x, bits, group):
    """What a cache of `bits` gives back for x, by the definition: numpy on the host, with the roundings that the format has and no others."""
    import numpy as np
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


def _turned(x, angle, weight, eps):
    """Pairs (x_i, x_{i + half}) as complex numbers times e^{i angle}, in 64 bits."""
    half = angle.shape[-1]
    y = x.double()
    if weight is not None:
        y = weight.double() * y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    z = torch.complex(y[..., :half], y[..., half:2 * half]) * angle[:, None]
    return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)


def _exact_heads(case, state):
    half, positions = case["rotary"] // 2, state["positions"]
    angle = torch.empty(case["tokens"], half, device="cuda", dtype=torch.complex128)
    for i, axis in enumerate(_axis_of(case["sections"], half, case.get("interleaved"))):
        at = positions[axis] if case["sections"] else positions
        angle[:, i] = torch.complex(state["cos"][at, i].double(), state["sin"][at, i].double())
    leaves = [None if state[n] is None else state[n].detach().double().requires_grad_("grads" in state) for n in ("q", "k", "q_weight", "k_weight")]
    out = [_turned(x, angle, w, state["eps"]) for x, w in zip(leaves[:2], leaves[2:])]
    if "grads" in state:
        back = torch.autograd.grad(out, [x for x in leaves if x is not None], [g.double() for g in state["grads"]])
        return [o.detach() for o in out] + list(back)
    return out


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


def _exact_window(case, state):
    q, kv, share = state["q"], case["kv_heads"], case["heads"] // case["kv_heads"]
    result = torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        sinks, first = _seen(case, n)
        at = torch.tensor(sorted(set(range(sinks)) | set(range(first, n))), device=q.device)
        slots = state["table"][b].long()[at // case["page"]] * case["page"] + at % case["page"]
        k, v = (_rows(state, case, name, slots).transpose(0, 1) for name in ("key", "value"))      # [kv, rows, dim]
        w = torch.softmax((k @ q[b].double().view(kv, share, -1).transpose(1, 2).contiguous()) / case["dim"] ** 0.5, dim=1)
        result[b] = (w.transpose(1, 2).contiguous() @ v.contiguous()).reshape(case["heads"], -1)
    return result


def _exact_prompt(case, state):
    """Head by head and sequence by sequence, gradients from torch's own differentiation."""
    share, prefix = case["heads"] // case["kv_heads"], case["prefix"]
    leaves = [state[n].detach().double() for n in "qkv"]
    outs = [torch.zeros_like(leaves[0])] + ([torch.zeros_like(t) for t in leaves] if case.get("backward") else [])
    start = 0
    for n in _documents(case):
        new, old = slice(start, start + n), slice(start, start + prefix + n)
        at = prefix + torch.arange(n, device="cuda")[:, None]
        t = torch.arange(prefix + n, device="cuda")[None]
        hidden = t > at
        if case["window"]:
            hidden = hidden | ((t <= at - case["window"]) & (t >= case["sinks"]))
        for h in range(case["heads"]):
            q, k, v = (x[s, i].detach().requires_grad_(len(outs) > 1) for x, s, i in zip(leaves, (new, old, old), (h, h // share, h // share)))
            out = torch.softmax((q @ k.t()).div(case["dim"] ** 0.5).masked_fill(hidden, float("-inf")), -1) @ v
            outs[0][new, h] = out.detach()
            if len(outs) > 1:
                for into, s, i, g in zip(outs[1:], (new, old, old), (h, h // share, h // share), torch.autograd.grad(out, (q, k, v), state["grad"][new, h].double())):
                    into[s, i] += g
        start += n
    return outs if len(outs) > 1 else outs[0]


def exact(case, seed):
    state = prepare(case, seed)
    path = case["path"]
    if path == "axes":
        return _exact_heads(case, state)
    if path == "append":
        q, k = _exact_heads(case, state)
        k = k.to(state["dtype"])                              # a cache is given keys in the inputs' own type
        if case["bits"] != 16:
            return [q] + [_stored(x, case["bits"], case["group"]) for x in (k, state["v"])]
        page, row = state["slots"] // case["page"], state["slots"] % case["page"]
        state["keys"][page, :, row], state["values"][page, :, row] = k, state["v"]
        return [q, state["keys"].double(), state["values"].double()]
    return _exact_window(case, state) if path == "window" else _exact_prompt(case, state)
