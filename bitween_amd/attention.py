"""What stands between the quantized linears of a decoder layer: rotation of queries and keys (with the norm of each head), a paged
key-value cache that may hold 8- or 4-bit codes, and the attention of one new token over it.

    q, k = rotate_heads(q, k, cos, sin, positions)
    cache.write(k, v, slots)
    out = cache.attend(q, page_table, lengths)

Each is one HIP kernel of libbitween_hip.so (the attention is joined by a second one where a sequence is cut, and so are the gradients of norm
weights); they run on torch's current stream, allocate their outputs and workspaces from its allocator, and can be captured in HIP
graphs.  Cache and attention have no derivatives: under grad mode a tensor that asks for gradients raises, a forward-mode tangent always (for the
rotation too).  There is no CPU path: CPU tensors raise.  The reference has no counterpart; its models bring these as eager torch operations.
"""
import torch
from torch.autograd import forward_ad

from .kernels import hip_loader as _hip

_HALF = (torch.float16, torch.bfloat16)


def _native(name):
    return getattr(_hip.host(), name)


def _tensor(t, what, *dtypes):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if dtypes and t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")


def _whole(t, what, dtype):
    """A tensor of whole numbers, contiguous and in the type that the kernels read."""
    _tensor(t, what)
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise TypeError(f"{what} must hold whole numbers, got {str(t.dtype)[6:]}")
    t = _hip._plain(t)
    if dtype is torch.int32 and t.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
        t = t.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)       # what lies outside stays outside
    return t.to(dtype).contiguous()


def _one_gpu(what, *tensors):
    for t in tensors:
        if t is not None:
            _hip.require_gpu(t, what)
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"{what}: tensors on {', '.join(sorted(map(str, devices)))}; one GPU is wanted")


def _no_tangent(what, *tensors):
    """Forward-mode derivatives are refused, with and without grad mode: a result without its tangent would be wrong without a word."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _hip.BitweenHipError(f"{what} has no forward-mode derivative")


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise _hip.BitweenHipError(f"{what} has no gradient: call it under torch.no_grad(), or on detached tensors")


def _checked_cache(what, keys, values, key_meta, value_meta, bits, group_size):
    """The head dimension of a cache whose tensors fit together."""
    if bits == 2:
        raise NotImplementedError(f"{what}: a cache holds 4, 8 or 16 bits")
    if bits not in (4, 8, 16):
        raise ValueError(f"{what}: a cache holds 4, 8 or 16 bits, got {bits!r}")
    stored = _HALF if bits == 16 else (torch.int32,)
    _tensor(keys, "keys", *stored)
    _tensor(values, "values", *stored)
    if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype or 0 in keys.shape:
        raise ValueError(f"{what}: keys and values must both be [pages, kv_heads, page_size, width] of one type")
    if bits == 16:
        if key_meta is not None or value_meta is not None:
            raise ValueError(f"{what}: a 16-bit cache has no key_meta / value_meta")
        dim, meta = keys.shape[3], ()
    else:
        dim, meta = keys.shape[3] * 32 // bits, (key_meta, value_meta)
        if not isinstance(group_size, int) or group_size < 1 or dim % group_size:
            raise ValueError(f"{what}: group_size {group_size!r} does not divide the head dimension {dim}")
        want = (keys.shape[0], keys.shape[1], dim // group_size, keys.shape[2], 2)
        for t, name in zip(meta, ("key_meta", "value_meta")):
            _tensor(t, name, torch.float16)
            if t.shape != want:
                raise ValueError(f"{what}: {name} must be [pages, kv_heads, dim / group_size, page_size, 2] = {list(want)}, got {list(t.shape)}")
    _one_gpu(what, keys, values, *meta)
    if not all(t.is_contiguous() for t in (keys, values, *meta)):
        raise ValueError(f"{what}: the tensors of a cache must be contiguous")
    return dim


def _cache_args(keys, values, key_meta, value_meta, bits, group_size):
    return tuple(None if t is None else _hip._plain(t) for t in (keys, values, key_meta, value_meta)) + (int(bits), int(group_size))


def _taken(what, out):
    if out is None:
        raise _hip.BitweenHipError(f"{what}: these arguments are not taken")
    return out


def rotate_heads(q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=1e-6):
    """Queries [..., q_heads, dim] and keys [..., k_heads, dim] turned by the angle of their token's position, as two new tensors:

        y = x * rsqrt(mean(x^2) + eps) * weight             (y = x without a weight)
        out_i = y_i cos_i - y_{i+h} sin_i,  out_{i+h} = y_{i+h} cos_i + y_i sin_i   for i < h;   out_i = y_i for i >= 2 h

    cos, sin: float32 [table rows, h], 2 h <= dim; positions: int64 with the leading dimensions of q and k.  A token whose position lies
    outside the table is padding: its outputs are zero and it has no part in gradients.  q_weight, k_weight: [dim] in q's dtype or float32,
    each may be None.  float16 or bfloat16; float32 arithmetic, one rounding.  Gradients of q, k and the weights (sums in a fixed order);
    none of cos and sin, and no second derivatives.  dim and 2 h are multiples of 8, dim up to 256.
    Leading dimensions that are not one stride (a transposed [batch, heads, tokens, dim]) are copied first."""
    out = _native("rotate_heads")(q, k, cos, sin, positions, q_weight, k_weight, eps)
    if out is not None:
        return out
    what = "rotate_heads"
    _tensor(q, "q", *_HALF)
    _tensor(k, "k", q.dtype)
    _tensor(cos, "cos", torch.float32, torch.float16, torch.bfloat16)
    _tensor(sin, "sin", torch.float32, torch.float16, torch.bfloat16)
    _tensor(positions, "positions")
    _one_gpu(what, q, k, cos, sin, positions, q_weight, k_weight)
    if cos.dim() != 2 or cos.shape != sin.shape or 0 in cos.shape:
        raise ValueError("cos and sin must both be [table rows, rotary / 2]")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise NotImplementedError("rotate_heads has no gradient of cos and sin")
    _no_tangent(what, cos, sin)
    for t, name in ((q, "q"), (k, "k")):
        if t.dim() != positions.dim() + 2 or t.shape[:-2] != positions.shape or 0 in t.shape[-2:]:
            raise ValueError(f"{name} must be [..., heads, dim] with the leading dimensions of positions {list(positions.shape)}, got {list(t.shape)}")
    dim = q.shape[-1]
    if k.shape[-1] != dim or 2 * cos.shape[1] > dim:
        raise ValueError(f"q and k must have one head dimension, at least twice the {cos.shape[1]} columns of cos")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        _tensor(w, "q_weight / k_weight", q.dtype, torch.float32)
        if w.shape != (dim,) or w.dtype != weights[0].dtype:
            raise ValueError(f"q_weight and k_weight must be [{dim}] of one type")
    # (a leaf goes on as it is: what a capture asks of its gradient's accumulation is asked of the leaf itself)
    plain = [t if t is None or type(t) in (torch.Tensor, torch.nn.Parameter) else t.as_subclass(torch.Tensor) for t in (q, k, q_weight, k_weight)]
    tables = [t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format) for t in (_hip._plain(t).float() for t in (cos, sin))]
    return _taken(what, _native("rotate_heads")(plain[0], plain[1], *tables, _whole(positions, "positions", torch.int64), plain[2], plain[3], float(eps)))


def write_cache(k, v, slots, keys, values, key_meta=None, value_meta=None, bits=16, group_size=64):
    """Keys and values [tokens, kv_heads, dim] into the rows `slots` (int64 [tokens]) of a paged cache, in place:

        16 bits   keys, values [pages, kv_heads, page_size, dim] float16 or bfloat16 (the type of k and v)
        8, 4      keys, values int32 [pages, kv_heads, page_size, dim * bits / 32], packed as quantize_rtn packs; key_meta, value_meta float16
                  [pages, kv_heads, dim / group_size, page_size, 2]: (scale, zero point) of every group of a head's values

    Slot n is row n % page_size of page n // page_size; a slot outside the cache is left out (padding).  The slots of one call must differ.
    k and v may be rows of the cache itself (they are copied first); keys and values must not share memory.
    A group's range includes zero, its scale is rounded up to float16, so that scale * (code - zero point) is within half a scale of the
    value; a group with an infinity or a NaN reads back as NaN.  dim is a multiple of 8 up to 256, page_size a power of two from 16 to 1024,
    group_size 32, 64 or 128."""
    if _native("cache_write")(k, v, slots, keys, values, key_meta, value_meta, bits, group_size):
        return
    what = "write_cache"
    dim = _checked_cache(what, keys, values, key_meta, value_meta, bits, group_size)
    for t, name in ((k, "k"), (v, "v")):
        _tensor(t, name, *((keys.dtype,) if bits == 16 else _HALF))
        if t.dim() != 3 or t.shape[1:] != (keys.shape[1], dim):
            raise ValueError(f"{name} must be [tokens, {keys.shape[1]}, {dim}], got {list(t.shape)}")
    _tensor(v, "v", k.dtype)
    _tensor(slots, "slots")
    if slots.dim() != 1 or not len(slots) == len(k) == len(v):
        raise ValueError("slots must be [tokens], one for every row of k and v")
    _one_gpu(what, keys, k, v, slots)
    _no_grad(what, k, v, keys, values, key_meta, value_meta)
    _no_tangent(what, k, v, keys, values, key_meta, value_meta)
    for a, b in ((keys, values), (key_meta, value_meta)):
        if a is not None and a.data_ptr() < b.data_ptr() + b.nbytes and b.data_ptr() < a.data_ptr() + a.nbytes:
            raise ValueError(f"{what}: keys and values of a cache that is written must not share memory")
    _taken(what, _native("cache_write")(_hip._plain(k), _hip._plain(v), _whole(slots, "slots", torch.int64),
                                        *_cache_args(keys, values, key_meta, value_meta, bits, group_size)))


def read_cache(slots, keys, values, key_meta=None, value_meta=None, bits=16, group_size=64, dtype=None):
    """The rows `slots` (int64 [tokens]) of a paged cache (see write_cache) as (k, v), both [tokens, kv_heads, dim] of `dtype`: float16 or
    bfloat16; the cache's own type at 16 bits, float16 otherwise where none is given.  Codes come back as scale * (code - zero point),
    rounded once; a slot outside the cache gives zeros."""
    if dtype is None:
        dtype = getattr(keys, "dtype", None) if bits == 16 else torch.float16
    if dtype not in _HALF or (bits == 16 and dtype != getattr(keys, "dtype", None)):
        raise TypeError(f"read_cache gives float16 or bfloat16 (a 16-bit cache its own type), not {dtype}")
    code = _hip._DTYPE_CODE[dtype]
    out = _native("cache_read")(slots, keys, values, key_meta, value_meta, bits, group_size, code)
    if out is not None:
        return out
    _checked_cache("read_cache", keys, values, key_meta, value_meta, bits, group_size)
    _tensor(slots, "slots")
    if slots.dim() != 1:
        raise ValueError("slots must be [tokens]")
    _one_gpu("read_cache", keys, slots)
    _no_grad("read_cache", keys, values, key_meta, value_meta)
    _no_tangent("read_cache", keys, values, key_meta, value_meta)
    return _taken("read_cache", _native("cache_read")(_whole(slots, "slots", torch.int64), *_cache_args(keys, values, key_meta, value_meta, bits, group_size), code))


def cache_attention(q, page_table, lengths, keys, values, key_meta=None, value_meta=None, bits=16, group_size=64, scale=None):
    """Attention of one new token of each sequence over a paged cache (see write_cache): q [batch, q_heads, dim] -> [batch, q_heads, dim],

        out = sum_t softmax_t(scale q . k_t) v_t   over t < lengths[b],

    token t of sequence b in row t % page_size of page page_table[b, t // page_size] (int32 [batch, pages of a sequence]); lengths int32
    [batch], the new token's own row included where it is written first.  kv_heads divides q_heads; query head h reads head
    h // (q_heads // kv_heads).  scale: 1 / sqrt(dim) where none is given.  q has the type of a 16-bit cache, float16 or bfloat16 over codes.

    A sequence of length 0 (an idle row of a padded batch) gives zeros.  What lies behind a sequence's last token is not looked at - neither the
    rows nor the table's entries.  A score of minus infinity (an infinity among the keys) has weight 0, and a sequence without any other score gives NaN, as
    one of plus infinity or NaN does; an infinity or a NaN among the values leaves nothing finite in its channel, whatever its weight.  A length beyond
    the table is cut to it; a page number outside the cache is a page without tokens.  Lengths and table are read on the GPU when the kernel runs, so a
    captured call follows them.  No gradients."""
    if scale is None:
        scale = q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    out = _native("cache_attention")(q, page_table, lengths, keys, values, key_meta, value_meta, bits, group_size, scale)
    if out is not None:
        return out
    what = "cache_attention"
    dim = _checked_cache(what, keys, values, key_meta, value_meta, bits, group_size)
    _tensor(q, "q", *((keys.dtype,) if bits == 16 else _HALF))
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] < 1 or q.shape[1] % keys.shape[1]:
        raise ValueError(f"q must be [batch, a multiple of {keys.shape[1]} heads, {dim}], got {list(q.shape)}")
    _tensor(page_table, "page_table")
    _tensor(lengths, "lengths")
    if page_table.dim() != 2 or page_table.shape[0] != q.shape[0] or page_table.shape[1] < 1 or lengths.shape != q.shape[:1]:
        raise ValueError(f"page_table must be [{q.shape[0]}, pages] and lengths [{q.shape[0]}]")
    _one_gpu(what, keys, q, page_table, lengths)
    _no_grad(what, q, keys, values, key_meta, value_meta)
    _no_tangent(what, q, keys, values, key_meta, value_meta)
    return _taken(what, _native("cache_attention")(_hip._plain(q), _whole(page_table, "page_table", torch.int32), _whole(lengths, "lengths", torch.int32),
                                                   *_cache_args(keys, values, key_meta, value_meta, bits, group_size), float(scale)))


class PagedCache:
    """The tensors of one layer's paged key-value cache and the calls on them.

    pages, page_size: how many pages of how many token rows; bits 16 (in `dtype`), 8 or 4 (codes, a float16 scale and zero point for every
    group_size values of a head).  Which pages a sequence has is the caller's: page_table[b, i] is the page of its tokens i * page_size and up."""

    __slots__ = ("keys", "values", "key_meta", "value_meta", "bits", "group_size", "dtype")

    def __init__(self, pages, kv_heads, head_dim, page_size=64, bits=16, group_size=64, dtype=torch.float16, device="cuda"):
        if bits not in (2, 4, 8, 16):
            raise ValueError("Only 4, 8 or 16 bits are supported.")
        if bits == 2:
            raise NotImplementedError("PagedCache holds 4, 8 or 16 bits")
        if dtype not in _HALF:
            raise TypeError(f"PagedCache: dtype must be float16 or bfloat16, got {dtype}")
        if min(pages, kv_heads, head_dim, page_size) < 1:
            raise ValueError("PagedCache: pages, kv_heads, head_dim and page_size must be at least 1")
        if head_dim % 8 or head_dim > 256 or not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise NotImplementedError("PagedCache: head_dim must be a multiple of 8 up to 256, page_size a power of two from 16 to 1024")
        self.bits, self.group_size, self.dtype = bits, group_size, dtype
        if bits == 16:
            self.keys = torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
            self.values, self.key_meta, self.value_meta = torch.zeros_like(self.keys), None, None
            return
        if group_size < 1 or head_dim % group_size:
            raise ValueError(f"PagedCache: group_size {group_size} does not divide head_dim {head_dim}")
        if group_size not in (32, 64, 128):
            raise NotImplementedError("PagedCache: group_size must be 32, 64 or 128")
        self.keys = torch.zeros(pages, kv_heads, page_size, head_dim * bits // 32, dtype=torch.int32, device=device)
        self.key_meta = torch.zeros(pages, kv_heads, head_dim // group_size, page_size, 2, dtype=torch.float16, device=device)
        self.values, self.value_meta = torch.zeros_like(self.keys), torch.zeros_like(self.key_meta)

    @property
    def page_size(self):
        return self.keys.shape[2]

    def write(self, k, v, slots):
        """write_cache into this cache."""
        write_cache(k, v, slots, self.keys, self.values, self.key_meta, self.value_meta, self.bits, self.group_size)

    def read(self, slots):
        """read_cache of this cache, in its dtype."""
        return read_cache(slots, self.keys, self.values, self.key_meta, self.value_meta, self.bits, self.group_size, self.dtype)

    def attend(self, q, page_table, lengths, scale=None):
        """cache_attention over this cache."""
        return cache_attention(q, page_table, lengths, self.keys, self.values, self.key_meta, self.value_meta, self.bits, self.group_size, scale)

    def slots(self, page_table, positions, sequences=None):
        """The slots (int64) of the tokens at `positions` (int64 [tokens]): of the sequences 0, 1, ... one each, or of `sequences` (int64 [tokens]).
        A position that the table has no page for - a negative one of a padded batch, one behind the last page - has the slot -1: padding."""
        size = self.keys.shape[2]
        if sequences is None:
            if len(positions) != len(page_table):
                raise ValueError(f"positions must be [{len(page_table)}], one for each sequence, where no sequences are given")
            pages = page_table
        else:
            pages = page_table[sequences]
        if pages.shape[1] == 0:                                  # (nothing that could be looked up)
            return torch.full_like(positions, -1, dtype=torch.int64)
        column = positions // size
        kept = (column >= 0) & (column < pages.shape[1])
        page = pages.gather(1, column.clamp(0, pages.shape[1] - 1).long()[:, None])[:, 0].long()
        return torch.where(kept & (page >= 0) & (page < self.keys.shape[0]), page * size + positions % size, -1)
