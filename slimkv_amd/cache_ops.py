"""Operators over a full-width K/V cache beside its decode: attention for a tree
of drafted tokens, the attention weight that its rows gather, and eviction by it.

    tree_attention     every drafted token over the cached rows and its ancestors
    attention_weights  the weight each cached row gets from a step's queries
    select_rows        the rows that a smaller cache keeps by that weight
    compact_rows       those rows' K, V and weights moved to the front

A cache is given as dense rows k, v [B, N, Hkv, D] or as raw pages
[blocks, block, 2, Hkv, D] (RawPages' format) with a block table [B, cols] int64;
`lengths` [B] int32 are the rows each sequence holds (default: all N).  Element
types bf16 and fp16 (one for all tensors of a call), head_dim 64 or 128, keys
rotated.  Cache rows start on 16-byte boundaries and lie less than 2^23 elements
apart.  Up to 65535 sequences, 4096 query heads, 256 of them a KV head; softmax
scales in [1e-18, 1e18] (zero, negative ones and NaN raise ValueError).

A speculative step over a bounded cache: tree_attention gives the drafted
tokens' outputs and LSEs; the accepted path's K/V rows are appended to the
cache (RawPages.write, kernels.raw_pages); attention_weights adds that path's
attention to the rows' weights; when a sequence passes its budget select_rows
and compact_rows bring it back.  Rows read through a block table follow torch's
indexing rules: an entry outside the pool raises IndexError after the call (one
host synchronisation), or is left in the caller's device int32 `status` word
(graph capture, serving loops; kernels.check_status).  The operators have no
gradients: they raise ValueError where one would be recorded or a forward-mode
tangent lost, and for negative views, whose memory holds other values.
"""
import struct
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib
from .kernels import _status_word, check_status

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_NO_WORKSPACE = 16         # what a query answers for a call that uses none
_CODES = {_lib.c_ptr: 'P', _lib.c_i64: 'q', _lib.c_f64: 'd', _lib.c_i32: 'i'}


def _packer(mirror):
    """The bytes of an argument struct from its field values: one struct.pack, where filling the ctypes mirror field by
    field takes longer than the rest of a call."""
    def codes(s):
        return ''.join(codes(kind) if hasattr(kind, '_fields_') else _CODES[kind] for _, kind in s._fields_)
    layout = struct.Struct(codes(mirror) + '0q')          # '0q': the trailing padding of an 8-byte aligned struct
    assert layout.size == _lib.ctypes.sizeof(mirror)
    return layout.pack


_pack_tree = _packer(_lib.TreeAttentionArgs)
_pack_weights = _packer(_lib.AttentionWeightsArgs)
_pack_select = _packer(_lib.SelectRowsArgs)
_pack_compact = _packer(_lib.CompactRowsArgs)


def _common(name, *tensors):
    """The device that holds every tensor; no gradient to record, no tangent to carry, memory that holds the values."""
    index = lowest = highest = tensors[0].get_device()
    grad, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    for t in tensors:
        if t is None:
            continue
        if t.is_neg():
            raise ValueError(f'{name} reads memory as it is: resolve negative views (resolve_neg)')
        if dual and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name} carries no tangent: detach the inputs')
        if grad and t.requires_grad:
            raise ValueError(f'{name} records no gradient: detach the inputs or run it under torch.no_grad()')
        at = t.get_device()
        if at != index:
            lowest, highest = min(lowest, at), max(highest, at)
    if lowest < 0:
        raise ValueError(f'{name} needs device tensors (no CPU path)')
    if lowest != highest:
        raise ValueError(f'{name}: tensors on devices {lowest} and {highest}')
    return tensors[0].device


def _dtype(name, *tensors):
    kind = tensors[0].dtype
    code = _DTYPES.get(kind)
    for t in tensors:
        if code is None or t is not None and t.dtype is not kind:
            raise ValueError(f'{name}: expected bfloat16 or float16 for every tensor, found '
                             f'{[t.dtype for t in tensors if t is not None]}')
    return code


def _rows16(t):
    """t [B, rows, H, D], or a copy where its rows do not start on 16-byte boundaries, or overlap, or lie far apart."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        st = t.stride()
        if st[3] == 1 and all(n == 1 or s % 8 == 0 for n, s in zip(t.shape, st[:3])) and \
                (t.shape[1] <= 1 or t.shape[3] <= st[1] < 1 << 23):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _span(t):
    """First and last byte address of t's elements."""
    size = t.element_size()
    last = t.numel() - 1 if t.is_contiguous() else sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    start = t.data_ptr()
    return start, start + last * size + size


def _reaches(target, terms, budget):
    """Whether 0 <= x_i <= n_i give sum x_i s_i = target, for terms (s_i, n_i) with s_i falling; true as well where that
    takes more than budget[0] steps to find out."""
    if not terms:
        return target == 0
    (step, most), rest = terms[0], terms[1:]
    reach = sum(s * n for s, n in rest)
    for x in range(max(0, -((reach - target) // step)), min(most, target // step) + 1):
        budget[0] -= 1
        if budget[0] < 0 or _reaches(target - x * step, rest, budget):
            return True
    return False


def _overlap(a, b):
    """Whether a byte belongs to elements of both a and b (views may lie interleaved and apart: the halves of one
    tensor): an element of a at a0 + x and one of b at b0 + y share one if the distance b0 - a0 is a sum of steps of
    both."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    steps = {1: a.element_size() + b.element_size() - 2}
    for t in (a, b):
        for n, s in zip(t.shape, t.stride()):
            if s and n > 1:
                s *= t.element_size()
                steps[s] = steps.get(s, 0) + n - 1
    terms = []
    for s, n in sorted(steps.items()):
        if terms and s % terms[-1][0] == 0 and s // terms[-1][0] <= terms[-1][1] + 1:
            terms[-1] = (terms[-1][0], terms[-1][1] + s // terms[-1][0] * n)      # the steps below reach up to this one
        elif n:
            terms.append((s, n))
    # y counted down from b's last byte, so that all steps add up
    return _reaches(b1 - 1 - a0, terms[::-1], [1000])


def _apart(written, read):
    """Whether no tensor written shares memory with another one (None: not there)."""
    written = [(*_span(t), t) for t in written if t is not None and t.numel()]
    spans = written + [(*_span(t), t) for t in read if t is not None and t.numel()]
    return not any(a0 < b1 and b0 < a1 and _overlap(a, b)
                   for i, (a0, a1, a) in enumerate(written) for b0, b1, b in spans[i + 1:])


def _folded(t):
    """Whether elements of t share memory (expanded views), or its steps do not show that none do: each past all that
    the smaller ones reach."""
    if t.numel() < 2 or t.is_contiguous():
        return False
    reach = 0
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s <= reach:
            return True
        reach += s * (n - 1)
    return False


def _lengths(name, lengths, batch):
    if lengths is None:
        return None
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] != batch:
        raise ValueError(f'{name}: lengths must be int32 [{batch}]')
    return lengths if lengths.is_contiguous() else lengths.contiguous()


def _new(dtype, device, a, b, c):
    """An uninitialised contiguous [a, b, c] (strides given: half torch.empty's time)."""
    return torch.empty_strided((a, b, c), (b * c, c, 1), dtype=dtype, device=device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _status(name, status, device, needed):
    """(status word, owned); no word where nothing can be reported."""
    if status is None:
        if not needed:
            return None, False
        if torch.cuda.is_current_stream_capturing():
            raise ValueError(f'{name} under graph capture needs a caller status word')
    return _status_word(status, device)


def _cache(name, k, v, pages, table, lengths, keys, batch, values=True):
    """A cache as the C struct's values but for the status word: (fields, rows, heads, features, paged, the tensors
    they point into).  k alone where V is not read."""
    if (k is None) == (pages is None):
        raise ValueError(f'{name}: give the cache either as dense rows or as pages with a block table')
    lengths = _lengths(name, lengths, batch)
    if pages is None:
        if table is not None or keys is not None:
            raise ValueError(f'{name}: a block table and keys belong to pages')
        if values and v is None:
            raise ValueError(f'{name}: dense rows need both k and v')
        ks = k.stride()
        if k.dim() != 4 or k.shape[0] != batch or ks[3] != 1:
            raise ValueError(f'{name}: cache rows must be [{batch}, N, Hkv, D] with contiguous features')
        _, rows, heads, dim = k.shape
        vs = (0, 0, 0, 1)
        if values:
            vs = v.stride()
            if v.shape != k.shape or vs[3] != 1:
                raise ValueError(f'{name}: v must have the shape of k with contiguous features')
        fields = (k.data_ptr(), *ks[:3], v.data_ptr() if values else 0, *vs[:3], 0, 0, 0, 0, 0, _ptr(lengths), rows)
        return fields, rows, heads, dim, False, lengths
    if v is not None:
        raise ValueError(f'{name}: pages hold both K and V')
    if pages.dim() != 5 or pages.shape[2] != 2 or pages.stride(4) != 1:
        raise ValueError(f'{name}: pages must be [blocks, block, 2, Hkv, D] with contiguous features')
    if table is None or table.dtype is not torch.int64 or table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f'{name}: pages need an int64 block table [{batch}, cols]')
    if table.stride(1) != 1:
        table = table.contiguous()
    blocks, block, _, heads, dim = pages.shape
    cols = table.shape[1]
    rows = cols * block if keys is None else int(keys)
    if not 0 <= rows <= cols * block:
        raise ValueError(f'{name}: keys must lie in [0, {cols * block}] (cols * block)')
    sb, sn, skind, sh, _ = pages.stride()
    base = pages.data_ptr()
    place = (table.data_ptr(), table.stride(0), cols, blocks, block) if rows else (0, 0, 0, 0, 0)
    fields = (base, sb, sn, sh, base + skind * pages.element_size(), sb, sn, sh, *place, _ptr(lengths), rows)
    return fields, rows, heads, dim, rows > 0, (table, lengths)


def _queries(name, q, heads, dim):
    if q.dim() != 4 or q.shape[3] != dim or q.shape[2] % heads:
        raise ValueError(f'{name}: q must be [B, rows, Hq, {dim}] with Hq a multiple of {heads}')


def _on(device):
    """None where the device is current already, else a guard that makes it so."""
    return None if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _call(device, entry, args, nbytes=None):
    """One entry point on torch's current stream of `device`, whichever device is current, with a workspace of
    `nbytes` where it takes one."""
    guard = _on(device)
    if guard is not None:
        with guard:
            return _call(device, entry, args, nbytes)
    if nbytes is None:
        check(entry(args, _lib.stream_handle(device)))
    elif nbytes <= _NO_WORKSPACE:
        check(entry(args, None, 0, _lib.stream_handle(device)))
    else:
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=device)
        check(entry(args, ws.data_ptr(), nbytes, _lib.stream_handle(device)))


def _asked(entry, a, index):
    with torch.cuda.device(index):
        nbytes = entry(_lib.ctypes.byref(a))
    if nbytes == 0:
        check(-1)
    return nbytes


# The workspace queries go by sizes (and the device) alone: asked once for each.
@lru_cache(1024)
def _tree_bytes(index, B, T, Hq, H, D):
    return _asked(lib().slimkv_tree_attention_workspace, _lib.TreeAttentionArgs(
        q=16, batch=B, drafted=T, heads=Hq, kv_heads=H, head_dim=D, scale=1.0), index)


@lru_cache(1024)
def _weights_bytes(index, B, L, Hq, H, D, keys):
    return _asked(lib().slimkv_attention_weights_workspace, _lib.AttentionWeightsArgs(
        cache=_lib.CacheRows(keys=keys), batch=B, queries=L, heads=Hq, kv_heads=H, head_dim=D, scale=1.0), index)


@lru_cache(1024)
def _select_bytes(index, B, H, keys, keep, sink, recent):
    return _asked(lib().slimkv_select_rows_workspace, _lib.SelectRowsArgs(
        batch=B, heads=H, keys=keys, keep=keep, sink=sink, recent=recent), index)


def tree_attention(q, draft_k, draft_v, scale, k=None, v=None, *, pages=None, table=None, lengths=None, keys=None,
                   mask=None, out=None, lse=None, status=None):
    """Attention of drafted tokens over a cache and over each other.

    q [B, T, Hq, D], draft_k / draft_v [B, T, Hkv, D] (rotated, not yet in the
    cache; T up to 1024); the cache dense or paged (`keys`: the longest
    sequence's rows, default cols * block).  mask [T, T] or [B, T, T] bool:
    drafted token t sees drafted token j where mask[.., t, j] (itself included
    only if so marked); None is a chain (j <= t).  Every token sees all rows of
    its sequence's cache.  Returns (out [B, T, Hq, D], lse [B, Hq, T] fp32); a
    row that sees nothing gives 0 and -inf, and what lies in unseen rows has no
    influence, infinities and NaN included.  T = 1 decodes a single token.
    Softmax weights are rounded to the element type for their product with v
    (half a step of each weight; fp16 ones keep 2^-39 of the row's largest),
    their sum and the LSE are fp32."""
    name = 'tree_attention'
    B = q.shape[0]
    place, rows, H, D, paged, keep = _cache(name, k, v, pages, table, lengths, keys, B)
    first = pages if k is None else k
    code = _dtype(name, q, draft_k, draft_v, first, v, out)
    _queries(name, q, H, D)
    _, T, Hq, _ = q.shape
    draft = (B, T, H, D)
    if draft_k.shape != draft or draft_v.shape != draft:
        raise ValueError(f'{name}: draft_k and draft_v must be [{B}, {T}, {H}, {D}]')
    m = (0, 0, 0)
    if mask is not None:
        if mask.dtype is not torch.bool or mask.shape not in ((T, T), (B, T, T)):
            raise ValueError(f'{name}: mask must be bool [{T}, {T}] or [{B}, {T}, {T}]')
        if mask.stride(-1) != 1:
            mask = mask.contiguous()
        m = (mask.data_ptr(), mask.stride(0) if mask.dim() == 3 else 0, mask.stride(-2))
    inputs = (q, draft_k, draft_v, k, v, pages, table, lengths, mask)
    if out is not None and (out.shape != q.shape or out.stride(3) != 1 or _folded(out) or
                            any(t is not None and _overlap(out, t) for t in inputs)):
        raise ValueError(f'{name}: out must have the shape of q with contiguous features, no expanded view and apart '
                         'from the inputs')
    if lse is not None and (lse.shape != (B, Hq, T) or lse.dtype is not torch.float32 or not lse.is_contiguous() or
                            any(t is not None and _overlap(lse, t) for t in (*inputs, out))):
        raise ValueError(f'{name}: lse must be a contiguous float32 [{B}, {Hq}, {T}], apart from the other tensors')
    device = _common(name, q, draft_k, draft_v, k, v, pages, table, lengths, mask, out, lse)
    q, draft_k, draft_v = _rows16(q), _rows16(draft_k), _rows16(draft_v)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if lse is None:
        lse = _new(torch.float32, device, B, Hq, T)
    status, owned = _status(name, status, device, paged)
    nbytes = _tree_bytes(device.index, B, T, Hq, H, D)
    a = _pack_tree(*place, _ptr(status), q.data_ptr(), *q.stride()[:3], draft_k.data_ptr(), *draft_k.stride()[:3],
                   draft_v.data_ptr(), *draft_v.stride()[:3], *m, out.data_ptr(), *out.stride()[:3], lse.data_ptr(),
                   B, T, Hq, H, D, float(scale), code)
    _call(device, lib().slimkv_tree_attention, a, nbytes)
    if owned:
        check_status(status)
    return out, lse


def attention_weights(q, lse, scale, k=None, *, pages=None, table=None, lengths=None, keys=None, causal=True,
                      previous=None, out=None, status=None):
    """The attention weight of every cached row, added to what it has gathered:

        out[b, h, j] = previous[b, h, j] + sum over l, g of exp(scale q[b, l, hG + g] . k[b, j, h] - lse[b, hG + g, l])

    q [B, L, Hq, D] rotated and lse [B, Hq, L] fp32 as the attention left it
    (tree_attention, kernels.attention_forward, kernels.prefill_attention); the
    cache dense (k alone) or paged.  With `causal` the last query stands at the
    sequence's last row and query l sees rows up to length - L + l; a query row
    whose LSE is -inf counts nothing (padding).  previous [B, Hkv, N] fp32,
    None for zeros; N = the dense rows or `keys` (default cols * block).  Rows
    at or past a sequence's length keep `previous`.  Returns out [B, Hkv, N]
    fp32, which may be `previous` itself."""
    name = 'attention_weights'
    B = q.shape[0]
    place, rows, H, D, paged, keep = _cache(name, k, None, pages, table, lengths, keys, B, values=False)
    code = _dtype(name, q, pages if k is None else k)
    _queries(name, q, H, D)
    _, L, Hq, _ = q.shape
    if lse.shape != (B, Hq, L) or lse.dtype is not torch.float32:
        raise ValueError(f'{name}: lse must be float32 [{B}, {Hq}, {L}]')
    shape = (B, H, rows)
    for what, t in (('previous', previous), ('out', out)):
        if t is not None and (t.shape != shape or t.dtype is not torch.float32 or t.stride(2) != 1 and rows > 1):
            raise ValueError(f'{name}: {what} must be float32 {list(shape)} with contiguous rows')
    if out is not None and previous is not None and _overlap(out, previous) and \
            (out.data_ptr() != previous.data_ptr() or out.stride() != previous.stride()):
        raise ValueError(f'{name}: out must be previous itself or lie apart from it')
    if out is not None and (_folded(out) or any(t is not None and _overlap(out, t)
                                                  for t in (lse, q, k, pages, table, lengths))):
        raise ValueError(f'{name}: out must not be an expanded view and lie apart from lse and the other inputs')
    device = _common(name, q, lse, k, pages, table, lengths, previous, out)
    if out is None:
        out = _new(torch.float32, device, *shape)
    q = _rows16(q)
    status, owned = _status(name, status, device, paged)
    nbytes = _weights_bytes(device.index, B, L, Hq, H, D, rows)
    a = _pack_weights(*place, _ptr(status), q.data_ptr(), *q.stride()[:3], lse.data_ptr(), *lse.stride(),
                      *((previous.data_ptr(), *previous.stride()[:2]) if previous is not None else (0, 0, 0)),
                      out.data_ptr(), *out.stride()[:2], B, L, Hq, H, D, float(scale), bool(causal), code)
    _call(device, lib().slimkv_attention_weights, a, nbytes)
    if owned:
        check_status(status)
    return out


def select_rows(weights, keep, *, lengths=None, sink=0, recent=0):
    """The rows a cache of `keep` rows holds on to: the first `sink`, the last
    `recent`, and of those between the heaviest by weights [B, H, N] fp32 (H
    the KV heads, or 1 for one choice for all heads).  Equal weights: the lower
    index first; NaN ranks below every number.  Returns (rows [B, H, keep]
    int32, ascending, -1 past the count; counts [B] int32 = min(length, keep))."""
    name = 'select_rows'
    if weights.dim() != 3 or weights.dtype is not torch.float32:
        raise ValueError(f'{name}: weights must be float32 [B, H, N]')
    B, H, N = weights.shape
    keep, sink, recent = int(keep), int(sink), int(recent)
    if keep <= 0 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError(f'{name}: needs keep > 0 and 0 <= sink + recent <= keep')
    if weights.stride(2) != 1:
        weights = weights.contiguous()
    lengths = _lengths(name, lengths, B)
    device = _common(name, weights, lengths)
    rows = _new(torch.int32, device, B, H, keep)
    counts = torch.empty_strided((B,), (1,), dtype=torch.int32, device=device)
    a = _pack_select(weights.data_ptr(), *weights.stride()[:2], _ptr(lengths), rows.data_ptr(), counts.data_ptr(), B, H, N,
                     keep, sink, recent)
    nbytes = _select_bytes(device.index, B, H, N, keep, sink, recent)
    _call(device, lib().slimkv_select_rows, a, nbytes)
    return rows, counts


def compact_rows(rows, counts, k=None, v=None, *, pages=None, table=None, weights=None, out_k=None, out_v=None,
                 in_place=False, status=None):
    """Rows rows[b, h, :counts[b]] of every sequence and KV head, moved to the
    front of a cache; rows int32 [B, Hkv or 1, keep], counts int32 [B].

    Out of place (the default): returns (k, v [B, keep, Hkv, D], weights
    [B, Hw, keep] or None), rows from counts[b] on zero.  in_place: within the
    given k / v or pages and within `weights`, for choices in strictly
    ascending order (select_rows'); cache rows from counts[b] on stay as they
    are, weights from there on become zero; returns the given tensors (None,
    None for pages).  weights [B, rows' head count, N] fp32 move along.  A row
    outside the cache (in place: or out of order) moves nothing and raises
    IndexError after the call, or is left in `status`.  In place, no other
    sequence's table may name the pages a sequence writes (an expanded table
    is refused), and k, v, weights and the index tensors share no memory."""
    name = 'compact_rows'
    if rows.dim() != 3 or rows.dtype is not torch.int32 or counts.dtype is not torch.int32 or \
            counts.shape != rows.shape[:1]:
        raise ValueError(f'{name}: rows must be int32 [B, heads, keep] and counts int32 [B]')
    B, Hw, keep = rows.shape
    place, _, H, D, _, held = _cache(name, k, v, pages, table, None, None, B)
    first = pages if k is None else k
    code = _dtype(name, first, v, out_k, out_v)
    if Hw not in (1, H):
        raise ValueError(f'{name}: rows must have 1 or {H} heads')
    rows = rows if rows.stride(2) == 1 else rows.contiguous()
    counts = counts.contiguous()
    if weights is not None and (weights.dim() != 3 or weights.shape[:2] != (B, Hw) or weights.stride(2) != 1 or
                                weights.dtype is not torch.float32):
        raise ValueError(f'{name}: weights must be float32 [{B}, {Hw}, N] with contiguous rows')
    out_weights = None
    if in_place:
        if out_k is not None or out_v is not None:
            raise ValueError(f'{name}: in place there are no outputs')
        for t in (k, v, pages, weights):
            if t is not None and _folded(t):
                raise ValueError(f'{name}: in place the cache and the weights must not be expanded or overlapping views')
        if not _apart((k, v, pages, weights), (rows, counts, table)):
            raise ValueError(f'{name}: in place k and v must be two tensors, and they, the weights and the index tensors '
                             'must share no memory')
        if table is not None and _folded(table):
            raise ValueError(f'{name}: in place each table entry names pages of its own: no expanded or overlapping table')
    for t in (out_k, out_v):
        if t is not None and (t.shape != (B, keep, H, D) or t.stride(3) != 1 or _folded(t) or
                              any(s is not None and _overlap(t, s) for s in (k, v, pages, table, rows, counts, weights))):
            raise ValueError(f'{name}: outputs must be [{B}, {keep}, {H}, {D}] with contiguous features, no expanded '
                             'views and apart from the cache and the other inputs')
    if out_k is not None and out_v is not None and _overlap(out_k, out_v):
        raise ValueError(f'{name}: out_k and out_v must lie apart')
    device = _common(name, rows, counts, k, v, pages, table, weights, out_k, out_v)
    outs = (0, 0, 0, 0, 0, 0, 0, 0)
    if not in_place:
        if out_k is None:
            out_k = torch.empty_strided((B, keep, H, D), (keep * H * D, H * D, D, 1), dtype=first.dtype, device=device)
        if out_v is None:
            out_v = torch.empty_like(out_k, memory_format=torch.contiguous_format)
        if weights is not None:
            out_weights = _new(torch.float32, device, B, Hw, keep)
        outs = (out_k.data_ptr(), *out_k.stride()[:3], out_v.data_ptr(), *out_v.stride()[:3])
    status, owned = _status(name, status, device, True)
    a = _pack_compact(*place, status.data_ptr(), rows.data_ptr(), rows.stride(0), rows.stride(1) if Hw > 1 else 0,
                      counts.data_ptr(), *outs,
                      *((weights.data_ptr(), *weights.stride()[:2]) if weights is not None else (0, 0, 0)),
                      *((out_weights.data_ptr(), *out_weights.stride()[:2]) if out_weights is not None else (0, 0, 0)),
                      *((0, 0) if weights is None else (Hw, weights.shape[2])), B, H, D, keep, bool(in_place), code)
    _call(device, lib().slimkv_compact_rows, a)
    if owned:
        check_status(status)
    if in_place:
        return k, v, weights
    return out_k, out_v, out_weights
