"""A K/V cache held in 4 bits, and the step around it.

    norm_rope            queries and keys, each head normalised and rotated
    quantize_rows        rows of K and V written into the cache
    dequantize_rows      rows of it as values of the element type
    quantized_attention  every new token over the cached rows and its ancestors

A decode step: norm_rope turns the projections' outputs into queries and keys,
quantized_attention attends to the cache and to the step's own rows (still in
the element type), quantize_rows appends the rows that stay.  A prefill window
reads the history with dequantize_rows or attends to it directly, up to 1024
tokens a call.

The cache is a uint8 tensor `pages` [pages, Hkv, bytes] (new_pages): `block` rows
of a page, a multiple of 16, take page_bytes(block, head_dim) = block * (D +
D / 16) bytes a KV head, 17 / 64 of bf16 or fp16 rows.  Blocks of 32 elements share a
power of two and hold 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6, and negative)
times it: an element is off by at most a fifth of its block's largest magnitude
(2^-129 where that is more; a quarter in blocks that reach past 15/16 of the power
of two at which the type ends, 65536 or 2^128).  A block that held an infinity or
NaN reads as NaN.  include/slimkv/quant_cache.h gives every byte's place.  With a
block table [B, cols] int64 row n of sequence b is row n % block of page table[b, n
// block]; without one sequence b is page b.

Element types bf16 and fp16 (one for all tensors of a call; the cache itself has
none), head_dim 64 or 128.  Up to 65535 sequences and 4096 heads.  Pages start on
16-byte boundaries.  Table entries follow torch's indexing rules; an entry outside
the pool, a row outside the cache or a position outside the rotation tables raises
IndexError after the call (one host synchronisation), or is left in the caller's
device int32 `status` word (graph capture, serving loops; kernels.check_status).
The operators have no gradients: they raise ValueError where one would be recorded
or a forward-mode tangent lost, and for negative views.
"""
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import lib
from .cache_ops import (_DTYPES, _asked, _call, _common, _dtype, _folded, _lengths, _new, _overlap, _packer, _ptr,
                        _rows16, _span, _status)
from .kernels import check_status

_pack_rows = _packer(_lib.QuantizeRowsArgs)
_pack_attention = _packer(_lib.QuantizedAttentionArgs)
_pack_norm_rope = _packer(_lib.NormRopeArgs)


def _device(name, *tensors):
    """cache_ops._common in the time that it takes where nothing is refused."""
    index = tensors[0].get_device()
    grad = torch.is_grad_enabled()
    if index < 0 or forward_ad._current_level >= 0:
        return _common(name, *tensors)
    for t in tensors:
        if t is not None and (t.get_device() != index or t.is_neg() or grad and t.requires_grad):
            return _common(name, *tensors)
    return tensors[0].device


def _clear_of(written, *read):
    """Whether `written` shares no memory with the other tensors: most lie before or behind it as a whole."""
    w0, w1 = _span(written)
    for t in read:
        if t is not None and t.data_ptr() < w1 and _span(t)[1] > w0 and _overlap(written, t):
            return False
    return True


def page_bytes(block, head_dim):
    """Bytes that the `block` rows (a multiple of 16) of a page take for one KV head."""
    if head_dim not in (64, 128) or block <= 0 or block % 16:
        raise ValueError('pages hold a multiple of 16 rows of head_dim 64 or 128')
    return block * (head_dim + head_dim // 16)


def new_pages(pages, kv_heads, block, head_dim, device='cuda'):
    """A pool of `pages` pages, all rows zero: uint8 [pages, kv_heads, page_bytes(block, head_dim)]."""
    return torch.zeros(pages, kv_heads, page_bytes(block, head_dim), dtype=torch.uint8, device=device)


def _pool(name, pages, table, batch, heads, dim):
    """A pool as the C struct's values but for the status word: (fields, rows of a sequence, KV heads, the table they
    point into)."""
    if dim != 128 and dim != 64:
        raise ValueError(f'{name}: head_dim must be 64 or 128')
    if pages.dim() != 3 or pages.dtype is not torch.uint8:
        raise ValueError(f'{name}: pages must be uint8 [pages, Hkv, bytes] with contiguous bytes')
    count, found, size = pages.shape
    page_stride, head_stride, step = pages.stride()
    if step != 1:
        raise ValueError(f'{name}: pages must be uint8 [pages, Hkv, bytes] with contiguous bytes')
    block, rest = divmod(size, dim + dim // 16)
    if rest or block == 0 or block % 16:
        raise ValueError(f'{name}: a page of {size} bytes is no multiple of 16 rows of head_dim {dim}')
    if found != heads and heads is not None:
        raise ValueError(f'{name}: pages of {found} KV heads, rows of {heads}')
    if table is None:
        if count < batch:
            raise ValueError(f'{name}: without a block table every sequence needs a page ({batch} for {count})')
        return (pages.data_ptr(), page_stride, head_stride, 0, 0, 0, count, block), block, found, None
    if table.dtype is not torch.int64 or table.dim() != 2 or table.shape[0] != batch or table.shape[1] == 0:
        raise ValueError(f'{name}: the block table must be int64 [{batch}, cols]')
    if table.stride(1) != 1:
        table = table.contiguous()
    cols = table.shape[1]
    return (pages.data_ptr(), page_stride, head_stride, table.data_ptr(), table.stride(0), cols, count, block), \
        cols * block, found, table


def _whole_numbers(name, what, t, batch):
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != batch:
        raise ValueError(f'{name}: {what} must be int32 [{batch}]')
    return t if t.is_contiguous() else t.contiguous()


def quantize_rows(k, v, pages, table=None, *, starts=None, counts=None, status=None):
    """Writes rows k, v [B, n, Hkv, D] into the cache: row i < counts[b] of sequence b (default: all n) becomes its cache
    row starts[b] + i (default: i).  starts and counts [B] int32.  A row outside the cache is not written and raises
    IndexError (or is left in `status`).  No two rows may go to one place: no expanded table, no page that two
    sequences write; rows that are not written keep their bytes.  Returns pages."""
    name = 'quantize_rows'
    if k.dim() != 4 or v.shape != k.shape or k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError(f'{name}: k and v must be [B, n, Hkv, D] with contiguous features')
    B, n, H, D = k.shape
    code = _dtype(name, k, v)
    given = table
    place, rows, _, table = _pool(name, pages, table, B, H, D)
    starts, counts = _whole_numbers(name, 'starts', starts, B), _whole_numbers(name, 'counts', counts, B)
    # the table as it was given: the copy of one that is expanded along its columns is no expanded view
    if not pages.is_contiguous() and _folded(pages) or given is not None and not given.is_contiguous() and _folded(given):
        raise ValueError(f'{name}: pages and table must not be expanded or overlapping views')
    if not _clear_of(pages, k, v, table, starts, counts):
        raise ValueError(f'{name}: pages must share no memory with the other tensors')
    device = _device(name, k, v, pages, table, starts, counts)
    k, v = _rows16(k), _rows16(v)
    status, owned = _status(name, status, device, table is not None or starts is not None or n > rows)
    a = _pack_rows(*place, _ptr(status), k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], _ptr(starts),
                   _ptr(counts), B, n, H, D, code)
    _call(device, lib().slimkv_quantize_rows, a)
    if owned:
        check_status(status)
    return pages


def dequantize_rows(pages, rows, head_dim, table=None, *, starts=None, counts=None, dtype=torch.bfloat16, out_k=None,
                    out_v=None, status=None):
    """Rows of the cache as values: (k, v), each [B, rows, Hkv, D] of `dtype` (bf16, exact, or fp16, rounded).  Row i <
    counts[b] (default: all) is cache row starts[b] + i (default: i) of sequence b; rows from counts[b] on are zero.
    A row outside the cache is zero and raises IndexError (or is left in `status`).  Without a table B is the length
    of starts or counts, or the number of pages."""
    name = 'dequantize_rows'
    rows, D = int(rows), int(head_dim)
    if rows < 0:
        raise ValueError(f'{name}: rows must not be negative')
    sized = table if table is not None else starts if starts is not None else counts if counts is not None else pages
    B = sized.shape[0] if sized.dim() else 0
    place, capacity, H, table = _pool(name, pages, table, B, None, D)
    starts, counts = _whole_numbers(name, 'starts', starts, B), _whole_numbers(name, 'counts', counts, B)
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f'{name}: dtype must be bfloat16 or float16')
    shape = (B, rows, H, D)
    for t in (out_k, out_v):
        if t is not None and (t.shape != shape or t.dtype is not dtype or t.stride(3) != 1 or _folded(t) or
                              not _clear_of(t, pages, table, starts, counts)):
            raise ValueError(f'{name}: outputs must be {dtype} {list(shape)} with contiguous features, no expanded views and '
                             'apart from the cache and the other inputs')
    if out_k is not None and out_v is not None and _overlap(out_k, out_v):
        raise ValueError(f'{name}: out_k and out_v must lie apart')
    device = _device(name, pages, table, starts, counts, out_k, out_v)
    row = H * D
    dense = (rows * row, row, D, 1)
    if out_k is None:
        out_k, k_strides = torch.empty_strided(shape, dense, dtype=dtype, device=device), dense
    else:
        k_strides = out_k.stride()
    if out_v is None:
        out_v, v_strides = torch.empty_strided(shape, dense, dtype=dtype, device=device), dense
    else:
        v_strides = out_v.stride()
    status, owned = _status(name, status, device, table is not None or starts is not None or rows > capacity)
    a = _pack_rows(*place, _ptr(status), out_k.data_ptr(), *k_strides[:3], out_v.data_ptr(), *v_strides[:3], _ptr(starts),
                   _ptr(counts), B, rows, H, D, code)
    _call(device, lib().slimkv_dequantize_rows, a)
    if owned:
        check_status(status)
    return out_k, out_v


# Asked for once for each set of sizes (and the device).
@lru_cache(1024)
def _attention_bytes(index, B, T, Hq, H, D, keys):
    return _asked(lib().slimkv_quantized_attention_workspace, _lib.QuantizedAttentionArgs(
        q=16, keys=keys, batch=B, tokens=T, heads=Hq, kv_heads=H, head_dim=D, scale=1.0), index)


def quantized_attention(q, draft_k, draft_v, scale, pages, table=None, *, lengths=None, keys=None, mask=None, out=None,
                        lse=None, status=None):
    """Attention of new tokens over a cache held in 4 bits and over each other: cache_ops.tree_attention with the
    cached rows read from `pages`.

    q [B, T, Hq, D] (rotated, T up to 1024); draft_k / draft_v [B, T, Hkv, D], the new tokens' own rows in the element
    type, or both None: the cache alone.  mask [T, T] or [B, T, T] bool: token t sees new token j where mask[.., t,
    j]; None is a chain (j <= t).  Every token sees rows 0 .. lengths[b] - 1 of its sequence (lengths [B] int32,
    default and at most `keys`, itself by default all rows the cache has room for).  Returns (out [B, T, Hq, D], lse
    [B, Hq, T] fp32); a row that sees nothing gives 0 and -inf, and what lies in unseen rows has no influence.  The
    cached rows enter as dequantize_rows returns them in the type of q: exact in bf16 and, of what fp16 wrote, in fp16;
    fp16 rounds numbers below 2^-22 that bf16 wrote and takes those past 65504 as infinities.  All other rounding is
    tree_attention's.  (out, lse) of the cache alone merge with another branch by kernels.merge."""
    name = 'quantized_attention'
    if q.dim() != 4 or pages.dim() != 3:
        raise ValueError(f'{name}: q must be [B, T, Hq, D] and pages [pages, Hkv, bytes]')
    B, T, Hq, D = q.shape
    place, capacity, H, table = _pool(name, pages, table, B, None, D)
    code = _dtype(name, q, draft_k, draft_v, out)
    if H == 0 or Hq % H or q.stride(3) != 1:
        raise ValueError(f'{name}: q must be [B, T, Hq, D] with Hq a multiple of {H} and contiguous features')
    if (draft_k is None) != (draft_v is None):
        raise ValueError(f'{name}: give both draft_k and draft_v or neither')
    if draft_k is not None and (draft_k.shape != (B, T, H, D) or draft_v.shape != (B, T, H, D)):
        raise ValueError(f'{name}: draft_k and draft_v must be [{B}, {T}, {H}, {D}]')
    lengths = _lengths(name, lengths, B)
    keys = capacity if keys is None else int(keys)
    if not 0 <= keys <= capacity:
        raise ValueError(f'{name}: keys must lie in [0, {capacity}]')
    m = (0, 0, 0)
    if mask is not None:
        if draft_k is None:
            raise ValueError(f'{name}: a mask belongs to drafted rows')
        if mask.dtype is not torch.bool or mask.shape not in ((T, T), (B, T, T)):
            raise ValueError(f'{name}: mask must be bool [{T}, {T}] or [{B}, {T}, {T}]')
        if mask.stride(-1) != 1:
            mask = mask.contiguous()
        m = (mask.data_ptr(), mask.stride(0) if mask.dim() == 3 else 0, mask.stride(-2))
    inputs = (q, draft_k, draft_v, pages, table, lengths, mask)
    if out is not None and (out.shape != q.shape or out.stride(3) != 1 or _folded(out) or not _clear_of(out, *inputs)):
        raise ValueError(f'{name}: out must have the shape of q with contiguous features, no expanded view and apart '
                         'from the inputs')
    if lse is not None and (lse.shape != (B, Hq, T) or lse.dtype is not torch.float32 or not lse.is_contiguous() or
                            not _clear_of(lse, *inputs, out)):
        raise ValueError(f'{name}: lse must be a contiguous float32 [{B}, {Hq}, {T}], apart from the other tensors')
    device = _device(name, *inputs, out, lse)
    q = _rows16(q)
    d = (0, 0, 0, 0, 0, 0, 0, 0)
    if draft_k is not None:
        draft_k, draft_v = _rows16(draft_k), _rows16(draft_v)
        d = (draft_k.data_ptr(), *draft_k.stride()[:3], draft_v.data_ptr(), *draft_v.stride()[:3])
    if out is None:
        row = Hq * D
        o_strides = (T * row, row, D, 1)
        out = torch.empty_strided((B, T, Hq, D), o_strides, dtype=q.dtype, device=device)
    else:
        o_strides = out.stride()
    if lse is None:
        lse = _new(torch.float32, device, B, Hq, T)
    status, owned = _status(name, status, device, table is not None and keys > 0)
    nbytes = _attention_bytes(device.index, B, T, Hq, H, D, keys)
    a = _pack_attention(*place, _ptr(status), _ptr(lengths), keys, q.data_ptr(), *q.stride()[:3], *d, *m, out.data_ptr(),
                        *o_strides[:3], lse.data_ptr(), B, T, Hq, H, D, float(scale), code)
    _call(device, lib().slimkv_quantized_attention, a, nbytes)
    if owned:
        check_status(status)
    return out, lse


def _packed16(t):
    """t, or a copy where it is not contiguous from a 16-byte boundary."""
    if t is None or t.data_ptr() % 16 == 0 and t.is_contiguous():
        return t
    return t.clone(memory_format=torch.contiguous_format)


def norm_rope(q, k, cos, sin, positions, *, q_weight=None, k_weight=None, eps=1e-6, out_q=None, out_k=None,
              status=None):
    """Queries and keys of a step or window, each head normalised by its root mean square, weighed and rotated:

        y = x / sqrt(mean(x^2) + eps) * weight        out = y * cos[pos] + rotate_half(y) * sin[pos]

    q [B, L, Hq, D] and k [B, L, Hkv, D] (None: queries alone), views of a fused projection's output among them;
    weights [D] of their type or float32 (both alike), or None for heads that are not normalised; cos, sin [rows, D]
    float32 (workloads.rope_tables), contiguous from a 16-byte boundary (others are copied whole, every call);
    positions int64 [B, L] or [1, L].  fp32 throughout and one rounding, where kernels.rope_decode takes the reference's
    bf16 steps; a normalised head's sum of squares has to lie within fp32.  A position outside the tables raises
    IndexError (or is left in `status`), its token's rows are not written.  Returns (out_q, out_k); out_q may be q itself,
    out_k k (where q and k are one tensor, neither)."""
    name = 'norm_rope'
    if q.dim() != 4 or q.stride(3) != 1:
        raise ValueError(f'{name}: q must be [B, L, Hq, D] with contiguous features')
    B, L, Hq, D = q.shape
    H = 0
    if k is not None:
        if k.dim() != 4 or k.stride(3) != 1 or k.shape[0] != B or k.shape[1] != L or k.shape[3] != D:
            raise ValueError(f'{name}: with q must be k [{B}, {L}, Hkv, {D}] with contiguous features')
        H = k.shape[2]
    code = _dtype(name, q, k, out_q, out_k)
    rows, width = cos.shape if cos.dim() == 2 else (0, 0)
    if width != D or sin.shape != cos.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f'{name}: cos and sin must be float32 [rows, {D}]')
    if positions.dtype is not torch.int64 or positions.shape not in ((B, L), (1, L)):
        raise ValueError(f'{name}: positions must be int64 [{B}, {L}] or [1, {L}]')
    kind = q.dtype
    for what, w in (('q_weight', q_weight), ('k_weight', k_weight)):
        if w is not None:
            if w.shape != (D,) or w.dtype not in (q.dtype, torch.float32):
                raise ValueError(f'{name}: {what} must be [{D}] of {q.dtype} or float32')
            kind = w.dtype
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise ValueError(f'{name}: q_weight and k_weight must be of one type')
    if k is None and (k_weight is not None or out_k is not None):
        raise ValueError(f'{name}: k_weight and out_k belong to keys')
    for what, x, other, t in (('out_q', q, k, out_q), ('out_k', k, q, out_k)):
        if t is None:
            continue
        if t.shape != x.shape or t.stride(3) != 1 or _folded(t):
            raise ValueError(f'{name}: {what} must have the shape of its input with contiguous features, no expanded view')
        same = t.data_ptr() == x.data_ptr() and t.stride() == x.stride()
        # by role: q and k may be one tensor, and what is in place for one is then not apart from the other
        if not _clear_of(t, other, cos, sin, positions, q_weight, k_weight, None if same else x):
            raise ValueError(f'{name}: {what} must be its input itself or lie apart from all inputs')
    if out_q is not None and out_k is not None and _overlap(out_q, out_k):
        raise ValueError(f'{name}: out_q and out_k must lie apart')
    device = _device(name, q, k, cos, sin, positions, q_weight, k_weight, out_q, out_k)
    q_weight, k_weight, cos, sin = _packed16(q_weight), _packed16(k_weight), _packed16(cos), _packed16(sin)
    q, k = _rows16(q), None if k is None else _rows16(k)
    if out_q is None:
        row = Hq * D
        q_strides = (L * row, row, D, 1)
        out_q = torch.empty_strided((B, L, Hq, D), q_strides, dtype=q.dtype, device=device)
    else:
        q_strides = out_q.stride()
    if out_k is None and k is not None:
        row = H * D
        k_strides = (L * row, row, D, 1)
        out_k = torch.empty_strided((B, L, H, D), k_strides, dtype=q.dtype, device=device)
    elif k is not None:
        k_strides = out_k.stride()
    none = (0, 0, 0, 0)
    status, owned = _status(name, status, device, True)
    a = _pack_norm_rope(q.data_ptr(), *q.stride()[:3], *(none if k is None else (k.data_ptr(), *k.stride()[:3])),
                        _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), rows, positions.data_ptr(),
                        positions.stride(0) if positions.shape[0] > 1 else 0, positions.stride(1), out_q.data_ptr(),
                        *q_strides[:3], *(none if k is None else (out_k.data_ptr(), *k_strides[:3])), status.data_ptr(), B, L,
                        Hq, H, D, float(eps), kind is torch.float32, code)
    _call(device, lib().slimkv_norm_rope, a)
    if owned:
        check_status(status)
    return out_q, out_k
