"""Cache operators on the GPU against their 64-bit plain forms (oracle/cache.py).

Tolerances follow from the arithmetic, element by element.  u is half a step of the element type (bf16 2^-8, fp16
2^-11).  A score is an fp32 sum of D exact products: its error is below d = 2^-24 (D + 8) sum|q k| scale plus the
roundings of the scaled exponent, 2^-22 (1 + |score|).  So a weight is off by at most d relative, plus u where it is
rounded for the matrix product; the output takes (2 d + u) sum(p |v|) and its own rounding u |out|.  fp16 weights
below 2^-14 have a half step of 2^-25: 2^-25 max|v| a key before the division by the row's sum.  An LSE takes d, the
fp32 sum of n positive terms (n / 4 + 64 additions in a row at most, 2^-24 each) and 2^-21 (1 + |lse|) for the
logarithm and its scaling.
"""
import numpy as np
import pytest
import torch

from oracle import cache as oc
from tests.helpers import bits, to_np

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16, gain=1.0):
    return (torch.randn(*shape, generator=g, device='cuda') * gain).to(dtype)


def make_cache(g, B, N, H, D, block, dtype, spare=3):
    """Dense k, v and the keywords that hand the same rows over: dense, or pages in scattered blocks whose unused rows
    hold NaN, with some table entries counted from the pool's end."""
    k, v = randn(g, B, N, H, D, dtype=dtype), randn(g, B, N, H, D, dtype=dtype)
    if not block:
        return k, v, dict(k=k, v=v)
    cols = -(-max(N, 1) // block)
    pool = B * cols + spare
    table = torch.randperm(pool, generator=g, device='cuda')[:B * cols].view(B, cols)
    pages = torch.full((pool, block, 2, H, D), float('nan'), dtype=dtype, device='cuda')
    for b in range(B):
        rows = torch.full((cols * block, 2, H, D), float('nan'), dtype=dtype, device='cuda')
        rows[:N, 0], rows[:N, 1] = k[b], v[b]
        pages[table[b]] = rows.view(cols, block, 2, H, D)
    table = torch.where(torch.arange(cols, device='cuda') % 3 == 1, table - pool, table)
    return k, v, dict(pages=pages, table=table, keys=N)


def lengths_of(lengths):
    return None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')


def f64(t):
    return to_np(t)


def check_tree(out, lse, q, k, v, lengths, dk, dv, mask, scale, what=''):
    B, T, Hq, D = q.shape
    n = [k.shape[1]] * B if lengths is None else [max(0, min(x, k.shape[1])) for x in lengths]
    m = None if mask is None else mask.cpu().numpy()
    eo, el, terms, top, mass, total = oc.tree_attention(f64(q), f64(k), f64(v), n, f64(dk), f64(dv), m, scale)
    u = HALF[q.dtype]
    d = 2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top)
    d = d.transpose(0, 2, 1)[..., None]
    biggest = max([np.abs(f64(x)[np.isfinite(f64(x))]).max(initial=0.0) for x in (v, dv)])
    tiny = 2.0 ** -25 * (max(n) + T) * biggest / total.transpose(0, 2, 1)[..., None] if q.dtype is torch.float16 else 0.0
    tol = (2 * d + u) * terms + u * np.abs(eo) * (1 + u) + tiny + 1e-30
    o, s = f64(out), lse.double().cpu().numpy()
    assert np.isfinite(o).all(), what
    worst = (np.abs(o - eo) / tol).max() if o.size else 0.0
    print(what, 'worst output error over its bound', worst, flush=True)
    assert worst <= 1.0, what
    empty = np.isneginf(el)
    assert (np.isneginf(s) == empty).all(), what
    assert not o.transpose(0, 2, 1, 3)[empty].any(), what
    fin = ~empty
    tl = 2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top) + 2.0 ** -24 * ((max(n) + T) / 4 + 64) + 2.0 ** -21 * (
        1 + np.abs(np.where(fin, el, 0)))
    assert (np.abs(s[fin] - el[fin]) <= tl[fin]).all(), what


def tree_mask(g, B, T, kind):
    if kind is None:
        return None
    if kind == 'none':
        return torch.zeros(B, T, T, dtype=torch.bool, device='cuda')
    mask = torch.rand(B, T, T, generator=g, device='cuda') < 0.4
    if kind == 'rows':                   # rows that see nothing of the draft
        mask[:, ::3] = False
    return mask[0] if kind == 'shared' else mask


TREE = [
    # B, T, Hq, Hkv, D, N, lengths, block, dtype, mask
    (1, 1, 8, 2, 128, 1, None, 0, 'bf16', None),
    (1, 1, 8, 2, 128, 0, None, 0, 'bf16', None),
    (2, 1, 4, 4, 128, 65, [65, 0], 16, 'bf16', 'none'),
    (3, 1, 32, 8, 128, 517, [517, 64, 63], 16, 'bf16', None),
    (2, 5, 14, 2, 64, 200, [200, 129], 48, 'bf16', None),
    (2, 7, 8, 8, 128, 127, [1, 127], 1, 'fp16', 'rows'),
    (1, 9, 10, 2, 128, 700, None, 0, 'fp16', 'tree'),
    (2, 13, 8, 2, 128, 321, [320, 5], 3, 'bf16', 'shared'),
    (1, 26, 16, 4, 128, 1029, None, 0, 'bf16', 'tree'),
    (2, 40, 10, 2, 64, 256, [256, 250], 32, 'fp16', 'tree'),
    (1, 63, 5, 1, 128, 130, None, 0, 'bf16', 'rows'),
    (1, 130, 6, 2, 128, 67, [66], 16, 'bf16', 'tree'),
    (1, 130, 4, 2, 64, 40, None, 0, 'fp16', None),
    (70, 2, 4, 2, 64, 150, [(7 * i) % 151 for i in range(70)], 16, 'bf16', None),
    (1, 2, 2, 1, 128, 5003, None, 0, 'bf16', None),
    (2, 3, 2, 1, 64, 4001, [4001, 17], 16, 'fp16', 'none'),
    (1, 5, 32, 1, 128, 300, None, 0, 'bf16', 'tree'),
    (66, 9, 8, 1, 64, 140, [(11 * i) % 141 for i in range(66)], 16, 'fp16', 'tree'),
    (3, 33, 32, 4, 128, 200, [200, 0, 131], 7, 'bf16', 'rows'),
]
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


@pytest.mark.parametrize('case', TREE, ids=[str(i) for i in range(len(TREE))])
def test_tree_attention(case):
    from slimkv_amd import cache_ops
    B, T, Hq, H, D, N, lengths, block, dtype, kind = case
    print(case, flush=True)
    dt, g = TYPES[dtype], gen(7)
    k, v, place = make_cache(g, B, N, H, D, block, dt)
    q = randn(g, B, T, Hq, D, dtype=dt, gain=2.0)
    dk, dv = randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    mask = tree_mask(g, B, T, kind)
    scale = D ** -0.5
    out, lse = cache_ops.tree_attention(q, dk, dv, scale, lengths=lengths_of(lengths), mask=mask, **place)
    check_tree(out, lse, q, k, v, lengths, dk, dv, mask, scale, str(case))
    again, lse2 = cache_ops.tree_attention(q, dk, dv, scale, lengths=lengths_of(lengths), mask=mask, **place)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize('T,heads,kv', [(6, 8, 2), (24, 8, 2), (70, 8, 2)])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_tree_unseen_drafted_rows_have_no_influence(T, heads, kv, dtype):
    """Infinities and NaN in drafted tokens that a row does not see."""
    from slimkv_amd import cache_ops
    B, D, N, dt, g = 2, 128, 100, TYPES[dtype], gen(3)
    k, v, place = make_cache(g, B, N, kv, D, 0, dt)
    q = randn(g, B, T, heads, D, dtype=dt)
    dk, dv = randn(g, B, T, kv, D, dtype=dt), randn(g, B, T, kv, D, dtype=dt)
    dk[0, 1], dv[0, 1] = float('nan'), float('inf')
    dk[1, T - 1], dv[1, T - 1, :, ::3] = float('inf'), float('nan')
    mask = torch.ones(B, T, T, dtype=torch.bool, device='cuda').tril()
    mask[0, :, 1], mask[1, :, T - 1] = False, False
    out, lse = cache_ops.tree_attention(q, dk, dv, D ** -0.5, mask=mask, **place)
    check_tree(out, lse, q, k, v, None, dk, dv, mask, D ** -0.5)


def test_tree_visible_nan_reaches_only_its_rows():
    from slimkv_amd import cache_ops
    g, D = gen(4), 128
    k, v, place = make_cache(g, 1, 70, 2, D, 0, torch.bfloat16)
    q, dk, dv = randn(g, 1, 8, 8, D), randn(g, 1, 8, 2, D), randn(g, 1, 8, 2, D)
    dv[0, 5, 1] = float('nan')
    out, _ = cache_ops.tree_attention(q, dk, dv, D ** -0.5, **place)
    bad = torch.isnan(out.float()).any(-1)[0]
    assert bad[5:, 4:].all() and not bad[:5].any() and not bad[:, :4].any()


def test_tree_strides_and_given_outputs():
    """Heads-first q, K and V as halves of one tensor, a batch that shares one cache, outputs inside larger buffers."""
    from slimkv_amd import cache_ops
    B, T, Hq, H, D, N, g = 3, 4, 8, 2, 128, 90, gen(5)
    q = randn(g, B, Hq, T, D).transpose(1, 2)
    kv = randn(g, 1, N, 2, H, D).expand(B, N, 2, H, D)
    draft = randn(g, B, H, T, 2 * D)
    dk, dv = draft[..., :D].transpose(1, 2), draft[..., D:].transpose(1, 2)
    mask = tree_mask(g, B, T, 'tree').transpose(1, 2)
    buf = torch.full((B, T, Hq + 1, 2 * D), 7.0, dtype=torch.bfloat16, device='cuda')
    out = buf[:, :, :Hq, :D]
    lse = torch.empty(B, Hq, T, device='cuda')
    a, b = cache_ops.tree_attention(q, dk, dv, D ** -0.5, kv[:, :, 0], kv[:, :, 1], mask=mask, out=out, lse=lse)
    assert a is out and b is lse
    check_tree(out, lse, q, kv[:, :, 0], kv[:, :, 1], None, dk, dv, mask, D ** -0.5)
    assert (buf[:, :, Hq] == 7).all() and (buf[..., D:] == 7).all()
    odd = torch.empty(B * T * Hq * D + 1, dtype=torch.bfloat16, device='cuda')[1:].view(B, T, Hq, D)
    odd.copy_(q)
    again, _ = cache_ops.tree_attention(odd, dk, dv, D ** -0.5, kv[:, :, 0], kv[:, :, 1], mask=mask)
    assert torch.equal(again, out)


def test_tree_offsets_past_32_bits():
    """Rows 2^21 elements apart: the last ones lie past 2^31 elements (4 GiB) from the first."""
    from slimkv_amd import cache_ops
    g, N, D, step = gen(6), 1100, 128, 1 << 21
    store = torch.empty(N * step, dtype=torch.bfloat16, device='cuda')
    big = store.view(1, N, step)
    k, v = randn(g, 1, N, 1, D), randn(g, 1, N, 1, D)
    big[:, :, :D], big[:, :, D:2 * D] = k[:, :, 0], v[:, :, 0]
    kk, vv = big[:, :, None, :D], big[:, :, None, D:2 * D]
    q, dk, dv = randn(g, 1, 3, 4, D), randn(g, 1, 3, 1, D), randn(g, 1, 3, 1, D)
    out, lse = cache_ops.tree_attention(q, dk, dv, D ** -0.5, kk, vv)
    same, lse2 = cache_ops.tree_attention(q, dk, dv, D ** -0.5, k, v)
    assert torch.equal(out, same) and torch.equal(lse, lse2)
    w = cache_ops.attention_weights(q, lse, D ** -0.5, kk)
    assert torch.equal(w, cache_ops.attention_weights(q, lse, D ** -0.5, k))
    rows, counts = cache_ops.select_rows(w, 300, sink=2, recent=20)
    a, b = cache_ops.compact_rows(rows, counts, kk, vv)[:2], cache_ops.compact_rows(rows, counts, k, v)[:2]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('block', [1, 5, 16])
@pytest.mark.parametrize('T,dtype', [(1, 'bf16'), (40, 'fp16')])
def test_long_runs_over_small_pages(T, dtype, block):
    """Runs longer than the stretch of page numbers kept in LDS: the bits of the same rows given densely."""
    from slimkv_amd import cache_ops
    B, H, D, N, g, dt = 2, 4, 64, 140001, gen(8), TYPES[dtype]
    k, v = randn(g, B, N, H, D, dtype=dt), randn(g, B, N, H, D, dtype=dt)
    cols = -(-N // block)
    table = torch.randperm(B * cols, generator=g, device='cuda').view(B, cols)
    pages = torch.zeros(B * cols, block, 2, H, D, dtype=dt, device='cuda')
    for b in range(B):
        rows = torch.zeros(cols * block, 2, H, D, dtype=dt, device='cuda')
        rows[:N, 0], rows[:N, 1] = k[b], v[b]
        pages[table[b]] = rows.view(cols, block, 2, H, D)
    lengths = lengths_of([N, 70003])
    q = randn(g, B, T, 2 * H, D, dtype=dt)
    dk, dv = randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    want = cache_ops.tree_attention(q, dk, dv, 0.125, k, v, lengths=lengths)
    got = cache_ops.tree_attention(q, dk, dv, 0.125, pages=pages, table=table, keys=N, lengths=lengths)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w = cache_ops.attention_weights(q, want[1], 0.125, k, lengths=lengths)
    assert torch.equal(cache_ops.attention_weights(q, want[1], 0.125, pages=pages, table=table, keys=N, lengths=lengths), w)


def test_the_widest_tree_and_no_wider():
    from slimkv_amd import cache_ops
    g, D, T = gen(9), 64, 1024
    q, dk, dv, k = (randn(g, 1, n, 1, D) for n in (T, T, T, 70))
    out, lse = cache_ops.tree_attention(q, dk, dv, 0.125, k, k)
    rows = torch.tensor([0, 1, 500, 1023], device='cuda')
    keys = torch.cat([k, dk], 1)[0, :, 0].double().cpu()
    values = torch.cat([k, dv], 1)[0, :, 0].double().cpu()
    for t in rows.tolist():
        s = (keys[:70 + t + 1] @ q[0, t, 0].double().cpu()) * 0.125
        e = torch.softmax(s, 0) @ values[:70 + t + 1]
        assert (out[0, t, 0].double().cpu() - e).abs().max() <= 2.0 ** -7 * values.abs().max()
        assert abs(lse[0, 0, t].item() - torch.logsumexp(s, 0).item()) <= 1e-4
    wide = randn(g, 1, T + 1, 1, D)
    with pytest.raises(ValueError):
        cache_ops.tree_attention(wide, wide, wide, 0.125, k, k)


def test_pages_without_rows():
    from slimkv_amd import cache_ops
    g, D = gen(10), 128
    pages = torch.full((4, 16, 2, 2, D), float('nan'), dtype=torch.bfloat16, device='cuda')
    table = torch.full((1, 2), 99, dtype=torch.int64, device='cuda')        # no entry is read
    q, dk, dv = randn(g, 1, 3, 4, D), randn(g, 1, 3, 2, D), randn(g, 1, 3, 2, D)
    out, lse = cache_ops.tree_attention(q, dk, dv, D ** -0.5, pages=pages, table=table, keys=0)
    none = torch.zeros(1, 0, 2, D, dtype=torch.bfloat16, device='cuda')
    check_tree(out, lse, q, none, none, None, dk, dv, None, D ** -0.5)
    again, _ = cache_ops.tree_attention(q, dk, dv, D ** -0.5, pages=pages, table=table, lengths=lengths_of([0]))
    assert torch.equal(again, out)
    assert not cache_ops.attention_weights(q, lse, 1.0, pages=pages, table=table, lengths=lengths_of([0])).any()


def test_two_streams_at_once():
    """The same calls on two streams side by side, each with its own workspace."""
    from slimkv_amd import cache_ops
    a, b = step_inputs(71)[0], step_inputs(72)[0]
    want = [run_step(cache_ops, a), run_step(cache_ops, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    words = [torch.zeros(1, dtype=torch.int32, device='cuda') for _ in streams]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                got[i].append(run_step(cache_ops, s, words[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_tree_empty_calls():
    from slimkv_amd import cache_ops
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device='cuda')
    out, lse = cache_ops.tree_attention(z(2, 0, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), 1.0, z(2, 9, 2, 64), z(2, 9, 2, 64))
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    out, lse = cache_ops.tree_attention(z(0, 3, 4, 64), z(0, 3, 2, 64), z(0, 3, 2, 64), 1.0, z(0, 9, 2, 64), z(0, 9, 2, 64))
    assert out.shape == (0, 3, 4, 64)


WEIGHTS = [
    # B, L, Hq, Hkv, D, N, lengths, block, dtype, causal, previous
    (1, 1, 8, 2, 128, 1, None, 0, 'bf16', True, False),
    (2, 1, 32, 8, 128, 517, [517, 0], 16, 'bf16', True, True),
    (2, 5, 14, 2, 64, 200, [200, 3], 48, 'fp16', True, True),
    (1, 32, 10, 2, 128, 333, None, 0, 'bf16', True, False),
    (2, 70, 8, 4, 128, 129, [129, 128], 0, 'fp16', True, True),
    (2, 65, 4, 4, 64, 300, [300, 64], 1, 'bf16', False, True),
    (1, 200, 4, 1, 128, 257, [201], 3, 'bf16', True, True),
    (3, 9, 6, 2, 64, 131, [131, 7, 130], 16, 'bf16', True, True),
    (67, 18, 8, 2, 64, 300, [(13 * i) % 301 for i in range(67)], 16, 'bf16', True, True),
    (2, 130, 8, 2, 128, 1400, [1400, 611], 0, 'fp16', True, True),
    (1, 40, 6, 1, 128, 3001, None, 48, 'bf16', True, False),
    (2, 19, 7, 1, 64, 515, [515, 100], 0, 'bf16', False, True),
]


@pytest.mark.parametrize('case', WEIGHTS, ids=[str(i) for i in range(len(WEIGHTS))])
def test_attention_weights(case):
    from slimkv_amd import cache_ops
    B, L, Hq, H, D, N, lengths, block, dtype, causal, with_previous = case
    print(case, flush=True)
    dt, g, scale = TYPES[dtype], gen(11), D ** -0.5
    k, v, place = make_cache(g, B, N, H, D, block, dt)
    place.pop('v', None)
    q = randn(g, B, L, Hq, D, dtype=dt, gain=1.5)
    lse = torch.randn(B, Hq, L, generator=g, device='cuda') + 4.0
    lse[:, :, ::7] = float('-inf')
    previous = torch.rand(B, H, N, generator=g, device='cuda') if with_previous else None
    n = [N] * B if lengths is None else lengths
    got = cache_ops.attention_weights(q, lse, scale, causal=causal, previous=previous, lengths=lengths_of(lengths), **place)
    want, added, top, mass = oc.attention_weights(f64(q), lse.double().cpu().numpy(), f64(k), n, scale, causal,
                                                  None if previous is None else previous.double().cpu().numpy())
    d = 2.0 ** -24 * (D + 8) * mass + 2.0 ** -21 * (1 + top)      # relative error of one weight
    tol = added * (2 * d + 2.0 ** -24 * (L * Hq // H + 80)) + 2.0 ** -23 * np.abs(want) + 1e-37
    err = np.abs(got.double().cpu().numpy() - want)
    print('worst over its bound', (err / tol).max() if err.size else 0, flush=True)
    assert (err <= tol).all()
    for b in range(B):
        if previous is not None:
            assert torch.equal(got[b, :, n[b]:], previous[b, :, n[b]:])
        else:
            assert not got[b, :, n[b]:].any()
    if previous is not None:
        mine = previous.clone()
        same = cache_ops.attention_weights(q, lse, scale, causal=causal, previous=mine, out=mine,
                                           lengths=lengths_of(lengths), **place)
        assert same is mine and torch.equal(same, got)


def test_weights_of_unseen_rows():
    """NaN in cache rows that no counted query sees, queries that are padding."""
    from slimkv_amd import cache_ops
    g, D = gen(12), 128
    k, q = randn(g, 1, 100, 2, D), randn(g, 1, 6, 4, D)
    lse = torch.zeros(1, 4, 6, device='cuda')
    lse[..., :3] = float('-inf')
    q[:, :3] = float('nan')
    lengths = lengths_of([90])
    clean = cache_ops.attention_weights(q, lse, D ** -0.5, k, lengths=lengths)
    assert torch.isfinite(clean).all() and not clean[:, :, 90:].any()
    k[:, 90:] = float('nan')
    assert torch.equal(cache_ops.attention_weights(q, lse, D ** -0.5, k, lengths=lengths), clean)
    k[:, 89] = float('inf')              # seen by the last query only
    got = cache_ops.attention_weights(q, lse, D ** -0.5, k, lengths=lengths)
    assert torch.equal(got[:, :, :89], clean[:, :, :89])


def test_no_queries_and_no_rows():
    from slimkv_amd import cache_ops
    k = torch.zeros(2, 5, 2, 64, dtype=torch.float16, device='cuda')
    previous = torch.rand(2, 2, 5, device='cuda')
    q, lse = torch.zeros(2, 0, 4, 64, dtype=torch.float16, device='cuda'), torch.zeros(2, 4, 0, device='cuda')
    assert torch.equal(cache_ops.attention_weights(q, lse, 1.0, k, previous=previous), previous)
    assert cache_ops.attention_weights(q, lse, 1.0, k[:, :0]).shape == (2, 2, 0)
    rows, counts = cache_ops.select_rows(previous[:, :, :0], 3)
    assert (rows == -1).all() and not counts.any()


SELECT = [
    # B, H, N, keep, lengths, sink, recent
    (1, 1, 1, 1, None, 0, 0),
    (1, 2, 10, 4, None, 1, 1),
    (2, 2, 100, 40, [100, 39], 4, 8),
    (3, 1, 1000, 64, [1000, 65, 64], 0, 64),
    (2, 3, 4097, 1024, [4097, 2000], 3, 100),
    (1, 2, 5000, 4999, None, 0, 0),
    (1, 1, 70001, 513, None, 4, 32),
    (1, 1, 300, 1, None, 0, 0),
    (2, 1, 20000, 3000, [20000, 9001], 5, 40),
    (1, 3, 40007, 20001, [40000], 0, 0),
    (130, 2, 9001, 100, [(97 * i) % 9002 for i in range(130)], 2, 3),
    (2, 2, 32768, 30000, [32768, 30001], 0, 1),
    (1, 2, 32769, 8000, None, 1, 0),
    (1030, 1, 33001, 100, [33001 - i if i % 103 == 0 else (7 * i) % 400 for i in range(1030)], 4, 8),
]


@pytest.mark.parametrize('case', SELECT, ids=[str(i) for i in range(len(SELECT))])
@pytest.mark.parametrize('values', ['spread', 'ties', 'special'])
def test_select_rows(case, values):
    from slimkv_amd import cache_ops
    B, H, N, keep, lengths, sink, recent = case
    g = gen(21)
    w = torch.exp(torch.randn(B, H, N, generator=g, device='cuda') * 3)
    if values == 'ties':
        w = (w * 2).floor().clamp(max=4.0)
    if values == 'special':
        pick = torch.rand(B, H, N, generator=g, device='cuda')
        for at, x in enumerate((0.0, -0.0, float('nan'), float('inf'), float('-inf'), -1.5, 1e-45)):
            w[(pick > 0.1 * at) & (pick < 0.1 * at + 0.09)] = x
    rows, counts = cache_ops.select_rows(w, keep, lengths=lengths_of(lengths), sink=sink, recent=recent)
    er, ec = oc.select_rows(w.cpu().numpy(), keep, [N] * B if lengths is None else lengths, sink, recent)
    assert (counts.cpu().numpy() == ec).all()
    assert (rows.cpu().numpy() == er).all()


COMPACT = [
    # B, H, D, N, keep, shared, block, dtype
    (1, 2, 128, 40, 11, False, 0, 'bf16'),
    (2, 3, 64, 133, 64, True, 16, 'bf16'),
    (2, 8, 128, 700, 257, False, 48, 'fp16'),
    (1, 1, 128, 300, 300, False, 1, 'bf16'),
    (3, 2, 64, 90, 33, True, 0, 'fp16'),
    (1, 2, 128, 9000, 4500, False, 16, 'bf16'),
    (8, 8, 128, 2900, 2300, False, 32, 'fp16'),
    (1, 1, 64, 20000, 18001, False, 0, 'bf16'),
]


@pytest.mark.parametrize('case', COMPACT, ids=[str(i) for i in range(len(COMPACT))])
@pytest.mark.parametrize('in_place', [False, True])
def test_compact_rows(case, in_place):
    from slimkv_amd import cache_ops
    B, H, D, N, keep, shared, block, dtype = case
    g = gen(31)
    k, v, place = make_cache(g, B, N, H, D, block, TYPES[dtype])
    keys = place.pop('keys', None)
    Hw = 1 if shared else H
    w = torch.rand(B, Hw, N, generator=g, device='cuda')
    lengths = [N - 17 * b for b in range(B)]
    if B > 1:
        lengths[-1] = keep // 2
    rows, counts = cache_ops.select_rows(w, keep, lengths=lengths_of(lengths), sink=2, recent=5)
    r, c = rows.cpu().numpy(), counts.cpu().numpy()
    ek, ev = (oc.compact_rows(r, c, bits(x), keep) for x in (k, v))
    ew = oc.compact_rows(r, c, w.transpose(1, 2).cpu().numpy(), keep).transpose(0, 2, 1)
    before = place['pages'].clone() if block else None
    gk, gv, gw = cache_ops.compact_rows(rows, counts, weights=w, in_place=in_place, **place)
    if not in_place:
        assert (bits(gk) == ek).all() and (bits(gv) == ev).all() and (gw.cpu().numpy() == ew).all()
        if block:
            assert torch.equal(place['pages'].view(torch.int16), before.view(torch.int16))
        return
    assert gw is w
    kk, vv = bits(k), bits(v)                         # dense rows: moved in these tensors
    if block:
        assert gk is None and gv is None
        got = bits(place['pages'])
        table = place['table'].cpu().numpy()
        kk, vv = oc.dense_rows(got, table, N)
        untouched = np.ones(got.shape[0], bool)
        untouched[table.reshape(-1)] = False
        assert (got[untouched] == bits(before)[untouched]).all()
    for b in range(B):
        assert (kk[b, :c[b]] == ek[b, :c[b]]).all() and (vv[b, :c[b]] == ev[b, :c[b]]).all()
        if block:
            old = oc.dense_rows(bits(before), table, N)
            assert (kk[b, c[b]:] == old[0][b, c[b]:]).all() and (vv[b, c[b]:] == old[1][b, c[b]:]).all()
    assert (w.cpu().numpy()[:, :, :keep] == ew).all() and not w[:, :, keep:].any()


def test_nothing_kept_in_place():
    from slimkv_amd import cache_ops
    g = gen(34)
    k, v, _ = make_cache(g, 2, 9, 2, 64, 0, torch.bfloat16)
    before, w = k.clone(), torch.rand(2, 2, 9, generator=g, device='cuda')
    for keep in (0, 3):
        rows = torch.zeros(2, 2, keep, dtype=torch.int32, device='cuda')
        cache_ops.compact_rows(rows, torch.zeros(2, dtype=torch.int32, device='cuda'), k, v, weights=w, in_place=True)
        assert torch.equal(k, before) and not w.any()
        w.fill_(1.0)


def test_compact_reports_bad_rows():
    from slimkv_amd import cache_ops
    g, D = gen(32), 64
    k, v, _ = make_cache(g, 1, 20, 2, D, 0, torch.bfloat16)
    rows = torch.tensor([[[3, 20, 5], [-1, 7, 7]]], dtype=torch.int32, device='cuda')
    counts = torch.tensor([3], dtype=torch.int32, device='cuda')
    with pytest.raises(IndexError):
        cache_ops.compact_rows(rows, counts, k, v)
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    ok, ov, _ = cache_ops.compact_rows(rows, counts, k, v, status=status)
    assert status.item() != 0
    assert torch.equal(ok[0, 0, 0], k[0, 3, 0]) and not ok[0, 1, 0].any() and not ov[0, 0, 1].any()
    assert torch.equal(ok[0, 1, 1], k[0, 7, 1]) and torch.equal(ok[0, 2, 1], k[0, 7, 1])
    before = k.clone(), v.clone()
    with pytest.raises(IndexError):                    # out of order in place
        cache_ops.compact_rows(rows, counts, k, v, in_place=True)
    assert torch.equal(k[0, 3:], before[0][0, 3:])


@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('held', [0, 4])
def test_weights_shorter_than_the_choice(held, in_place):
    from slimkv_amd import cache_ops
    g = gen(35)
    k, v, _ = make_cache(g, 1, 9, 2, 64, 0, torch.bfloat16)
    w = torch.rand(1, 2, held, generator=g, device='cuda')
    rows = torch.tensor([[[0, 2, 5, 8], [1, 2, 3, 4]]], dtype=torch.int32, device='cuda')
    counts = torch.tensor([4], dtype=torch.int32, device='cuda')
    before, kept = k.clone(), w.clone()
    with pytest.raises(IndexError):
        cache_ops.compact_rows(rows, counts, k, v, weights=w, in_place=in_place)
    if in_place:                                       # rows that the cache has are moved all the same
        assert torch.equal(k[0, :4, 0], before[0, [0, 2, 5, 8], 0])
        if held:
            assert torch.equal(w[0, 0, :2], kept[0, 0, [0, 2]]) and torch.equal(w[0, 1, :3], kept[0, 1, 1:4])
    else:
        assert torch.equal(k, before) and torch.equal(w, kept)


def test_bad_pages_are_reported():
    from slimkv_amd import cache_ops
    g, D = gen(33), 128
    k, v, place = make_cache(g, 2, 70, 2, D, 16, torch.bfloat16)
    place['table'][1, 2] = place['pages'].shape[0]
    q, dk, dv = randn(g, 2, 3, 4, D), randn(g, 2, 3, 2, D), randn(g, 2, 3, 2, D)
    with pytest.raises(IndexError):
        cache_ops.tree_attention(q, dk, dv, 1.0, lengths=lengths_of([70, 70]), **place)
    # the entry is not needed where the sequence ends before it
    out, lse = cache_ops.tree_attention(q, dk, dv, D ** -0.5, lengths=lengths_of([70, 32]), **place)
    check_tree(out, lse, q, k, v, [70, 32], dk, dv, None, D ** -0.5)
    with pytest.raises(IndexError):
        cache_ops.attention_weights(q, lse, 1.0, **place)
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    cache_ops.attention_weights(q, lse, 1.0, status=status, **place)
    assert status.item() != 0
    rows = torch.tensor([[[1, 2]], [[3, 40]]], dtype=torch.int32, device='cuda')
    counts = torch.tensor([2, 2], dtype=torch.int32, device='cuda')
    place.pop('keys')
    with pytest.raises(IndexError):
        cache_ops.compact_rows(rows, counts, **place)


def run_step(cache_ops, s, status=None):
    """A speculative step over a paged cache brought back to its budget."""
    out, lse = cache_ops.tree_attention(s['q'], s['dk'], s['dv'], s['scale'], pages=s['pages'], table=s['table'],
                                        lengths=s['lengths'], mask=s['mask'], status=status)
    w = cache_ops.attention_weights(s['q'], lse, s['scale'], pages=s['pages'], table=s['table'], lengths=s['lengths'],
                                    previous=s['weights'], causal=False, status=status)
    rows, counts = cache_ops.select_rows(w, s['keep'], lengths=s['lengths'], sink=2, recent=8)
    k, v, kept = cache_ops.compact_rows(rows, counts, pages=s['pages'], table=s['table'], weights=w, status=status)
    return out, lse, w, rows, counts, k, v, kept


def step_inputs(seed, B=3, T=6, Hq=8, H=2, D=128, N=300):
    g = gen(seed)
    k, v, place = make_cache(g, B, N, H, D, 16, torch.bfloat16)
    cols = place['table'].shape[1]
    s = dict(pages=place['pages'], table=place['table'], lengths=lengths_of([300, 77, 12]), scale=D ** -0.5, keep=64,
             q=randn(g, B, T, Hq, D), dk=randn(g, B, T, H, D), dv=randn(g, B, T, H, D), mask=tree_mask(g, B, T, 'tree'),
             weights=torch.rand(B, H, cols * 16, generator=g, device='cuda'))
    return s, k, v


def test_graph_replays_a_step():
    """A captured step replayed with new inputs and eager work between the replays."""
    from slimkv_amd import cache_ops
    s, _, _ = step_inputs(41)
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_step(cache_ops, s, status)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_step(cache_ops, s, status)
    for seed in (42, 43, 44):
        fresh, _, _ = step_inputs(seed)
        for name in ('pages', 'table', 'q', 'dk', 'dv', 'mask', 'weights'):
            s[name].copy_(fresh[name])
        s['lengths'].copy_(lengths_of([300 - seed, 65, seed]))
        graph.replay()
        torch.cuda.synchronize()
        want = run_step(cache_ops, s, status)
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.int16) if a.dtype is torch.bfloat16 else a,
                               b.view(torch.int16) if b.dtype is torch.bfloat16 else b)
    assert status.item() == 0


def test_capture_without_a_status_word_is_refused():
    from slimkv_amd import cache_ops
    s, _, _ = step_inputs(45)
    run_step(cache_ops, s)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match='status'):
        with torch.cuda.graph(graph):
            run_step(cache_ops, s)


def test_side_stream():
    from slimkv_amd import cache_ops
    s, _, _ = step_inputs(46)
    want = run_step(cache_ops, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_step(cache_ops, s)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_speculative_steps_over_a_bounded_paged_cache():
    """Verify a draft, commit the accepted path into the pages, weigh the rows with the path's own queries, evict in
    place when over budget; outputs and weights against the plain forms on the rows the cache then holds."""
    from slimkv_amd import cache_ops, kernels
    g, B, T, Hq, H, D, block, budget = gen(51), 2, 5, 8, 2, 128, 16, 48
    scale, cols = D ** -0.5, 6
    pool = torch.randperm(B * cols, generator=g, device='cuda').view(B, cols)
    pages = torch.full((B * cols, block, 2, H, D), float('nan'), dtype=torch.bfloat16, device='cuda')
    held = [[], []]                                    # plain form: the rows each head holds, per sequence
    lengths = torch.tensor([30, 41], dtype=torch.int32, device='cuda')
    first_k, first_v = randn(g, B, H, 41, D), randn(g, B, H, 41, D)
    kernels.raw_pages(pages, pool, first_k, first_v, start=0, count=41, to_pages=True, lengths=lengths)
    plain_k = [f64(first_k[b, :, :int(lengths[b])]) for b in range(B)]
    plain_v = [f64(first_v[b, :, :int(lengths[b])]) for b in range(B)]
    weights = torch.zeros(B, H, cols * block, device='cuda')
    mask = torch.eye(T, dtype=torch.bool, device='cuda')
    for t, parent in ((1, 0), (2, 0), (3, 1), (4, 3)):
        mask[t] |= mask[parent]
    path = torch.tensor([0, 1, 3], device='cuda')      # the accepted chain
    evicted = 0
    for step in range(6):
        q = randn(g, B, T, Hq, D)
        dk, dv = randn(g, B, T, H, D), randn(g, B, T, H, D)
        out, lse = cache_ops.tree_attention(q, dk, dv, scale, pages=pages, table=pool, lengths=lengths, mask=mask)
        for b in range(B):
            n = int(lengths[b])
            k = torch.from_numpy(plain_k[b]).transpose(0, 1)[None].cuda()
            v = torch.from_numpy(plain_v[b]).transpose(0, 1)[None].cuda()
            check_tree(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, [n], dk[b:b + 1], dv[b:b + 1], mask, scale)
        new_k, new_v = (x[:, path].transpose(1, 2).contiguous() for x in (dk, dv))
        kernels.raw_pages(pages, pool, new_k, new_v, start=0, count=3, to_pages=True, starts=lengths.long())
        lengths += 3
        plain_k = [np.concatenate([a, f64(new_k[b])], 1) for b, a in enumerate(plain_k)]
        plain_v = [np.concatenate([a, f64(new_v[b])], 1) for b, a in enumerate(plain_v)]
        before = weights.clone()
        cache_ops.attention_weights(q[:, path], lse[:, :, path].contiguous(), scale, pages=pages, table=pool,
                                    lengths=lengths, previous=weights, out=weights)
        # every accepted query gave its whole attention to the rows it sees
        added = (weights - before).sum(-1)
        assert torch.allclose(added, torch.full_like(added, 3.0 * Hq / H), rtol=1e-4)
        rows, counts = cache_ops.select_rows(weights, budget, lengths=lengths, sink=2, recent=8)
        r, c = oc.select_rows(weights.cpu().numpy(), budget, lengths.tolist(), 2, 8)
        assert (rows.cpu().numpy() == r).all()
        evicted += int((lengths - counts).sum())
        cache_ops.compact_rows(rows, counts, pages=pages, table=pool, weights=weights, in_place=True)
        plain_k = [np.stack([a[h, r[b, h, :c[b]]] for h in range(H)]) for b, a in enumerate(plain_k)]
        plain_v = [np.stack([a[h, r[b, h, :c[b]]] for h in range(H)]) for b, a in enumerate(plain_v)]
        lengths.copy_(counts)
    assert evicted > 0


def test_gradients_are_refused():
    from slimkv_amd import cache_ops
    q, k = randn(gen(61), 1, 2, 4, 64), randn(gen(62), 1, 2, 2, 64)
    q.requires_grad_()
    with pytest.raises(ValueError, match='gradient'):
        cache_ops.tree_attention(q, k, k, 1.0, k, k)
    with torch.no_grad():
        cache_ops.tree_attention(q, k, k, 1.0, k, k)


def test_torch_operators():
    import slimkv_amd.torch_ops  # noqa: F401
    s, _, _ = step_inputs(63)
    ops, status = torch.ops.slimkv, torch.zeros(1, dtype=torch.int32, device='cuda')
    want = run_step(__import__('slimkv_amd.cache_ops', fromlist=['x']), s)
    tree = (s['q'], s['dk'], s['dv'], s['scale'], None, None, s['pages'], s['table'], s['lengths'], None, s['mask'], status)
    torch.library.opcheck(ops.tree_attention.default, tree)
    out, lse = ops.tree_attention(*tree)
    weigh = (s['q'], lse, s['scale'], None, s['pages'], s['table'], s['lengths'], None, False, s['weights'], status)
    torch.library.opcheck(ops.attention_weights.default, weigh)
    w = ops.attention_weights(*weigh)
    torch.library.opcheck(ops.select_rows.default, (w, s['keep'], s['lengths'], 2, 8))
    rows, counts = ops.select_rows(w, s['keep'], s['lengths'], 2, 8)
    move = (rows, counts, None, None, s['pages'], s['table'], w, status)
    torch.library.opcheck(ops.compact_rows.default, move)
    got = (out, lse, w, rows, counts, *ops.compact_rows(*move))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('T', [2, 30, 70])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_scores_of_a_thousand_million_and_more(T, dtype):
    """Scores whose products with the scale are rounded to steps of 64 to 2^24: two equal ones in different tiles share
    the row, all others are nothing.  The LSE takes four roundings: of the scale and of ln 2, of the products with
    them."""
    from slimkv_amd import cache_ops
    D, N, dt = 128, 300, TYPES[dtype]
    q = torch.full((1, T, 2, D), 3001.0, dtype=dt, device='cuda')
    k = torch.zeros(1, N, 2, D, dtype=dt, device='cuda')
    k[:, 7], k[:, 100], k[:, 200] = 2999.0, -2999.0, 2999.0
    v = torch.full((1, N, 2, D), 100.0, dtype=dt, device='cuda')
    v[:, 7], v[:, 200] = 1.5, 4.5
    nothing = torch.zeros(T, T, dtype=torch.bool, device='cuda')
    for scale in (1.0, 1.7, 0.0931, 1e5):
        out, lse = cache_ops.tree_attention(q, k[:, :T], v[:, :T], scale, k, v, mask=nothing)
        assert (out == 3.0).all(), scale
        s = D * float(q[0, 0, 0, 0]) * float(k[0, 7, 0, 0]) * scale
        assert (lse.double() - s).abs().max() <= s * 2.0 ** -22 + 1.0, scale


@pytest.mark.parametrize('T', [1, 20, 40, 70])
@pytest.mark.parametrize('ahead', [12.0, 17.5, 22.0])
def test_fp16_rows_far_behind_the_first_keep_their_weight(T, ahead):
    """One row `ahead` nats before thousands of equal ones whose values alone are not zero, every item in one run.
    Weights are held 2^15 times as large as their share of the row's largest, so the half step 2^-25 of fp16's
    subnormals is 2^-40 of it: 2^-40 max|v| a key, divided by the row's sum.  The output may be subnormal too."""
    from slimkv_amd import cache_ops
    B, H, D, N, g, dt = 64, 8, 128, 2003, gen(73), torch.float16
    scale = D ** -0.5
    q = torch.full((1, T, H, D), 2.0, dtype=dt, device='cuda')
    k = torch.zeros(1, N, H, D, dtype=dt, device='cuda')
    k[:, 0] = ahead / (2.0 * D * scale)
    v = (500.0 + 50.0 * torch.randn(1, N, H, D, generator=g, device='cuda')).to(dt)
    v[:, 0] = 0.0
    dk, dv = torch.zeros(1, T, H, D, dtype=dt, device='cuda'), v[:, 1:T + 1].clone()
    every = lambda x: x.expand(B, -1, -1, -1)
    out, lse = cache_ops.tree_attention(every(q), every(dk), every(dv), scale, every(k), every(v))
    eo, el, terms, top, mass, total = oc.tree_attention(f64(q), f64(k), f64(v), [N], f64(dk), f64(dv), None, scale)
    d = 2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top)
    of_rows = lambda x: x.transpose(0, 2, 1)[..., None]
    u = HALF[dt]
    tol = (2 * of_rows(d) + u) * terms + u * np.abs(eo) * (1 + u) + 2.0 ** -25 + \
        2.0 ** -40 * (N + T) * np.abs(f64(v)).max() / of_rows(total)
    err = np.abs(f64(out) - eo)
    print('expected', eo.min(), eo.max(), 'worst error over its bound', (err / tol).max(), flush=True)
    assert (err <= tol).all()
    tl = d + 2.0 ** -24 * ((N + T) / 4 + 64) + 2.0 ** -21 * (1 + np.abs(el))
    assert (np.abs(lse.double().cpu().numpy() - el) <= tl).all()


def test_outputs_interleaved_with_other_tensors():
    """The output beside q, the moved K and V as halves of one tensor, the sums beside what they are added to."""
    from slimkv_amd import cache_ops
    B, T, Hq, H, D, N, keep, g = 2, 3, 8, 2, 64, 40, 16, gen(75)
    k, v, _ = make_cache(g, B, N, H, D, 0, torch.bfloat16)
    both, sums = randn(g, B, T, Hq, 2, D), torch.rand(B, H, 2, N, generator=g, device='cuda')
    dk, dv = randn(g, B, T, H, D), randn(g, B, T, H, D)
    q, before = both[:, :, :, 0], both.clone()
    want, lse = cache_ops.tree_attention(q.contiguous(), dk, dv, 0.125, k, v)
    got, _ = cache_ops.tree_attention(q, dk, dv, 0.125, k, v, out=both[:, :, :, 1])
    assert torch.equal(got, want) and torch.equal(q, before[:, :, :, 0])
    kept = sums[:, :, 0].clone()
    want = cache_ops.attention_weights(q, lse, 0.125, k, previous=kept, causal=False)
    w = cache_ops.attention_weights(q, lse, 0.125, k, previous=sums[:, :, 0], out=sums[:, :, 1], causal=False)
    assert torch.equal(w, want) and torch.equal(sums[:, :, 0], kept)
    rows, counts = cache_ops.select_rows(w, keep)
    halves = torch.empty(B, keep, 2, H, D, dtype=torch.bfloat16, device='cuda')
    want = cache_ops.compact_rows(rows, counts, k, v)
    cache_ops.compact_rows(rows, counts, k, v, out_k=halves[:, :, 0], out_v=halves[:, :, 1])
    assert torch.equal(halves[:, :, 0], want[0]) and torch.equal(halves[:, :, 1], want[1])


def test_more_query_rows_than_runs():
    """Blocks of query rows past two workgroups a CU: one run, no partial results, no workspace."""
    from slimkv_amd import _lib, cache_ops
    B, T, Hq, D, N, g = 2, 1024, 40, 64, 150, gen(76)
    assert _lib.lib().slimkv_tree_attention_workspace(_lib.ctypes.byref(_lib.TreeAttentionArgs(
        q=16, batch=B, drafted=T, heads=Hq, kv_heads=1, head_dim=D, scale=1.0))) == 16
    k, v = randn(g, B, N, 1, D), randn(g, B, N, 1, D)
    q, dk, dv = randn(g, B, T, Hq, D), randn(g, B, T, 1, D), randn(g, B, T, 1, D)
    mask = tree_mask(g, B, T, 'rows')
    out, lse = cache_ops.tree_attention(q, dk, dv, 0.125, k, v, lengths=lengths_of([N, 0]), mask=mask)
    for b, n in enumerate((N, 0)):
        for t in (0, 1, 333, 700, 1023):
            sees = mask[b, t].cpu().numpy()
            eo, el, terms, top, mass, total = oc.tree_attention(
                f64(q[b:b + 1, t:t + 1]), f64(k[b:b + 1]), f64(v[b:b + 1]), [n], f64(dk[b:b + 1])[:, sees],
                f64(dv[b:b + 1])[:, sees], np.ones((1, int(sees.sum())), bool), 0.125)
            u = HALF[q.dtype]
            d = (2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top)).transpose(0, 2, 1)[..., None]
            assert (np.abs(f64(out[b:b + 1, t:t + 1]) - eo) <= (2 * d + u) * terms + u * np.abs(eo) * (1 + u) + 1e-30).all()
            got = lse[b, :, t].double().cpu().numpy()
            assert (np.isneginf(got) == np.isneginf(el[0, :, 0])).all()
            seen = ~np.isneginf(got)
            assert (np.abs(got[seen] - el[0, seen, 0]) <= 1e-4).all()


def long_step_inputs(seed):
    """A step whose weights are split over query rows and whose selection cuts rows into chunks: both with workspaces."""
    from slimkv_amd import cache_ops
    B, T, Hq, H, D, N, g = 2, 128, 8, 2, 64, 33100, gen(seed)
    pages, cols = randn(g, B * 2100, 16, 2, H, D), 2069
    table = torch.randperm(B * 2100, generator=g, device='cuda')[:B * cols].view(B, cols)
    lengths = lengths_of([N - seed, 32900 + seed])
    s = dict(pages=pages, table=table, lengths=lengths, scale=D ** -0.5, keep=5000, q=randn(g, B, T, Hq, D),
             dk=randn(g, B, T, H, D), dv=randn(g, B, T, H, D), mask=tree_mask(g, B, T, 'tree'),
             weights=torch.rand(B, H, cols * 16, generator=g, device='cuda') * 1e-3)
    index = torch.cuda.current_device()
    assert cache_ops._tree_bytes(index, B, T, Hq, H, D) > 16 and cache_ops._weights_bytes(index, B, T, Hq, H, D, cols * 16) > 16
    assert cache_ops._select_bytes(index, B, H, cols * 16, s['keep'], 2, 8) > 16
    return s


def same(got, want):
    return all(torch.equal(a.view(torch.int16) if a.dtype is torch.bfloat16 else a,
                           b.view(torch.int16) if b.dtype is torch.bfloat16 else b) for a, b in zip(got, want))


def test_calls_with_workspaces_side_by_side():
    from slimkv_amd import cache_ops
    inputs = [long_step_inputs(81), long_step_inputs(82)]
    want = [run_step(cache_ops, s) for s in inputs]
    rows, counts = (x.cpu().numpy() for x in want[0][3:5])
    er, ec = oc.select_rows(want[0][2].cpu().numpy(), 5000, inputs[0]['lengths'].tolist(), 2, 8)
    assert (rows == er).all() and (counts == ec).all()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    words = [torch.zeros(1, dtype=torch.int32, device='cuda') for _ in streams]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (s, st) in enumerate(zip(inputs, streams)):
            with torch.cuda.stream(st):
                got[i].append(run_step(cache_ops, s, words[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(same(out, want[i]) for out in got[i]) and words[i].item() == 0


def test_two_graphs_with_workspaces_replayed_side_by_side():
    """Two captured steps, replayed on two streams at once with new inputs and eager work between the replays."""
    from slimkv_amd import cache_ops
    inputs = [long_step_inputs(83), long_step_inputs(84)]
    words = [torch.zeros(1, dtype=torch.int32, device='cuda') for _ in inputs]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, word in zip(inputs, words):
        run_step(cache_ops, s, word)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run_step(cache_ops, s, word))
    for seed in (85, 87, 89):
        for s, add in zip(inputs, (0, 1)):
            fresh = long_step_inputs(seed + add)
            for name in ('pages', 'table', 'lengths', 'q', 'dk', 'dv', 'mask', 'weights'):
                s[name].copy_(fresh[name])
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for s, out, word in zip(inputs, outs, words):
            assert same(out, run_step(cache_ops, s, word)) and word.item() == 0


@pytest.mark.parametrize('T', [30, 70, 130])
@pytest.mark.parametrize('kind', [None, 'tree'])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_visible_infinities_and_nan_reach_the_rows_that_see_them(T, kind, dtype):
    """Drafted values that are not finite, in several tiles: their rows' columns take them, all others are as if they
    were 0."""
    from slimkv_amd import cache_ops
    B, Hq, H, D, N, dt, g = 2, 4, 2, 64, 100, TYPES[dtype], gen(91)
    k, v, place = make_cache(g, B, N, H, D, 0, dt)
    q, dk, dv = randn(g, B, T, Hq, D, dtype=dt), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    mask = tree_mask(g, B, T, kind)
    inf, nan = float('inf'), float('nan')
    wild = [(0, 5, 0, 3, inf), (0, T - 2, 0, 3, -inf), (0, T // 2, 1, 17, nan), (1, T - 1, 1, 63, inf), (1, 0, 0, 0, -inf)]
    clean = dv.clone()
    for b, t, h, c, x in wild:
        dv[b, t, h, c], clean[b, t, h, c] = x, 0.0
    out, lse = cache_ops.tree_attention(q, dk, dv, 0.125, mask=mask, **place)
    sees = torch.ones(B, T, T, dtype=torch.bool).tril() if mask is None else mask.cpu()
    extra = np.zeros((B, T, Hq, D))
    with np.errstate(invalid='ignore'):
        for b, t, h, c, x in wild:
            extra[b, sees[b, :, t].numpy(), h * 2:h * 2 + 2, c] += x
    got = f64(out)
    bad = ~np.isfinite(extra)
    assert bad.sum() > T and np.array_equal(got[bad], extra[bad], equal_nan=True)
    out = torch.where(torch.from_numpy(bad).cuda(), torch.zeros_like(out), out)
    eo, el, terms, top, mass, total = oc.tree_attention(f64(q), f64(k), f64(v), [N] * B, f64(dk), f64(clean),
                                                        None if mask is None else mask.cpu().numpy(), 0.125)
    d = 2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top)
    u = HALF[dt]
    tiny = 2.0 ** -40 * (N + T) * np.abs(f64(clean)).max() / total.transpose(0, 2, 1)[..., None] + 2.0 ** -25 if dt is torch.float16 else 0.0
    tol = (2 * d.transpose(0, 2, 1)[..., None] + u) * terms + u * np.abs(eo) * (1 + u) + tiny
    assert (np.abs(f64(out) - eo)[~bad] <= tol[~bad]).all()
    assert np.isfinite(lse.double().cpu().numpy()).all()


@pytest.mark.parametrize('scale', [0.0, -0.125, 1e19, 1e-19, float('inf'), float('nan')])
def test_softmax_scales_outside_the_range_are_refused(scale):
    from slimkv_amd import cache_ops
    q, k = randn(gen(92), 1, 2, 4, 64), randn(gen(93), 1, 2, 2, 64)
    with pytest.raises(ValueError, match='scale'):
        cache_ops.tree_attention(q, k, k, scale, k, k)
    with pytest.raises(ValueError, match='scale'):
        cache_ops.attention_weights(q, torch.zeros(1, 4, 2, device='cuda'), scale, k)
