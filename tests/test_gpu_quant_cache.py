"""The 4-bit cache on the GPU against its 64-bit plain forms (oracle/quant.py).

Writing and reading are compared bit by bit: the scale is a power of two and every rounding is to the nearest, so
there is one right answer (bf16 holds it exactly; fp16 rounds it once, as numpy does).

Attention takes the bounds of tests/test_gpu_cache_ops.py over the rows that the cache stands for: the conversion to the
element type is exact for the values drawn here, so scores, weights and sums are those of full-width rows.

norm_rope: the sum of D squares is off by at most D 2^-24 of itself (D - 1 additions and D products of half a step
each, all of one sign), the mean's root by half of that and three roundings, y by three more, and the two products of
the rotation by one each with one for their sum: (D / 2 + 16) 2^-24 of |y cos| + |y' sin| in all, then half a step of
the result (fp16 below 2^-14: 2^-25).
"""
import numpy as np
import pytest
import torch

from oracle import quant as oq
from tests.helpers import bits, to_np
from tests.test_gpu_cache_ops import HALF, TYPES, check_tree, gen, lengths_of, randn, tree_mask

pytestmark = pytest.mark.gpu


def ints(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device='cuda')


def scattered(g, B, cols, spare=3):
    """(pool size, table [B, cols] of scattered pages, some entries counted from the pool's end)."""
    count = B * cols + spare
    table = torch.randperm(count, generator=g, device='cuda')[:B * cols].view(B, cols)
    return count, torch.where(torch.arange(cols, device='cuda') % 3 == 1, table - count, table)


def filled_pool(g, B, N, H, D, block, dtype, gain=1.0):
    """A cache whose rows below N of each sequence are quantised noise by the plain form and whose other bytes are
    noise too, NaN scales among them: (pages, table, k, v [B, N, H, D] float32 as the cache stands for them)."""
    dt = TYPES[dtype]
    if block:
        cols = -(-max(N, 1) // block)
        count, table = scattered(g, B, cols)
        order = table.cpu().numpy() % count
        rows = block
    else:
        rows = -(-max(N, 1) // 16) * 16
        count, table, order = B + 1, None, np.arange(B)[:, None]
    pages = torch.randint(0, 256, (count, H, rows * (D + D // 16)), generator=g, device='cuda', dtype=torch.uint8)
    pages[:, :, rows * D:][pages[:, :, rows * D:] > 200] = 255
    p = pages.cpu().numpy()
    k, v = to_np(randn(g, B, N, H, D, dtype=dt, gain=gain)), to_np(randn(g, B, N, H, D, dtype=dt, gain=gain))
    (kc, ks), (vc, vs) = oq.quantize(k, dtype), oq.quantize(v, dtype)
    for b in range(B):
        for n0 in range(0, N, rows):
            at = np.arange(n0, min(N, n0 + rows))
            for h in range(H):
                oq.write_page(p[order[b, n0 // rows], h], at - n0, (kc[b, at, h], ks[b, at, h]), (vc[b, at, h], vs[b, at, h]), D)
    make = lambda c, s: torch.from_numpy(oq.values(c, s)).float().cuda()
    return torch.from_numpy(p).cuda(), table, make(kc, ks), make(vc, vs)


ROWS = [
    # B, n, H, D, block, capacity in rows, starts, counts, dtype
    (1, 1, 1, 128, 0, 16, None, None, 'bf16'),
    (1, 1, 8, 128, 16, 64, [37], None, 'bf16'),
    (2, 5, 2, 64, 16, 48, [0, 43], [5, 2], 'fp16'),
    (3, 40, 3, 128, 32, 96, [0, 13, 56], None, 'fp16'),
    (2, 100, 2, 128, 48, 144, [44, 3], [100, 0], 'bf16'),
    (2, 33, 1, 64, 0, 128, [95, 17], None, 'bf16'),
    (16, 1, 8, 128, 16, 80, [(13 * b) % 80 for b in range(16)], None, 'bf16'),
    (1, 333, 2, 64, 128, 512, [129], [300], 'bf16'),
    (5, 7, 40, 128, 16, 32, None, [7, 1, 0, 3, 7], 'fp16'),
    (300, 2, 1, 64, 16, 16, [b % 15 for b in range(300)], None, 'bf16'),
]


def special(x, dtype):
    """Zeros, signed zeros, subnormals, the largest numbers, ties, infinities and NaN among the rows x."""
    flat = x.view(-1, 32)
    n = flat.shape[0]
    small, large = (2.0 ** -133, 2.0 ** 127 * 1.9921875) if dtype == 'bf16' else (2.0 ** -24, 65504.0)
    kinds = [lambda f: f.zero_(), lambda f: f.mul_(small * 8), lambda f: f.fill_(-0.0), lambda f: f[3:4].fill_(large),
             lambda f: f.copy_(torch.linspace(-7, 8.5, 32)), lambda f: f[31:].fill_(float('inf')),
             lambda f: f[7:8].fill_(float('nan')), lambda f: f.fill_(small), lambda f: f.fill_(-large)]
    for i, kind in enumerate(kinds):
        if n > 3 * i:
            kind(flat[(7 * i + 1) % n])
    return x


@pytest.mark.parametrize('kind', ['noise', 'special'])
@pytest.mark.parametrize('case', ROWS, ids=[str(i) for i in range(len(ROWS))])
def test_rows_written_and_read(case, kind):
    from slimkv_amd import quant_cache
    B, n, H, D, block, capacity, starts, counts, dtype = case
    print(case, kind, flush=True)
    dt, g = TYPES[dtype], gen(41)
    k, v = (randn(g, B, n, H, D, dtype=dt) * torch.exp(randn(g, 1, 1, H, D, gain=2.0).float()).to(dt) for _ in range(2))
    if kind == 'special':
        k, v = special(k, dtype), special(v.flip(1).contiguous(), dtype)
    table, count = None, B + 1
    if block:
        count, table = scattered(g, B, capacity // block)
    pages = torch.randint(0, 256, (count, H, (block or capacity) * (D + D // 16)), generator=g, device='cuda',
                          dtype=torch.uint8)
    want = pages.cpu().numpy().copy()
    order = np.arange(B)[:, None] if table is None else table.cpu().numpy() % count
    rows = block or capacity
    (kc, ks), (vc, vs) = oq.quantize(to_np(k), dtype), oq.quantize(to_np(v), dtype)
    many = [n] * B if counts is None else counts
    first = [0] * B if starts is None else starts
    for b in range(B):
        for i in range(many[b]):
            r = first[b] + i
            for h in range(H):
                oq.write_page(want[order[b, r // rows], h], [r % rows], (kc[b, i:i + 1, h], ks[b, i:i + 1, h]),
                              (vc[b, i:i + 1, h], vs[b, i:i + 1, h]), D)
    got = quant_cache.quantize_rows(k, v, pages, table, starts=ints(starts), counts=ints(counts))
    assert got is pages
    assert (pages.cpu().numpy() == want).all()                       # every other byte as it was
    a, c = quant_cache.dequantize_rows(pages, n, D, table, starts=ints(starts) if starts or table is not None else ints([0] * B),
                                       counts=ints(counts), dtype=dt)
    assert a.dtype is dt and a.shape == c.shape == k.shape
    np16 = (lambda x: x) if dtype == 'bf16' else (lambda x: x.astype(np.float16).astype(np.float64))
    for out, (codes, scales) in ((a, (kc, ks)), (c, (vc, vs))):
        values = np16(oq.values(codes, scales))
        for b in range(B):
            assert np.array_equal(to_np(out)[b, :many[b]], values[b, :many[b]], equal_nan=True)
            assert not bits(out)[b, many[b]:].any()


def test_every_scale_and_code_is_read():
    """All 256 scale bytes with all codes, as bf16 and fp16.  The two largest scales, which no write makes, give numbers
    from 2^128 on, infinities in bf16 as in fp32; all other numbers bf16 holds."""
    from slimkv_amd import quant_cache
    for D in (64, 128):
        block = 256
        page = np.random.default_rng(3).integers(0, 256, (1, 2, block * (D + D // 16)), dtype=np.uint8)
        for h in (0, 1):
            page[0, h, block * D:] = (np.arange(block * D // 16) // (D // 32)) % 256
        want = oq.read_pages(page, D)
        for dt in TYPES.values():
            got = quant_cache.dequantize_rows(torch.from_numpy(page).cuda(), block, D, dtype=dt)
            for x, y in zip(got, want):
                with np.errstate(over='ignore'):
                    y = y.astype(np.float32 if dt is torch.bfloat16 else np.float16).astype(np.float64)
                x = to_np(x)
                assert np.array_equal(x, y, equal_nan=True) and (np.signbit(x) == np.signbit(y))[~np.isnan(y)].all()


def test_rows_given_as_views():
    """K and V as parts of a projection's output, heads first, on odd addresses; outputs inside larger buffers; pages that
    are a part of a larger pool."""
    from slimkv_amd import quant_cache
    g, B, n, H, D, block = gen(42), 2, 21, 3, 128, 16
    whole = randn(g, B, n, 10, D)
    k, v = whole[:, :, 4:7], whole[:, :, 7:]
    count, table = scattered(g, B, 2)
    fresh = quant_cache.new_pages(count, H, block, D)
    quant_cache.quantize_rows(k.contiguous(), v.contiguous(), fresh, table)
    big = torch.full((count, 2 * H + 1, 2176 + 32), 9, dtype=torch.uint8, device='cuda')
    part = big[:, 1::2, :2176][:, :H]
    part.zero_()
    quant_cache.quantize_rows(k, v, part, table)
    assert torch.equal(part, fresh)
    assert (big[:, ::2] == 9).all() and (big[:, :, 2176:] == 9).all()
    for x in (k.transpose(1, 2).contiguous().transpose(1, 2),
              torch.empty(k.numel() + 1, dtype=torch.bfloat16, device='cuda')[1:].view(k.shape).copy_(k)):
        part.zero_()
        quant_cache.quantize_rows(x, v, part, table)
        assert torch.equal(part, fresh)
    assert not quant_cache.new_pages(1, H, block, D).any()
    outs = torch.full((B, H, n + 1, 2, D + 8), 7.0, dtype=torch.bfloat16, device='cuda')
    ok, ov = (outs[:, :, :n, x, :D].transpose(1, 2) for x in (0, 1))
    a, b = quant_cache.dequantize_rows(part, n, D, table, out_k=ok, out_v=ov)
    want = quant_cache.dequantize_rows(fresh, n, D, table)
    assert a is ok and b is ov and torch.equal(ok, want[0]) and torch.equal(ov, want[1])
    assert (outs[:, :, n] == 7).all() and (outs[..., D:] == 7).all()


def test_rows_outside_the_cache_are_reported():
    from slimkv_amd import quant_cache
    from slimkv_amd.kernels import check_status
    g, B, n, H, D, block = gen(43), 3, 10, 2, 64, 16
    k, v = randn(g, B, n, H, D), randn(g, B, n, H, D)
    count, table = scattered(g, B, 2)
    for starts, kept in (([0, 25, 4], 7), ([0, -3, 4], None), ([0, 32, 4], 0), ([0, 2 ** 31 - 5, 4], 0),
                         ([0, -2 ** 31, 4], 0)):
        pages = quant_cache.new_pages(count, H, block, D)
        status = torch.zeros(1, dtype=torch.int32, device='cuda')
        quant_cache.quantize_rows(k, v, pages, table, starts=ints(starts), status=status)
        with pytest.raises(IndexError):
            check_status(status)
        with pytest.raises(IndexError):
            quant_cache.quantize_rows(k, v, pages, table, starts=ints(starts))
        ref = quant_cache.new_pages(count, H, block, D)
        good = [0, 0, 4]
        if kept is not None:
            good[1] = starts[1] if kept else 0
            quant_cache.quantize_rows(k, v, ref, table, starts=ints(good), counts=ints([n, kept, n]))
        else:
            quant_cache.quantize_rows(torch.cat([k[1:2, 3:], k[1:2, :3]], 1), torch.cat([v[1:2, 3:], v[1:2, :3]], 1), ref,
                                      table[1:2], counts=ints([n - 3]))
            quant_cache.quantize_rows(k[::2].contiguous(), v[::2].contiguous(), ref, table[::2].contiguous(), starts=ints([0, 4]))
        assert torch.equal(pages, ref)
        status.zero_()
        a, _ = quant_cache.dequantize_rows(pages, n, D, table, starts=ints(starts), status=status)
        assert status.item() != 0
        inside = [0 <= starts[1] + i < 32 for i in range(n)]
        assert not a[1][torch.tensor([not x for x in inside], device='cuda')].any()
        if kept:
            assert a[1, :kept].any()
    quant_cache.quantize_rows(k, v, pages, table, starts=ints([0, 25, 4]), counts=ints([n, 7, n]))     # the last row fits
    a, _ = quant_cache.dequantize_rows(pages, 40, D, table, counts=ints([32, 0, 32]))                   # no row past the end asked for
    assert not a[:, 32:].any() and not a[1].any()


def test_bad_pages_are_reported():
    from slimkv_amd import quant_cache
    g, B, n, H, D, block = gen(44), 2, 32, 2, 128, 16
    k, v = randn(g, B, n, H, D), randn(g, B, n, H, D)
    count, table = scattered(g, B, 2)
    for bad in (count, -count - 1, 1 << 40):
        wrong = table.clone()
        wrong[1, 1] = bad
        pages = quant_cache.new_pages(count, H, block, D)
        with pytest.raises(IndexError):
            quant_cache.quantize_rows(k, v, pages, wrong)
        ref = quant_cache.new_pages(count, H, block, D)
        quant_cache.quantize_rows(k, v, ref, table, counts=ints([32, 16]))
        assert torch.equal(pages, ref)
        with pytest.raises(IndexError):
            quant_cache.dequantize_rows(pages, n, D, wrong)
        a, _ = quant_cache.dequantize_rows(pages, n, D, wrong, counts=ints([32, 16]))       # the entry is not read
        assert a[1, :16].any() and not a[1, 16:].any()
        for T in (1, 40):
            q = randn(g, B, T, 4, D)
            dk = randn(g, B, T, H, D)
            with pytest.raises(IndexError):
                quant_cache.quantized_attention(q, dk, dk, 1.0, pages, wrong)
            quant_cache.quantized_attention(q, dk, dk, 1.0, pages, wrong, lengths=ints([32, 16]))


def test_empty_calls():
    from slimkv_amd import quant_cache
    pages = quant_cache.new_pages(2, 2, 16, 64)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device='cuda')
    quant_cache.quantize_rows(z(2, 0, 2, 64), z(2, 0, 2, 64), pages)
    quant_cache.quantize_rows(z(0, 3, 2, 64), z(0, 3, 2, 64), pages)
    assert quant_cache.dequantize_rows(pages, 0, 64)[0].shape == (2, 0, 2, 64)
    assert quant_cache.dequantize_rows(pages, 3, 64, counts=ints([]))[0].shape == (0, 3, 2, 64)
    out, lse = quant_cache.quantized_attention(z(2, 0, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), 1.0, pages)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    out, _ = quant_cache.quantized_attention(z(0, 3, 4, 64), None, None, 1.0, pages)
    assert out.shape == (0, 3, 4, 64)
    cos = torch.zeros(4, 64, device='cuda')
    a, b = quant_cache.norm_rope(z(2, 0, 4, 64), z(2, 0, 2, 64), cos, cos, torch.zeros(2, 0, dtype=torch.int64, device='cuda'))
    assert a.shape == (2, 0, 4, 64) and b.shape == (2, 0, 2, 64)


ATTENTION = [
    # B, T, Hq, Hkv, D, N, lengths, block, dtype, mask ('alone': no drafted rows)
    (1, 1, 8, 2, 128, 1, None, 0, 'bf16', None),
    (1, 1, 8, 2, 128, 0, None, 0, 'bf16', None),
    (2, 1, 4, 4, 128, 65, [65, 0], 16, 'bf16', 'none'),
    (2, 1, 4, 4, 128, 65, [65, 0], 16, 'bf16', 'alone'),
    (3, 1, 32, 8, 128, 517, [517, 64, 63], 16, 'bf16', None),
    (2, 5, 14, 2, 64, 200, [200, 129], 48, 'bf16', None),
    (2, 7, 8, 8, 128, 127, [1, 127], 16, 'fp16', 'rows'),
    (1, 9, 10, 2, 128, 700, None, 0, 'fp16', 'tree'),
    (2, 13, 8, 2, 128, 321, [320, 5], 32, 'bf16', 'shared'),
    (1, 26, 16, 4, 128, 1029, None, 0, 'bf16', 'tree'),
    (2, 40, 10, 2, 64, 256, [256, 250], 32, 'fp16', 'tree'),
    (1, 63, 5, 1, 128, 130, None, 0, 'bf16', 'rows'),
    (1, 130, 6, 2, 128, 67, [66], 16, 'bf16', 'tree'),
    (1, 130, 4, 2, 64, 40, None, 0, 'fp16', None),
    (2, 70, 6, 2, 128, 300, [0, 300], 64, 'fp16', 'alone'),
    (2, 20, 6, 2, 64, 300, [299, 0], 16, 'bf16', 'alone'),
    (70, 2, 4, 2, 64, 150, [(7 * i) % 151 for i in range(70)], 16, 'bf16', None),
    (1, 2, 2, 1, 128, 5003, None, 0, 'bf16', None),
    (2, 3, 2, 1, 64, 4001, [4001, 17], 16, 'fp16', 'none'),
    (1, 5, 32, 1, 128, 300, None, 0, 'bf16', 'tree'),
    (66, 9, 8, 1, 64, 140, [(11 * i) % 141 for i in range(66)], 16, 'fp16', 'tree'),
    (3, 33, 32, 4, 128, 200, [200, 0, 131], 112, 'bf16', 'rows'),
    (1, 4, 32, 4, 128, 1000, [-5], 16, 'bf16', None),
    (1, 4, 28, 4, 128, 777, [10 ** 6], 256, 'bf16', None),
]


@pytest.mark.parametrize('case', ATTENTION, ids=[str(i) for i in range(len(ATTENTION))])
def test_quantized_attention(case):
    from slimkv_amd import quant_cache
    B, T, Hq, H, D, N, lengths, block, dtype, kind = case
    print(case, flush=True)
    dt, g = TYPES[dtype], gen(45)
    pages, table, k, v = filled_pool(g, B, N, H, D, block, dtype)
    q = randn(g, B, T, Hq, D, dtype=dt, gain=2.0)
    dk, dv = randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    mask = None if kind == 'alone' else tree_mask(g, B, T, kind)
    scale = D ** -0.5
    draft = (None, None) if kind == 'alone' else (dk, dv)
    call = lambda: quant_cache.quantized_attention(q, *draft, scale, pages, table, lengths=lengths_of(lengths), keys=N, mask=mask)
    out, lse = call()
    blind = torch.zeros(B, T, T, dtype=torch.bool, device='cuda')
    check_tree(out, lse, q, k, v, lengths, dk, dv, blind if kind == 'alone' else mask, scale, str(case))
    again, lse2 = call()
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize('T', [1, 12, 40])
def test_attention_and_reading_agree(T):
    """Written by quantize_rows, read by both: the attention over the cache is the attention over dequantize_rows."""
    from slimkv_amd import cache_ops, quant_cache
    g, B, N, H, D = gen(46), 2, 600, 2, 128
    lengths = ints([600, 333])
    for dt in TYPES.values():
        count, table = scattered(g, B, 19)
        pages = quant_cache.new_pages(count, H, 32, D)
        quant_cache.quantize_rows(randn(g, B, N, H, D, dtype=dt), randn(g, B, N, H, D, dtype=dt), pages, table)
        k, v = quant_cache.dequantize_rows(pages, N, D, table, counts=lengths, dtype=dt)
        q, dk, dv = randn(g, B, T, 8, D, dtype=dt), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
        out, lse = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, table, lengths=lengths, keys=N)
        check_tree(out, lse, q, k, v, [600, 333], dk, dv, None, D ** -0.5)
        same, lse2 = cache_ops.tree_attention(q, dk, dv, D ** -0.5, k, v, lengths=lengths)
        assert (lse - lse2).abs().max() <= 2.0 ** -14


@pytest.mark.parametrize('T', [2, 30])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_blocks_that_read_as_nan_reach_what_sees_them(T, dtype):
    """A block of K that held an infinity makes its head's rows NaN, one of V its 32 columns; behind the length neither
    has an influence."""
    from slimkv_amd import quant_cache
    g, N, H, D, dt = gen(47), 200, 2, 128, TYPES[dtype]
    k, v = randn(g, 2, N, H, D, dtype=dt), randn(g, 2, N, H, D, dtype=dt)
    k[1, 77, 0, 40] = float('inf')
    v[1, 150, 1, 100] = float('nan')
    pages = quant_cache.new_pages(2, H, 208, D)
    quant_cache.quantize_rows(k, v, pages)
    q, dk, dv = randn(g, 2, T, 8, D, dtype=dt), randn(g, 2, T, H, D, dtype=dt), randn(g, 2, T, H, D, dtype=dt)
    out, lse = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, lengths=ints([N, N]))
    bad = torch.isnan(out)
    assert not bad[0].any() and bad[1, :, :4].all()
    assert bad[1, :, 4:, 96:].all() and not bad[1, :, 4:, :96].any()
    assert torch.isnan(lse[1, :4]).all() and torch.isfinite(lse[1, 4:]).all()
    out, lse = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, lengths=ints([N, 77]))
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()


def test_attention_views_and_given_outputs():
    """Heads-first q, a shared table, pages that are a part of a pool, outputs inside larger buffers, odd addresses."""
    from slimkv_amd import quant_cache
    B, T, Hq, H, D, N, g = 3, 4, 8, 2, 128, 90, gen(48)
    pages, table, k, v = filled_pool(g, 1, N, H, D, 16, 'bf16')
    big = torch.zeros(pages.shape[0], 2 * H, 2176 + 16, dtype=torch.uint8, device='cuda')
    part = big[:, H:, :2176]
    part.copy_(pages)
    q = randn(g, B, Hq, T, D).transpose(1, 2)
    draft = randn(g, B, H, T, 2 * D)
    dk, dv = draft[..., :D].transpose(1, 2), draft[..., D:].transpose(1, 2)
    mask = tree_mask(g, B, T, 'tree').transpose(1, 2)
    buf = torch.full((B, T, Hq + 1, 2 * D), 7.0, dtype=torch.bfloat16, device='cuda')
    out, lse = buf[:, :, :Hq, :D], torch.empty(B, Hq, T, device='cuda')
    a, b = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, part, table.expand(B, -1), keys=N, mask=mask, out=out, lse=lse)
    assert a is out and b is lse
    check_tree(out, lse, q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), None, dk, dv, mask, D ** -0.5)
    assert (buf[:, :, Hq] == 7).all() and (buf[..., D:] == 7).all()
    odd = torch.empty(B * T * Hq * D + 1, dtype=torch.bfloat16, device='cuda')[1:].view(B, T, Hq, D)
    odd.copy_(q)
    again, _ = quant_cache.quantized_attention(odd, dk, dv, D ** -0.5, part, table.expand(B, -1), keys=N, mask=mask)
    assert torch.equal(again, out)


@pytest.mark.parametrize('T', [1, 40])
def test_offsets_past_32_bits(T):
    """Pages 2^27 bytes apart, the last past 4 GiB from the first; and one page of a sequence that long."""
    from slimkv_amd import quant_cache
    g, N, H, D, step = gen(49), 600, 2, 128, 1 << 27
    store = torch.zeros(38 * step + 2 * 2176, dtype=torch.uint8, device='cuda')
    pages = store.as_strided((38, H, 2176), (step, 2176, 1))
    near = quant_cache.new_pages(38, H, 16, D)
    table = torch.arange(37, -1, -1, device='cuda')[None]
    k, v = randn(g, 1, N, H, D), randn(g, 1, N, H, D)
    quant_cache.quantize_rows(k, v, near, table)
    quant_cache.quantize_rows(k, v, pages, table)
    assert torch.equal(pages, near)
    for x, y in zip(quant_cache.dequantize_rows(pages, N, D, table), quant_cache.dequantize_rows(near, N, D, table)):
        assert torch.equal(x, y)
    q, dk, dv = randn(g, 1, T, 4, D), randn(g, 1, T, H, D), randn(g, 1, T, H, D)
    want = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, near, table, keys=N)
    got = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, table, keys=N)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    del store, pages
    # rows 2^25 on of one page lie past 2^31 bytes
    block = (1 << 25) + 4096
    one = torch.empty(1, 1, block * 136, dtype=torch.uint8, device='cuda')
    at = ints([block - N])
    quant_cache.quantize_rows(k[:, :, :1], v[:, :, :1], one, starts=at)
    small = quant_cache.new_pages(1, 1, 608, D)
    quant_cache.quantize_rows(k[:, :, :1], v[:, :, :1], small)
    for x, y in zip(quant_cache.dequantize_rows(one, N, D, starts=at), quant_cache.dequantize_rows(small, N, D)):
        assert torch.equal(x, y)


@pytest.mark.parametrize('T,N,dtype', [(1, 4300, 'bf16'), (20, 2200, 'fp16'), (40, 1100, 'bf16'), (70, 1200, 'fp16')])
def test_large_ragged_batches(T, N, dtype):
    """So many items and tiles that workgroups take parts of several items, one after another."""
    from slimkv_amd import quant_cache
    B, H, D, g, dt = 64, 8, 64, gen(58), TYPES[dtype]
    lengths = [N - (61 * b) % N if b % 9 else 0 for b in range(B)]
    lengths[5], lengths[6], lengths[63] = 1, N, N - 16
    k, v = randn(g, B, N, H, D, dtype=dt), randn(g, B, N, H, D, dtype=dt)
    count, table = scattered(g, B, -(-N // 32))
    pages = quant_cache.new_pages(count, H, 32, D)
    quant_cache.quantize_rows(k, v, pages, table)
    q, dk, dv = randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    kc, vc = quant_cache.dequantize_rows(pages, N, D, table, dtype=dt)
    for draft in ((dk, dv), (None, None)):
        out, lse = quant_cache.quantized_attention(q, *draft, 0.125, pages, table, lengths=ints(lengths), keys=N)
        pick = [0, 5, 6, 31, 63]
        mask = None if draft[0] is not None else torch.zeros(len(pick), T, T, dtype=torch.bool, device='cuda')
        check_tree(out[pick], lse[pick], q[pick], kc[pick], vc[pick], [lengths[b] for b in pick], dk[pick], dv[pick], mask, 0.125)
        again, lse2 = quant_cache.quantized_attention(q, *draft, 0.125, pages, table, lengths=ints(lengths), keys=N)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize('T', [1, 40])
def test_one_page_past_32_bits(T):
    """One sequence of 2^26 and more rows in one page, codes past 2^32 bytes: zero keys weigh alike, so the output is the
    sum of the values over their number; only the last rows have values."""
    from slimkv_amd import quant_cache
    D, n = 128, (1 << 26) + 4112
    pages = torch.zeros(1, 1, n * 136, dtype=torch.uint8, device='cuda')
    v = torch.full((1, 7, 1, D), 2.0 ** 60, dtype=torch.bfloat16, device='cuda')
    quant_cache.quantize_rows(torch.zeros_like(v), v, pages, starts=ints([n - 9]))
    q = randn(gen(59), 1, T, 1, D)
    out, lse = quant_cache.quantized_attention(q, None, None, 1.0, pages, lengths=ints([n - 2]))
    # the fp32 sums of at most 2^20 equal weights a lane and of 2^9 runs: 2^-24 each; the output's rounding 2^-8
    want = 7 * 2.0 ** 60 / (n - 2)
    assert ((out.double() / want - 1).abs() <= 2.0 ** -8 + 2.0 ** -12).all()
    assert (lse.double() - float(np.log(n - 2))).abs().max() <= 2.0 ** -12
    out, _ = quant_cache.quantized_attention(q, None, None, 1.0, pages, lengths=ints([n - 9]))
    assert not out.any()


@pytest.mark.parametrize('T,dtype', [(1, 'bf16'), (40, 'fp16')])
def test_long_caches_over_pages_of_any_size(T, dtype):
    """The bits of one page a sequence, whatever the pages' size."""
    from slimkv_amd import quant_cache
    B, H, D, N, g, dt = 2, 2, 64, 70001, gen(50), TYPES[dtype]
    k, v = randn(g, B, N, H, D, dtype=dt), randn(g, B, N, H, D, dtype=dt)
    q, dk, dv = randn(g, B, T, 2 * H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    lengths = ints([N, 35003])
    want = None
    for block in (70016, 16, 48, 4096):
        cols = -(-N // block)
        count, table = (B, None) if block > N else scattered(g, B, cols)
        pages = quant_cache.new_pages(count, H, block, D)
        quant_cache.quantize_rows(k, v, pages, table)
        got = quant_cache.quantized_attention(q, dk, dv, 0.125, pages, table, keys=N, lengths=lengths)
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_widest_call_and_no_wider():
    from slimkv_amd import quant_cache
    g, D, T = gen(51), 64, 1024
    pages, table, k, v = filled_pool(g, 1, 70, 1, D, 16, 'bf16')
    q, dk, dv = (randn(g, 1, T, 1, D) for _ in range(3))
    out, lse = quant_cache.quantized_attention(q, dk, dv, 0.125, pages, table, keys=70)
    keys = torch.cat([k.double(), dk.double()], 1)[0, :, 0].cpu()
    values = torch.cat([v.double(), dv.double()], 1)[0, :, 0].cpu()
    for t in (0, 1, 500, 1023):
        s = (keys[:70 + t + 1] @ q[0, t, 0].double().cpu()) * 0.125
        e = torch.softmax(s, 0) @ values[:70 + t + 1]
        assert (out[0, t, 0].double().cpu() - e).abs().max() <= 2.0 ** -7 * values.abs().max()
        assert abs(lse[0, 0, t].item() - torch.logsumexp(s, 0).item()) <= 1e-4
    wide = randn(g, 1, T + 1, 1, D)
    with pytest.raises(ValueError):
        quant_cache.quantized_attention(wide, wide, wide, 0.125, pages, table, keys=70)


def test_drafted_infinities_reach_only_the_rows_that_see_them():
    from slimkv_amd import quant_cache
    for T in (6, 24, 70):
        g, B, H, D, N = gen(52), 2, 2, 128, 100
        pages, table, k, v = filled_pool(g, B, N, H, D, 16, 'bf16')
        q, dk, dv = randn(g, B, T, 8, D), randn(g, B, T, H, D), randn(g, B, T, H, D)
        dk[0, 1], dv[0, 1] = float('nan'), float('inf')
        dv[1, T - 1, :, ::3] = float('nan')
        mask = torch.ones(B, T, T, dtype=torch.bool, device='cuda').tril()
        mask[0, :, 1], mask[1, :, T - 1] = False, False
        out, lse = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, table, keys=N, mask=mask)
        check_tree(out, lse, q, k, v, None, dk, dv, mask, D ** -0.5)
        mask[1, 0, T - 1] = True
        out, _ = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, table, keys=N, mask=mask)
        bad = torch.isnan(out)
        assert bad[1, 0, :, ::3].all() and not bad[0].any() and not bad[1, 1:].any()


NORM = [
    # B, L, Hq, Hkv, D, dtype, weights, fused
    (1, 1, 32, 8, 128, 'bf16', 'own', True),
    (2, 3, 14, 2, 64, 'fp16', 'own', True),
    (1, 5, 1, 1, 64, 'bf16', 'f32', False),
    (3, 7, 40, 8, 128, 'bf16', 'f32', True),
    (2, 2, 3, 0, 128, 'fp16', 'own', False),
    (1, 9, 5, 5, 128, 'fp16', None, False),
    (2, 100, 9, 3, 64, 'bf16', 'q only', False),
    (1, 4, 28, 4, 128, 'bf16', 'k only', True),
    (5, 1, 130, 1, 64, 'bf16', 'own', False),
]


@pytest.mark.parametrize('case', NORM, ids=[str(i) for i in range(len(NORM))])
@pytest.mark.parametrize('in_place', [False, True])
def test_norm_rope(case, in_place):
    from slimkv_amd import quant_cache
    B, L, Hq, H, D, dtype, weights, fused = case
    print(case, in_place, flush=True)
    dt, g = TYPES[dtype], gen(53)
    rows, eps = 5000, 1e-5
    angle = torch.arange(rows, dtype=torch.float64, device='cuda')[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, dtype=torch.float64, device='cuda') / D)
    cos, sin = (f(torch.cat([angle, angle * 1.01], 1)).float() for f in (torch.cos, torch.sin))     # halves that differ
    positions = torch.randint(0, rows, (B, L), generator=g, device='cuda')
    positions.view(-1)[0], positions.view(-1)[-1] = 0, rows - 1
    if fused:
        both = randn(g, B, L, Hq + 2 * H, D, dtype=dt, gain=3.0)
        q, k = both[:, :, :Hq], both[:, :, Hq:Hq + H]
    else:
        q, k = randn(g, B, L, Hq, D, dtype=dt, gain=3.0), randn(g, B, L, H, D, dtype=dt, gain=3.0)
    q[0, 0, 0] = 0.0
    wt = torch.float32 if weights == 'f32' else dt
    qw = randn(g, D, dtype=wt) if weights not in (None, 'k only') else None
    kw = randn(g, D, dtype=wt) if weights not in (None, 'q only') and H else None
    x = [(q.clone(), qw)] + ([(k.clone(), kw)] if H else [])
    after = both[:, :, Hq + H:].clone() if fused else None
    kk = k if H else None
    out = quant_cache.norm_rope(q, kk, cos, sin, positions, q_weight=qw, k_weight=kw, eps=eps,
                                **(dict(out_q=q, out_k=kk) if in_place else {}))
    assert (out[0] is q) == in_place and (H or out[1] is None)
    c, s = (to_np(t)[positions.cpu().numpy()][:, :, None] for t in (cos, sin))
    for got, (t, w) in zip(out, x):
        want, terms = oq.norm_rope(to_np(t), None if w is None else to_np(w), c, s, eps)
        tol = terms * (D / 2 + 16) * 2.0 ** -24
        tol = tol + HALF[dt] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == 'fp16' else 1e-38)
        err = np.abs(to_np(got) - want)
        print('worst over its bound', (err / tol).max(), flush=True)
        assert (err <= tol).all()
    if fused:
        assert torch.equal(both[:, :, Hq + H:], after)


@pytest.mark.parametrize('B,L,Hq,H,D,dtype', [(3, 2001, 33, 7, 64, 'bf16'), (2, 4097, 33, 7, 128, 'fp16'), (1, 5461, 17, 8, 128, 'bf16'),
                                              (5, 3001, 40, 3, 64, 'fp16')])
def test_norm_rope_of_many_tokens(B, L, Hq, H, D, dtype):
    """The bits of calls of a few tokens, where a wave takes several rounds of heads and rows go past the caches: heads
    that fill neither the last round nor the last wave."""
    from slimkv_amd import quant_cache
    g, dt = gen(59), TYPES[dtype]
    both = randn(g, B, L, Hq + 2 * H, D, dtype=dt)
    q, k, rest = both[:, :, :Hq], both[:, :, Hq:Hq + H], both[:, :, Hq + H:].clone()
    cos, sin = torch.rand(700, D, generator=g, device='cuda'), torch.rand(700, D, generator=g, device='cuda')
    positions = torch.randint(0, 700, (B, L), generator=g, device='cuda')
    weights = dict(q_weight=randn(g, D, dtype=dt), k_weight=randn(g, D, dtype=dt))
    pieces = [quant_cache.norm_rope(q[:, i:i + 127], k[:, i:i + 127], cos, sin, positions[:, i:i + 127], **weights)
              for i in range(0, L, 127)]
    want = [torch.cat(x, 1) for x in zip(*pieces)]
    got = quant_cache.norm_rope(q, k, cos, sin, positions, **weights)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    quant_cache.norm_rope(q, k, cos, sin, positions, out_q=q, out_k=k, **weights)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(both[:, :, Hq + H:], rest)


def test_norm_rope_shared_positions_views_and_bad_positions():
    from slimkv_amd import quant_cache
    g, B, L, D = gen(54), 3, 6, 128
    q, k = randn(g, B, 8, L, D).transpose(1, 2), randn(g, B, 2, L, D).transpose(1, 2)
    cos, sin = torch.rand(50, D, generator=g, device='cuda'), torch.rand(50, D, generator=g, device='cuda')
    row = torch.randint(0, 50, (1, L), generator=g, device='cuda')
    want = quant_cache.norm_rope(q.contiguous(), k.contiguous(), cos, sin, row.expand(B, L).contiguous())
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device='cuda')[1:].view(B, L, 8, D).copy_(q)
    for args in ((q, k, row), (q, k, row.expand(B, L)), (odd, k, row)):
        got = quant_cache.norm_rope(*args[:2], cos, sin, args[2])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    strided = torch.stack([row, row], 2)[..., 0]
    got = quant_cache.norm_rope(q, k, cos[:, :], sin, strided)
    assert torch.equal(got[0], want[0])
    for bad in (-1, 50, 1 << 40):
        wrong = row.expand(B, L).clone()
        wrong[1, 2] = bad
        with pytest.raises(IndexError):
            quant_cache.norm_rope(q, k, cos, sin, wrong)
        oq_, ok_ = torch.full((B, L, 8, D), 7.0, dtype=q.dtype, device='cuda'), torch.full((B, L, 2, D), 7.0, dtype=q.dtype, device='cuda')
        status = torch.zeros(1, dtype=torch.int32, device='cuda')
        quant_cache.norm_rope(q, k, cos, sin, wrong, out_q=oq_, out_k=ok_, status=status)
        assert status.item() != 0 and (oq_[1, 2] == 7).all() and (ok_[1, 2] == 7).all()
        oq_[1, 2], ok_[1, 2] = want[0][1, 2], want[1][1, 2]
        assert torch.equal(oq_, want[0]) and torch.equal(ok_, want[1])


def step_inputs(seed, dt=torch.bfloat16):
    """A decode step of three requests over a paged cache."""
    from slimkv_amd import quant_cache
    g, B, T, Hq, H, D, block = gen(seed), 3, 4, 16, 2, 128, 16
    count, table = scattered(g, B, 40)
    s = dict(pages=quant_cache.new_pages(count, H, block, D), table=table, lengths=ints([600, 17, 301]),
             rows=randn(g, B, T, Hq + 2 * H, D, dtype=dt), qw=randn(g, D, dtype=dt), kw=randn(g, D, dtype=dt),
             cos=torch.rand(700, D, generator=g, device='cuda'), sin=torch.rand(700, D, generator=g, device='cuda'),
             positions=torch.randint(0, 700, (B, T), generator=g, device='cuda'),
             status=torch.zeros(1, dtype=torch.int32, device='cuda'))
    quant_cache.quantize_rows(randn(g, B, 620, H, D, dtype=dt), randn(g, B, 620, H, D, dtype=dt), s['pages'], table)
    return s


def run_step(s):
    from slimkv_amd import quant_cache
    Hq = s['rows'].shape[2] - 4
    q, k = quant_cache.norm_rope(s['rows'][:, :, :Hq], s['rows'][:, :, Hq:Hq + 2], s['cos'], s['sin'], s['positions'],
                                 q_weight=s['qw'], k_weight=s['kw'], status=s['status'])
    v = s['rows'][:, :, Hq + 2:]
    out, lse = quant_cache.quantized_attention(q, k, v, q.shape[3] ** -0.5, s['pages'], s['table'], lengths=s['lengths'],
                                               keys=620, status=s['status'])
    quant_cache.quantize_rows(k, v, s['pages'], s['table'], starts=s['lengths'], status=s['status'])
    back = quant_cache.dequantize_rows(s['pages'], 8, q.shape[3], s['table'], starts=s['lengths'] - 4, dtype=q.dtype,
                                       status=s['status'])
    return (q, k, out, lse, *back)


def test_steps_over_a_growing_cache():
    """Prefill written, then tokens one after another and a few at a time, each step against the plain forms."""
    from slimkv_amd import quant_cache
    g, B, Hq, H, D, block = gen(55), 2, 8, 2, 64, 16
    count, table = scattered(g, B, 10)
    pages = quant_cache.new_pages(count, H, block, D)
    lengths = [37, 64]
    kc, vc = np.zeros((B, 160, H, D)), np.zeros((B, 160, H, D))

    def held(x):
        return oq.values(*oq.quantize(to_np(x), 'bf16'))

    k, v = randn(g, B, 64, H, D), randn(g, B, 64, H, D)
    quant_cache.quantize_rows(k, v, pages, table, counts=ints(lengths))
    for b in range(B):
        kc[b, :lengths[b]], vc[b, :lengths[b]] = held(k)[b, :lengths[b]], held(v)[b, :lengths[b]]
    for T in (1, 1, 5, 1, 17, 1):
        q, dk, dv = randn(g, B, T, Hq, D), randn(g, B, T, H, D), randn(g, B, T, H, D)
        out, lse = quant_cache.quantized_attention(q, dk, dv, 0.125, pages, table, lengths=ints(lengths))
        dense = [torch.from_numpy(x).float() for x in (kc, vc)]
        check_tree(out, lse, q, *dense, lengths, dk, dv, None, 0.125)
        quant_cache.quantize_rows(dk, dv, pages, table, starts=ints(lengths))
        for b in range(B):
            rows = slice(lengths[b], lengths[b] + T)
            kc[b, rows], vc[b, rows] = held(dk)[b], held(dv)[b]
            lengths[b] += T
    a, c = quant_cache.dequantize_rows(pages, 160, D, table, counts=ints(lengths))
    for b in range(B):
        assert (to_np(a)[b, :lengths[b]] == kc[b, :lengths[b]]).all() and (to_np(c)[b, :lengths[b]] == vc[b, :lengths[b]]).all()


def test_the_cache_alone_merges_with_another_branch():
    """The recent rows in full width by tree_attention, the history in 4 bits, merged by kernels.merge."""
    from slimkv_amd import cache_ops, kernels, quant_cache
    g, B, H, D, N, R = gen(56), 2, 2, 128, 300, 40
    pages, table, k, v = filled_pool(g, B, N, H, D, 16, 'bf16')
    q, rk, rv = randn(g, B, 1, 8, D), randn(g, B, R, H, D), randn(g, B, R, H, D)
    old, old_lse = quant_cache.quantized_attention(q, None, None, D ** -0.5, pages, table, keys=N)
    new, new_lse = cache_ops.tree_attention(q, rk[:, -1:], rv[:, -1:], D ** -0.5, rk[:, :-1], rv[:, :-1])
    got = kernels.merge(old.transpose(1, 2), old_lse[..., None].view(B, 8, 1), new.transpose(1, 2), new_lse.view(B, 8, 1))
    keys = torch.cat([k, rk.float()], 1)
    values = torch.cat([v, rv.float()], 1)
    want, _, terms, *_ = __import__('oracle.cache', fromlist=['x']).tree_attention(
        to_np(q), to_np(keys[:, :-1]), to_np(values[:, :-1]), [N + R - 1] * B, to_np(keys[:, -1:]), to_np(values[:, -1:]), None,
        D ** -0.5)
    err = np.abs(to_np(got.transpose(1, 2)) - want)
    assert (err <= 4 * 2.0 ** -8 * terms + 2.0 ** -8 * np.abs(want) + 1e-30).all()


def test_graph_replays_a_step():
    a = step_inputs(61)
    want = run_step(a)
    static = step_inputs(61)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run_step(static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_step(static)
    for seed in (61, 62, 63, 61):
        fresh = step_inputs(seed)
        for name in ('pages', 'table', 'lengths', 'rows', 'qw', 'kw', 'cos', 'sin', 'positions'):
            static[name].copy_(fresh[name])
        want = run_step(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(static['pages'], fresh['pages'])
        assert static['status'].item() == 0


def test_two_graphs_and_two_streams_side_by_side():
    sets = [step_inputs(71), step_inputs(72, torch.float16)]
    want = [run_step(s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, got = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(run_step(s))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(x, y))
    eager = [[], []]
    for _ in range(4):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                eager[i].append(run_step(s))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, y) for out in eager[i] for x, y in zip(out, want[i]))


def test_capture_without_a_status_word_is_refused():
    from slimkv_amd import quant_cache
    s = step_inputs(73)
    calls = [lambda: quant_cache.norm_rope(s['rows'][:, :, :16], None, s['cos'], s['sin'], s['positions']),
             lambda: quant_cache.quantize_rows(s['rows'][:, :, :2], s['rows'][:, :, 2:4], s['pages'], s['table']),
             lambda: quant_cache.dequantize_rows(s['pages'], 4, 128, s['table']),
             lambda: quant_cache.quantized_attention(s['rows'][:, :, :16], None, None, 1.0, s['pages'], s['table'])]
    for call in calls:
        call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(ValueError, match='status word'):
            with torch.cuda.graph(graph):
                torch.zeros(1, device='cuda')
                call()
        torch.cuda.synchronize()


def test_torch_operators():
    from slimkv_amd import quant_cache, torch_ops  # noqa: F401
    s = step_inputs(81)
    ops = torch.ops.slimkv
    q, k, v = s['rows'][:, :, :16].contiguous(), s['rows'][:, :, 16:18].contiguous(), s['rows'][:, :, 18:].contiguous()
    st = s['status']
    for op, args in ((ops.norm_rope, (q, k, s['cos'], s['sin'], s['positions'], s['qw'], None, 1e-6, st)),
                     (ops.quantized_attention, (q, k, v, 0.1, s['pages'], s['table'], s['lengths'], 620, None, st)),
                     (ops.dequantize_rows, (s['pages'], 9, 128, s['table'], s['lengths'], None, torch.float16, st)),
                     (ops.quantize_rows, (k, v, s['pages'], s['table'], s['lengths'], None, st))):
        torch.library.opcheck(op, args)
    want = quant_cache.quantized_attention(q, k, v, 0.1, s['pages'], s['table'], lengths=s['lengths'], keys=620)
    got = ops.quantized_attention(q, k, v, 0.1, s['pages'], s['table'], s['lengths'], 620, None, st)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_scores_of_a_thousand_million_and_more():
    """Scores past what an fp32 product holds to an integer: the largest still weighs one."""
    from slimkv_amd import quant_cache
    g, N, H, D = gen(57), 130, 1, 128
    for T in (1, 40):
        k = torch.zeros(1, N, H, D, dtype=torch.bfloat16, device='cuda')
        k[0, :, 0, 0] = 1.0
        k[0, 17, 0, 0] = 1.5
        v = randn(g, 1, N, H, D)
        pages = quant_cache.new_pages(1, H, 144, D)
        quant_cache.quantize_rows(k, v, pages)
        q = torch.zeros(1, T, 1, D, dtype=torch.bfloat16, device='cuda')
        q[..., 0] = 1.0
        _, back = quant_cache.dequantize_rows(pages, N, D)
        for scale in (1e10, 1e17):
            out, lse = quant_cache.quantized_attention(q, None, None, scale, pages, lengths=ints([N]))
            assert torch.equal(out[0, :, 0], back[0, 17, 0].expand(T, D))
            assert ((lse / (1.5 * scale) - 1).abs() <= 2.0 ** -21).all()


# query rows a KV head -> the kernel: up to 16 and 32 (few), 64 and more (many); of each, in both types and head sizes, items
# that stay whole, that are cut into splits of their own and (DEALT) that are dealt out with others
KERNELS = [
    # T, Hq, Hkv, N of a whole item, N of a split one, N of a dealt one
    (5, 6, 2, 701, 1500, 4300),
    (6, 16, 4, 399, 1029, 2200),
    (5, 14, 2, 201, 700, 1100),
    (26, 8, 2, 199, 1029, 1100),
]
EVERY = [(2, T, Hq, H, D, N, [N, part], block, dtype, mask)
         for D in (64, 128) for dtype in TYPES for T, Hq, H, whole, split, _ in KERNELS
         for N, part, block, mask in ((whole, 37, 16, None), (split, 129, 48, 'tree'), (split, split - 70, 32, 'alone'))]
# B, T, Hq, Hkv, D, N, dtype
DEALT = [(64, T, 8 * (Hq // H), 8, D, N, dtype) for D in (64, 128) for dtype in TYPES for T, Hq, H, _, _, N in KERNELS]


@pytest.mark.parametrize('case', EVERY, ids=[str(i) for i in range(len(EVERY))])
def test_every_kernel_over_whole_and_split_items(case):
    test_quantized_attention(case)


@pytest.mark.parametrize('case', DEALT, ids=[str(i) for i in range(len(DEALT))])
def test_every_kernel_over_dealt_items(case):
    from slimkv_amd import quant_cache
    B, T, Hq, H, D, N, dtype = case
    print(case, flush=True)
    g, dt = gen(62), TYPES[dtype]
    lengths = [N - (61 * b) % N if b % 9 else 0 for b in range(B)]
    lengths[5], lengths[6], lengths[63] = 1, N, N - 16
    count, table = scattered(g, B, -(-N // 32))
    pages = quant_cache.new_pages(count, H, 32, D)
    for b in range(0, B, 16):                                       # sixteen sequences' full-width rows at a time
        rows = [randn(g, 16, N, H, D, dtype=dt) for _ in range(2)]
        quant_cache.quantize_rows(*rows, pages, table[b:b + 16])
    q = randn(g, B, T, Hq, D, dtype=dt)
    dk, dv = randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    mask = tree_mask(g, B, T, 'tree')
    pick = [0, 5, 6, 63]
    kc, vc = quant_cache.dequantize_rows(pages, N, D, table[pick].contiguous(), dtype=dt)
    call = lambda: quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, table, lengths=ints(lengths), keys=N, mask=mask)
    out, lse = call()
    check_tree(out[pick], lse[pick], q[pick], kc, vc, [lengths[b] for b in pick], dk[pick], dv[pick], mask[pick], D ** -0.5, str(case))
    again, lse2 = call()
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize('T', [1, 6, 12, 40])
@pytest.mark.parametrize('D', [64, 128])
def test_attention_in_another_type_than_the_writing(T, D):
    """The cached rows enter as dequantize_rows gives them in the type of q: bf16 exact, fp16 with bf16's smallest numbers
    rounded and its largest infinite.  check_tree's bounds, for outputs below 2^-14 with half a step of fp16 there, 2^-25."""
    from oracle import cache as oc
    from slimkv_amd import quant_cache
    g, B, N, H = gen(63), 2, 300, 2
    lengths = [N, 3]
    for wrote, dt in ((torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)):
        k, v = randn(g, B, N, H, D, dtype=wrote), randn(g, B, N, H, D, dtype=wrote)
        # blocks of 2^-20 to 2^-25, some of whose numbers fp16 rounds
        v[..., 32:64] = (randn(g, B, N, H, 32).float() * 2.0 ** -(20 + torch.arange(N, device='cuda') % 6)[:, None, None]).to(wrote)
        pages = quant_cache.new_pages(B, H, 304, D)
        q, dk, dv = randn(g, B, T, 4, D, dtype=dt, gain=2.0), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
        dv[..., 32:64] = 0
        for huge in (False, True):
            if huge:
                if wrote is torch.float16:
                    continue
                v[1, 2, 1, 5], v[0, 17, 0, 31] = 3e5, -1e30
            quant_cache.quantize_rows(k, v, pages)
            rk, rv = quant_cache.dequantize_rows(pages, N, D, dtype=dt)
            exact = quant_cache.dequantize_rows(pages, N, D, dtype=torch.bfloat16)[1]
            assert torch.equal(exact.to(dt), rv) and (dt is torch.bfloat16 or not torch.equal(rv.float(), exact.float()))
            out, lse = quant_cache.quantized_attention(q, dk, dv, D ** -0.5, pages, lengths=ints(lengths))
            values = to_np(rv)
            if huge:                                                             # any weight makes an infinity of them
                assert np.isinf(values[1, 2, 1, 5]) and np.isinf(values[0, 17, 0, 31])
                got = to_np(out)
                assert (got[1, :, 2:, 5] == np.inf).all() and (got[0, :, :2, 31] == -np.inf).all()
                assert np.isfinite(np.delete(got, [5, 31], 3)).all() and np.isfinite(to_np(lse)).all()
                continue
            eo, el, terms, top, mass, total = oc.tree_attention(to_np(q), to_np(rk), values, lengths, to_np(dk), to_np(dv), None,
                                                                D ** -0.5)
            u = HALF[dt]
            d = (2.0 ** -24 * (D + 8) * mass + 2.0 ** -22 * (1 + top)).transpose(0, 2, 1)[..., None]
            tol = (2 * d + u) * terms + u * np.abs(eo) * (1 + u) + 1e-30
            if dt is torch.float16:
                tiny = 2.0 ** -25 * (N + T) / total.transpose(0, 2, 1)[..., None]
                columns = np.abs(values).max((0, 1, 2)).clip(np.abs(to_np(dv)).max((0, 1, 2)))
                tol = tol + tiny * columns + 2.0 ** -25
            worst = (np.abs(to_np(out) - eo) / tol).max()
            print(T, D, dt, 'worst output error over its bound', worst, flush=True)
            assert worst <= 1.0
            # the small columns are there, in steps of 2^-24 or finer than their sizes
            assert (np.abs(eo[..., 32:64]) > 2.0 ** -23).any() and to_np(out)[..., 32:64].any()
