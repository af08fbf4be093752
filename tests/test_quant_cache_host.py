"""The 4-bit cache without a GPU: the C header and its ctypes mirror, refusals before anything reaches the device, the
torch operators' shapes, and the 64-bit plain forms against numbers worked out by hand."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import quant as oq

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / 'include' / 'slimkv' / 'quant_cache.h'
BF16 = torch.bfloat16


def stripped():
    return re.sub(r'/\*.*?\*/', '', HEADER.read_text(), flags=re.S)


def structs():
    from slimkv_amd import _lib
    return (_lib.QuantPages, _lib.QuantizeRowsArgs, _lib.DequantizeRowsArgs, _lib.QuantizedAttentionArgs,
            _lib.NormRopeArgs)


def test_library_exports_what_the_header_declares():
    from slimkv_amd import _lib
    names = sorted(set(re.findall(r'\b(slimkv_[a-z0-9_]+)\s*\(', stripped())))
    assert len(names) == 6
    for name in names:
        assert hasattr(_lib.lib(), name) and name in _lib.SIGNATURES, name


def test_struct_layouts_match_the_c_compiler(tmp_path):
    if shutil.which('gcc') is None:
        pytest.skip('gcc not available')
    lines, want = [], []
    for s in structs():
        body = re.search(r'typedef struct %s \{(.*?)\}' % s.__name__, stripped(), re.S).group(1)
        assert re.findall(r'\*?\s*([a-z_][a-z0-9_]*)\s*(?=[,;])', body) == [f[0] for f in s._fields_], s.__name__
        lines.append(f'printf("%zu\\n", sizeof({s.__name__}));')
        want.append(ctypes.sizeof(s))
        for field, _ in s._fields_:
            lines.append(f'printf("%zu\\n", offsetof({s.__name__}, {field}));')
            want.append(getattr(s, field).offset)
    src = tmp_path / 'layout.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "slimkv/quant_cache.h"\nint main(void){\n' +
                   '\n'.join(lines) + '\nreturn 0;}\n')
    subprocess.run(['gcc', '-I', str(ROOT / 'include'), str(src), '-o', str(tmp_path / 'layout')], check=True)
    got = subprocess.run([str(tmp_path / 'layout')], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def test_interface_number():
    from slimkv_amd import _lib
    assert _lib.lib().slimkv_quant_abi_version() == _lib.QUANT_ABI_VERSION


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def pool(pages=6, heads=2, block=16, dim=64):
    return z(pages, heads, block * (dim + dim // 16), dtype=torch.uint8)


I32, I64, U8, F32 = torch.int32, torch.int64, torch.uint8, torch.float32
TABLE = z(2, 3, dtype=I64)
floats = z(3 * 8 * 64, dtype=F32)
shared = z(6 * 2 * 16 * 68 + 4096, dtype=U8)


def over_pool(n, dtype, *shape):
    """(pages, a tensor over their last n bytes)."""
    return shared[:6 * 2 * 16 * 68].view(6, 2, -1), shared[6 * 2 * 16 * 68 - n:][:shape_bytes(dtype, shape)].view(dtype).view(shape)


def shape_bytes(dtype, shape):
    return int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()


def quantize(**over):
    from slimkv_amd import quant_cache
    a = dict(k=z(2, 5, 2, 64), v=z(2, 5, 2, 64), pages=pool())
    a.update(over)
    return quant_cache.quantize_rows(a.pop('k'), a.pop('v'), a.pop('pages'), **a)


_pages_and_starts = over_pool(16, I32, 2)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(table=TABLE), 'device tensors'),
    (dict(v=z(2, 4, 2, 64)), 'k and v must be'),
    (dict(k=z(2, 5, 2, 64).transpose(2, 3), v=z(2, 5, 2, 64).transpose(2, 3)), 'k and v must be'),
    (dict(k=z(2, 5, 2, 64, dtype=F32), v=z(2, 5, 2, 64, dtype=F32)), 'bfloat16 or float16'),
    (dict(v=z(2, 5, 2, 64, dtype=torch.float16)), 'bfloat16 or float16'),
    (dict(k=z(2, 5, 2, 32), v=z(2, 5, 2, 32)), 'head_dim'),
    (dict(k=z(2, 5, 2, 128), v=z(2, 5, 2, 128)), 'multiple of 16 rows'),
    (dict(k=z(2, 5, 3, 64), v=z(2, 5, 3, 64)), 'KV heads'),
    (dict(pages=pool().view(torch.int8)), 'pages must be uint8'),
    (dict(pages=pool()[0]), 'pages must be uint8'),
    (dict(pages=pool(block=8)), 'multiple of 16 rows'),
    (dict(pages=z(6, 2, 0, dtype=U8)), 'multiple of 16 rows'),
    (dict(pages=pool(pages=1)), 'needs a page'),
    (dict(pages=pool(pages=1).expand(6, -1, -1)), 'expanded'),
    (dict(table=z(2, 3, dtype=I32)), 'block table'),
    (dict(table=z(1, 3, dtype=I64)), 'block table'),
    (dict(table=z(2, 0, dtype=I64)), 'block table'),
    (dict(table=z(1, 3, dtype=I64).expand(2, 3)), 'expanded'),
    (dict(starts=z(2, dtype=I64)), 'starts must be'),
    (dict(starts=z(3, dtype=I32)), 'starts must be'),
    (dict(counts=z(2, 1, dtype=I32)), 'counts must be'),
    (dict(pages=_pages_and_starts[0], starts=_pages_and_starts[1]), 'share no memory'),
    (dict(k=z(2, 5, 2, 64).requires_grad_()), 'gradient'),
])
def test_quantize_rows_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        quantize(**over)


def dequantize(**over):
    from slimkv_amd import quant_cache
    a = dict(pages=pool(), rows=5, head_dim=64)
    a.update(over)
    return quant_cache.dequantize_rows(a.pop('pages'), a.pop('rows'), a.pop('head_dim'), **a)


_pages_and_out = over_pool(16, BF16, 6, 1, 2, 64)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(table=TABLE), 'device tensors'),
    (dict(rows=-1), 'negative'),
    (dict(head_dim=32), 'head_dim'),
    (dict(head_dim=128), 'multiple of 16 rows'),
    (dict(dtype=F32), 'dtype must be'),
    (dict(table=TABLE, starts=z(3, dtype=I32)), 'starts must be'),
    (dict(starts=z(7, dtype=I32)), 'needs a page'),
    (dict(counts=z(2, dtype=I64)), 'counts must be'),
    (dict(out_k=z(6, 5, 2, 128)), 'outputs must be'),
    (dict(out_k=z(6, 5, 2, 64, dtype=torch.float16)), 'outputs must be'),
    (dict(out_v=z(1, 5, 2, 64).expand(6, 5, 2, 64)), 'outputs must be'),
    (dict(pages=_pages_and_out[0], out_k=_pages_and_out[1], rows=1), 'apart'),
    (dict(out_k=(both := z(6, 5, 2, 64)), out_v=both), 'lie apart'),
])
def test_dequantize_rows_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        dequantize(**over)


def attention(**over):
    from slimkv_amd import quant_cache
    a = dict(q=z(2, 3, 8, 64), draft_k=z(2, 3, 2, 64), draft_v=z(2, 3, 2, 64), scale=1.0, pages=pool())
    a.update(over)
    return quant_cache.quantized_attention(a.pop('q'), a.pop('draft_k'), a.pop('draft_v'), a.pop('scale'), a.pop('pages'),
                                           **a)


_pages_and_lse = over_pool(64, F32, 2, 8, 3)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(draft_k=None, draft_v=None), 'device tensors'),
    (dict(table=TABLE, keys=48), 'device tensors'),
    (dict(q=z(2, 3, 7, 64)), 'multiple of 2'),
    (dict(q=z(2, 3, 8, 128)), 'multiple of 16 rows'),
    (dict(q=z(2, 3, 8, 64, dtype=F32)), 'bfloat16 or float16'),
    (dict(q=z(3, 8, 64)), 'q must be'),
    (dict(draft_k=None), 'both draft_k and draft_v'),
    (dict(draft_k=z(2, 3, 2, 64, dtype=torch.float16)), 'bfloat16 or float16'),
    (dict(draft_v=z(2, 4, 2, 64)), 'draft_k and draft_v'),
    (dict(lengths=z(2, dtype=I64)), 'lengths must be int32'),
    (dict(keys=17), 'keys must lie'),
    (dict(keys=-1), 'keys must lie'),
    (dict(table=TABLE, keys=49), 'keys must lie'),
    (dict(mask=z(3, 3, dtype=U8)), 'mask must be bool'),
    (dict(mask=z(1, 3, 3, dtype=torch.bool)), 'mask must be bool'),
    (dict(mask=z(3, 3, dtype=torch.bool), draft_k=None, draft_v=None), 'belongs to drafted rows'),
    (dict(out=z(2, 3, 8, 32)), 'out must have'),
    (dict(out=z(1, 3, 8, 64).expand(2, 3, 8, 64)), 'no expanded view'),
    (dict(q=(same := z(2, 3, 8, 64)), out=same), 'apart from the inputs'),
    (dict(lse=z(2, 8, 3)), 'lse must be'),
    (dict(pages=_pages_and_lse[0], lse=_pages_and_lse[1]), 'lse must be .* apart'),
    (dict(lse=floats[:48].view(2, 8, 3), out=floats.view(BF16).view(2, 3, 8, 64)), 'lse must be .* apart'),
    (dict(pages=pool(pages=1)), 'needs a page'),
    (dict(table=z(2, 3, dtype=I32)), 'block table'),
    (dict(q=z(2, 3, 8, 64).requires_grad_()), 'gradient'),
])
def test_quantized_attention_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        attention(**over)


def norm(**over):
    from slimkv_amd import quant_cache
    a = dict(q=z(2, 3, 8, 64), k=z(2, 3, 2, 64), cos=z(9, 64, dtype=F32), sin=z(9, 64, dtype=F32),
             positions=z(2, 3, dtype=I64))
    a.update(over)
    return quant_cache.norm_rope(a.pop('q'), a.pop('k'), a.pop('cos'), a.pop('sin'), a.pop('positions'), **a)


fused = z(2, 3, 12, 64)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(k=None), 'device tensors'),
    (dict(q=fused[:, :, :8], k=fused[:, :, 8:10], out_q=fused[:, :, :8], out_k=fused[:, :, 8:10]), 'device tensors'),
    (dict(q=z(3, 8, 64)), 'q must be'),
    (dict(k=z(2, 4, 2, 64)), 'q must be'),
    (dict(k=z(2, 3, 2, 128)), 'q must be'),
    (dict(k=z(2, 3, 2, 64, dtype=torch.float16)), 'bfloat16 or float16'),
    (dict(cos=z(9, 32, dtype=F32)), 'cos and sin'),
    (dict(sin=z(9, 64)), 'cos and sin'),
    (dict(sin=z(8, 64, dtype=F32)), 'cos and sin'),
    (dict(positions=z(2, 3, dtype=I32)), 'positions must be'),
    (dict(positions=z(3, dtype=I64)), 'positions must be'),
    (dict(q_weight=z(32)), 'q_weight must be'),
    (dict(q_weight=z(64, dtype=torch.float16)), 'q_weight must be'),
    (dict(q_weight=z(64), k_weight=z(64, dtype=F32)), 'of one type'),
    (dict(k=None, k_weight=z(64)), 'belong to keys'),
    (dict(out_q=z(2, 3, 8, 32)), 'out_q must have'),
    (dict(out_q=z(1, 3, 8, 64).expand(2, 3, 8, 64)), 'out_q must have'),
    (dict(q=fused[:, :, :8], k=fused[:, :, 8:10], out_k=fused[:, :, 7:9]), 'out_k must be its input'),
    (dict(out_q=(mixed := z(2, 3, 10, 64))[:, :, :8], out_k=mixed[:, :, 7:9]), 'out_q and out_k'),
    (dict(q=z(2, 3, 8, 64).requires_grad_()), 'gradient'),
])
def test_norm_rope_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        norm(**over)


def test_pages_of_other_sizes_are_refused():
    from slimkv_amd import quant_cache
    assert quant_cache.page_bytes(16, 128) == 2176 and quant_cache.page_bytes(48, 64) == 3264
    assert quant_cache.new_pages(3, 2, 32, 64, 'cpu').shape == (3, 2, 2176)
    for block, dim in ((0, 128), (8, 128), (16, 96), (-16, 64)):
        with pytest.raises(ValueError):
            quant_cache.page_bytes(block, dim)


def test_the_c_entry_points_refuse_bad_sizes():
    from slimkv_amd import _lib
    lib = _lib.lib()
    refused = (-1, -2)                                             # arguments, never the launch of a kernel on made-up addresses
    cache = dict(pages=1 << 20, p_sb=2 * 1088, p_sh=1088, num_pages=4, block_size=16)
    rows = dict(k=1 << 12, k_sb=640, k_sn=128, k_sh=64, v=1 << 16, v_sb=640, v_sn=128, v_sh=64, batch=2, rows=5, kv_heads=2,
                head_dim=64)

    def rows_call(entry, mirror, cache_over={}, **over):
        return entry(ctypes.byref(mirror(cache=_lib.QuantPages(**{**cache, **cache_over}), **{**rows, **over})), None)

    bad_cache = [dict(pages=0), dict(pages=8), dict(p_sb=2 * 1088 + 8), dict(p_sh=1072), dict(p_sh=1096), dict(p_sb=-16),
                 dict(block_size=24), dict(block_size=0), dict(num_pages=1), dict(num_pages=0), dict(num_pages=1 << 31),
                 dict(block_size=(1 << 30) + 16), dict(table=64, t_cols=0), dict(table=64, t_cols=3, t_sb=2)]
    for entry, mirror in ((lib.slimkv_quantize_rows, _lib.QuantizeRowsArgs),
                          (lib.slimkv_dequantize_rows, _lib.DequantizeRowsArgs)):
        for over in bad_cache:
            assert rows_call(entry, mirror, over) in refused, over
        for over in (dict(head_dim=96), dict(dtype=2), dict(batch=-1), dict(batch=65536), dict(rows=-1), dict(kv_heads=0),
                     dict(kv_heads=4097), dict(k=0), dict(v=8), dict(k_sn=132), dict(rows=1 << 29),
                     dict(rows=(1 << 30) + 1)):
            assert rows_call(entry, mirror, **over) in refused, over
        assert rows_call(entry, mirror, batch=0) == 0 and rows_call(entry, mirror, rows=0) == 0
        assert entry(None, None) in refused

    att = dict(q=1 << 12, q_sb=1536, q_sl=512, q_sh=64, draft_k=1 << 16, dk_sb=384, dk_sn=128, dk_sh=64, draft_v=1 << 18,
               dv_sb=384, dv_sn=128, dv_sh=64, out=1 << 22, o_sb=1536, o_sl=512, o_sh=64, lse=1 << 24, batch=2, tokens=3, heads=8,
               kv_heads=2, head_dim=64, scale=1.0, keys=16)

    def att_call(cache_over={}, **over):
        a = _lib.QuantizedAttentionArgs(cache=_lib.QuantPages(**{**cache, **cache_over}), **{**att, **over})
        return lib.slimkv_quantized_attention(ctypes.byref(a), None, 0, None)

    for over in bad_cache:
        assert att_call(over) in refused, over
    for over in (dict(head_dim=32), dict(dtype=2), dict(batch=65536), dict(tokens=1025), dict(heads=7), dict(heads=4104),
                 dict(heads=1024), dict(kv_heads=0), dict(scale=0.0), dict(scale=float('nan')), dict(scale=1e19),
                 dict(q=0), dict(q=8), dict(out=0), dict(draft_v=0), dict(draft_k=0, draft_v=0, mask=64), dict(keys=17),
                 dict(keys=-1), dict(dk_sn=1 << 23), dict(dv_sn=56), dict(o_sh=68)):
        assert att_call(**over) in refused, over
    long = dict(block_size=4096, p_sb=2 * 4096 * 68, p_sh=4096 * 68)
    assert att_call(long, keys=4096) == -3                         # cut into parts that are merged: no workspace given
    assert att_call(batch=0) == 0 and att_call(tokens=0) == 0
    a = _lib.QuantizedAttentionArgs(cache=_lib.QuantPages(**cache), **{**att, 'head_dim': 32})
    assert lib.slimkv_quantized_attention_workspace(ctypes.byref(a)) == 0

    nr = dict(q=1 << 12, q_sb=1536, q_sl=512, q_sh=64, k=1 << 16, k_sb=384, k_sl=128, k_sh=64, cos=1 << 20, sin=1 << 21,
              table_rows=9, positions=1 << 22, pos_sb=3, pos_sl=1, out_q=1 << 23, oq_sb=1536, oq_sl=512, oq_sh=64,
              out_k=1 << 24, ok_sb=384, ok_sl=128, ok_sh=64, batch=2, length=3, heads=8, kv_heads=2, head_dim=64, eps=1e-6)
    for over in (dict(head_dim=256), dict(dtype=2), dict(batch=65536), dict(length=-1), dict(heads=0), dict(heads=4097),
                 dict(kv_heads=-1), dict(eps=-1.0), dict(eps=float('nan')), dict(eps=float('inf')), dict(q=0), dict(k=0),
                 dict(out_k=0), dict(cos=0), dict(cos=8), dict(table_rows=0), dict(q_sh=68), dict(q_weight=8),
                 dict(positions=0), dict(length=1 << 30)):
        assert lib.slimkv_norm_rope(ctypes.byref(_lib.NormRopeArgs(**{**nr, **over})), None) in refused, over
    assert lib.slimkv_norm_rope(ctypes.byref(_lib.NormRopeArgs(**{**nr, 'batch': 0})), None) == 0


def test_torch_operators_shapes():
    from slimkv_amd import torch_ops  # noqa: F401
    ops = torch.ops.slimkv
    with FakeTensorMode():
        e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device='cuda')
        pages, table = e(6, 2, 1088, dtype=U8), e(2, 3, dtype=I64)
        q, k = e(2, 3, 8, 64), e(2, 3, 2, 64)
        out, lse = ops.quantized_attention(q, k, k, 1.0, pages, table, None, None, None, None)
        assert out.shape == q.shape and lse.shape == (2, 8, 3) and lse.dtype is F32
        a, b = ops.norm_rope(q, k, e(9, 64, dtype=F32), e(9, 64, dtype=F32), e(2, 3, dtype=I64), None, None, 1e-6, None)
        assert a.shape == q.shape and b.shape == k.shape
        a, b = ops.dequantize_rows(pages, 7, 64, table, None, None, torch.float16, None)
        assert a.shape == b.shape == (2, 7, 2, 64) and a.dtype is torch.float16
        a, _ = ops.dequantize_rows(pages, 7, 64, None, e(4, dtype=I32), None, BF16, None)
        assert a.shape == (4, 7, 2, 64)
        assert ops.quantize_rows(k, k, pages, table, None, None, None) is None


def test_oracle_quantizes_by_hand():
    x = np.zeros((1, 64))
    x[0, :8] = [6.0, -5.0, 2.5, -0.25, 0.75, 3.5, 1.25, 0.26]       # e = 0: ties to the even code
    x[0, 32:36] = [7.0, 6.9, -3.5, 0.5]                             # 1.75 * 4: e = 1
    codes, scales = oq.quantize(x, 'bf16')
    assert scales.tolist() == [[127, 128]]
    assert codes[0, :9].tolist() == [7, 14, 4, 8, 2, 6, 2, 1, 0]
    assert codes[0, 32:37].tolist() == [6, 5, 12, 0, 0]             # 3.5 4, 3.45 3, -1.75 -2, 0.25 0
    assert oq.values(codes, scales)[0, :4].tolist() == [6.0, -4.0, 2.0, -0.0]
    assert oq.values(codes, scales)[0, 32:36].tolist() == [8.0, 6.0, -4.0, 0.0]
    top = np.zeros((4, 32))
    top[0, 0], top[1, 0], top[2, 0], top[3, 3] = 65504.0, 2.0 ** -24, np.inf, np.nan
    codes, scales = oq.quantize(top, 'fp16')
    assert scales[:, 0].tolist() == [140, 127 - 26, 255, 255]       # fp16 ends at 6 * 2^13
    assert codes[0, 0] == 7 and codes[1, 0] == 6 and not codes[2:].any()
    assert np.isnan(oq.values(codes, scales)[2:]).all()
    codes, scales = oq.quantize(np.zeros((1, 32)), 'bf16')
    assert scales[0, 0] == 0 and not codes.any()


def test_oracle_pages_by_hand():
    D, block = 64, 32
    page = np.zeros(block * 68, np.uint8)
    k = (np.zeros((1, D), np.uint8), np.full((1, 2), 5, np.uint8))
    v = (np.zeros((1, D), np.uint8), np.full((1, 2), 9, np.uint8))
    k[0][0, 33] = 7                      # element 33: high half of byte 16 of the row
    v[0][0, 50] = 3                      # 50 = 32 + 16 + 2: block 1, high, m = 2
    r = 23                               # second group of 16, g = 1, j = 3
    oq.write_page(page, [r], k, v, D)
    where = {r * 32 + 16: 0x70, 1024 + 512 + ((16 + 2) * 4 + 3) * 2 + 1: 0x30, 2048 + 2 * r: 5, 2048 + 2 * r + 1: 5,
             2112 + 2 * r: 9, 2112 + 2 * r + 1: 9}
    assert {i: int(x) for i, x in enumerate(page) if x} == where
    rk, rv = oq.read_pages(page[None, None], D)
    assert rk[0, r, 0, 33] == 6.0 * 2.0 ** (5 - 127) and rv[0, r, 0, 50] == 1.5 * 2.0 ** (9 - 127)
    assert np.count_nonzero(rk) == np.count_nonzero(rv) == 1


def test_oracle_rotates_by_hand():
    x, w = np.array([3.0, 4.0]), np.array([1.0, 2.0])
    out, terms = oq.norm_rope(x, w, np.array([0.6, 0.6]), np.array([0.8, 0.8]), 0.0)
    y = x / np.sqrt(12.5) * w
    assert np.allclose(out, [0.6 * y[0] - 0.8 * y[1], 0.6 * y[1] + 0.8 * y[0]])
    assert np.allclose(terms, [0.6 * y[0] + 0.8 * y[1], 0.6 * y[1] + 0.8 * y[0]])


@pytest.mark.parametrize('dim,heads,kv_heads', [(128, 8, 0), (128, 5, 3), (128, 12, 4), (128, 17, 0), (64, 16, 0), (64, 20, 12),
                                                (64, 33, 0), (128, 4096, 4096)])
def test_norm_rope_refuses_more_threads_than_a_launch_counts(dim, heads, kv_heads):
    """One, two, three and many rounds of heads a token: a wave takes two, and a launch counts its threads in 32 bits, 4 waves
    a workgroup of 256."""
    from slimkv_amd import _lib
    rounds = -(-(heads + kv_heads) * dim // 1024)
    chunks = -(-rounds // 2)
    most = 4 * (0xffffffff // 256) // chunks                        # tokens whose workgroups are launchable
    for tokens in (most + 1, most + 2, most + most // 3, 2 * most + 7, 4 * most):
        batch = next(b for b in range(tokens >> 30, 65536) if b and tokens % b == 0 and tokens // b <= 1 << 30)
        wide, narrow = heads * dim, max(kv_heads, 1) * dim
        a = _lib.NormRopeArgs(
            q=1 << 12, q_sb=wide, q_sl=wide, q_sh=dim, k=1 << 16, k_sb=narrow, k_sl=narrow, k_sh=dim, cos=1 << 20, sin=1 << 21,
            table_rows=9, positions=1 << 22, pos_sb=3, pos_sl=1, out_q=1 << 23, oq_sb=wide, oq_sl=wide, oq_sh=dim, out_k=1 << 24,
            ok_sb=narrow, ok_sl=narrow, ok_sh=dim, batch=batch, length=tokens // batch, heads=heads, kv_heads=kv_heads,
            head_dim=dim, eps=1e-6)
        assert _lib.lib().slimkv_norm_rope(ctypes.byref(a), None) == -1, tokens
        assert b'too many rows' in _lib.lib().slimkv_last_error(), tokens


def test_norm_rope_in_place_over_one_tensor_for_queries_and_keys():
    """Its key heads would read what its query heads wrote."""
    x = z(2, 3, 8, 64)
    for over in (dict(out_q=x), dict(out_k=x), dict(out_q=x, out_k=z(2, 3, 8, 64)), dict(out_q=z(2, 3, 8, 64), out_k=x)):
        with pytest.raises(ValueError, match='must be its input itself or lie apart'):
            norm(q=x, k=x, **over)
    with pytest.raises(ValueError, match='out_q and out_k must lie apart'):
        norm(q=x, k=x[:], out_q=(y := z(2, 3, 8, 64)), out_k=y)
    with pytest.raises(ValueError, match='device tensors'):               # read twice, written elsewhere
        norm(q=x, k=x, out_q=z(2, 3, 8, 64))
    with pytest.raises(ValueError, match='device tensors'):               # two views of one memory, each in place
        norm(q=fused[:, :, :8], k=fused[:, :, 8:10], out_q=fused[:, :, :8], out_k=fused[:, :, 8:10])
    one = z(1, 1, 1, 64)
    with pytest.raises(ValueError, match='must be its input itself or lie apart'):
        norm(q=one, k=z(1, 1, 1, 64), positions=z(1, 1, dtype=I64), q_weight=one.view(-1), out_q=one)


@pytest.mark.parametrize('table', [z(2, 1, dtype=I64).expand(2, 3), z(1, 1, dtype=I64).expand(2, 3),
                                   z(9, dtype=I64).as_strided((2, 3), (2, 2)), z(9, dtype=I64).as_strided((2, 3), (3, 0)),
                                   z(9, dtype=I64).as_strided((2, 3), (2, 1))])
def test_quantize_rows_refuses_tables_that_name_a_page_twice(table):
    """Expanded or overlapping along either dimension, before the copy that makes a table's rows contiguous."""
    with pytest.raises(ValueError, match='expanded or overlapping'):
        quantize(table=table)


def test_tables_with_steps_are_written_through():
    for table in (z(3, 2, dtype=I64).t(), z(2, 6, dtype=I64)[:, ::2], z(2, 9, dtype=I64)[:, 3:6], z(6, 2, dtype=I64)[::2].t()):
        with pytest.raises(ValueError, match='device tensors'):
            quantize(table=table)
        with pytest.raises(ValueError, match='device tensors'):
            dequantize(table=table)
    with pytest.raises(ValueError, match='device tensors'):               # reading, sequences may share pages
        dequantize(table=z(2, 1, dtype=I64).expand(2, 3))


def attention_form(B, T, Hq, H, N):
    """(kernel, how its items are cut) of a call, as the plan has it on 256 CUs."""
    rows = T * (Hq // H)
    kernel = 16 if rows <= 16 else 32 if rows <= 32 else 64 if rows <= 64 else 128
    tile = {16: 256, 32: 128}.get(kernel, 64)
    workgroups = B * H * -(-rows // kernel)
    tiles = -(-N // tile) + -(-T // 64)
    splits = 1 if tiles <= 5 else max(1, min(-(-tiles // 2), 512 // workgroups))
    return kernel, 'dealt' if -(-tiles // splits) > 16 else 'whole' if splits == 1 else 'split'


def test_every_attention_kernel_is_compared_with_the_plain_form():
    from tests import test_gpu_quant_cache as gpu
    have = {(D, dtype, *attention_form(B, T, Hq, H, N)) for B, T, Hq, H, D, N, _, _, dtype, _ in gpu.EVERY}
    have |= {(D, dtype, *attention_form(B, T, Hq, H, N)) for B, T, Hq, H, D, N, dtype in gpu.DEALT}
    assert have == {(D, dtype, kernel, cut) for D in (64, 128) for dtype in gpu.TYPES for kernel in (16, 32, 64, 128)
                    for cut in ('whole', 'split', 'dealt')}


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_the_stated_bound_of_a_written_element(dtype):
    """Every 16-bit number as its block's largest, beside random smaller ones: off by a fifth of the largest at most, by
    2^-129 where that is more, by a quarter in blocks past 15/16 of the power of two at which the type ends."""
    kind, end = (torch.bfloat16, 2.0 ** 128) if dtype == 'bf16' else (torch.float16, 2.0 ** 16)
    bits = torch.arange(1, 1 << 15, dtype=torch.int32).to(torch.int16)
    largest = bits.view(kind)
    largest = largest[torch.isfinite(largest)]
    g = torch.Generator().manual_seed(5)
    x = largest[:, None].repeat(1, 32)
    share = torch.rand(len(largest), 31, generator=g, dtype=torch.float64) * torch.randint(0, 2, (len(largest), 31), generator=g)
    x[:, 1:] = (share * largest[:, None].double()).to(kind)                          # 0 and anything up to the largest
    x = x.double().numpy()
    assert (x <= x[:, :1]).all()
    error = np.abs(oq.values(*oq.quantize(x, dtype)) - x).max(1)
    top = x[:, 0]
    last = top > 15 / 16 * end
    assert last.any() and (error[last] <= top[last] / 4).all() and (error[last] / top[last]).max() > 0.24
    usual = np.maximum(top / 5, 2.0 ** -129)
    assert (error[~last] <= usual[~last]).all() and (error / top)[~last & (top > 2.0 ** -120)].max() > 0.199
    if dtype == 'bf16':
        assert error[top < 2.0 ** -129].max() > 0.9 * 2.0 ** -129
