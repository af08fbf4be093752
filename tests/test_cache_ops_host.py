"""The cache operators without a GPU: the C header and its ctypes mirror, refusals before anything reaches the
device, the torch operators' shapes, and the 64-bit plain forms on cases small enough to check by hand."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import cache as oc

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / 'include' / 'slimkv' / 'cache_ops.h'
BF16 = torch.bfloat16


def stripped():
    return re.sub(r'/\*.*?\*/', '', HEADER.read_text(), flags=re.S)


def structs():
    from slimkv_amd import _lib
    return (_lib.CacheRows, _lib.TreeAttentionArgs, _lib.AttentionWeightsArgs, _lib.SelectRowsArgs, _lib.CompactRowsArgs)


def test_library_exports_what_the_header_declares():
    from slimkv_amd import _lib
    names = sorted(set(re.findall(r'\b(slimkv_[a-z0-9_]+)\s*\(', stripped())))
    assert len(names) == 8
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
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "slimkv/cache_ops.h"\nint main(void){\n' +
                   '\n'.join(lines) + '\nreturn 0;}\n')
    subprocess.run(['gcc', '-I', str(ROOT / 'include'), str(src), '-o', str(tmp_path / 'layout')], check=True)
    got = subprocess.run([str(tmp_path / 'layout')], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def test_interface_number():
    from slimkv_amd import _lib
    assert _lib.lib().slimkv_cache_abi_version() == _lib.CACHE_ABI_VERSION


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def tree(**over):
    from slimkv_amd import cache_ops
    a = dict(q=z(2, 3, 8, 64), draft_k=z(2, 3, 2, 64), draft_v=z(2, 3, 2, 64), scale=1.0, k=z(2, 9, 2, 64),
             v=z(2, 9, 2, 64))
    a.update(over)
    return cache_ops.tree_attention(a.pop('q'), a.pop('draft_k'), a.pop('draft_v'), a.pop('scale'), **a)


PAGED = dict(k=None, v=None, pages=z(6, 4, 2, 2, 64), table=z(2, 3, dtype=torch.int64))
shared = z(2 * 3 * 8 * 64 + 8)
floats = z(3 * 8 * 64, dtype=torch.float32)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (PAGED, 'device tensors'),
    (dict(q=z(2, 3, 7, 64)), 'multiple of 2'),
    (dict(q=z(2, 3, 8, 128)), 'q must be'),
    (dict(q=z(2, 3, 8, 64, dtype=torch.float32)), 'bfloat16 or float16'),
    (dict(draft_k=z(2, 3, 2, 64, dtype=torch.float16)), 'bfloat16 or float16'),
    (dict(draft_k=z(2, 4, 2, 64)), 'draft_k and draft_v'),
    (dict(draft_v=z(2, 3, 1, 64)), 'draft_k and draft_v'),
    (dict(v=z(2, 8, 2, 64)), 'v must have the shape'),
    (dict(v=None), 'both k and v'),
    (dict(k=None, v=None), 'either as dense rows or as pages'),
    (dict(k=z(1, 9, 2, 64), v=z(1, 9, 2, 64)), 'cache rows must be'),
    (dict(lengths=z(2, dtype=torch.int64)), 'lengths must be int32'),
    (dict(lengths=z(3, dtype=torch.int32)), 'lengths must be int32'),
    (dict(mask=z(3, 3, dtype=torch.uint8)), 'mask must be bool'),
    (dict(mask=z(1, 3, 3, dtype=torch.bool)), 'mask must be bool'),
    (dict(mask=z(2, 3, 4, dtype=torch.bool)), 'mask must be bool'),
    (dict(out=z(2, 3, 8, 32)), 'out must have'),
    (dict(q=shared[:-8].view(2, 3, 8, 64), out=shared[8:].view(2, 3, 8, 64)), 'apart from the inputs'),
    (dict(lse=z(2, 8, 3)), 'lse must be'),
    (dict(out=z(1, 3, 8, 64).expand(2, 3, 8, 64)), 'no expanded view'),
    (dict(lse=floats[:48].view(2, 8, 3), out=floats.view(BF16).view(2, 3, 8, 64)), 'lse must be .* apart'),
    (dict(lse=floats[8:56].view(2, 8, 3), lengths=floats.view(torch.int32)[55:57]), 'lse must be .* apart'),
    (dict(keys=9), 'belong to pages'),
    (dict(PAGED, keys=13), 'keys must lie'),
    (dict(PAGED, table=z(2, 3, dtype=torch.int32)), 'int64 block table'),
    (dict(PAGED, table=z(1, 3, dtype=torch.int64)), 'int64 block table'),
    (dict(PAGED, v=z(2, 9, 2, 64)), 'pages hold both'),
    (dict(PAGED, pages=z(6, 4, 3, 2, 64)), 'pages must be'),
])
def test_tree_attention_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        tree(**over)


def weights(**over):
    from slimkv_amd import cache_ops
    a = dict(q=z(2, 3, 8, 64), lse=z(2, 8, 3, dtype=torch.float32), scale=1.0, k=z(2, 9, 2, 64))
    a.update(over)
    return cache_ops.attention_weights(a.pop('q'), a.pop('lse'), a.pop('scale'), **a)


line = z(2 * 2 * 9 + 4, dtype=torch.float32)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(lse=z(2, 3, 8, dtype=torch.float32)), 'lse must be'),
    (dict(lse=z(2, 8, 3)), 'lse must be'),
    (dict(previous=z(2, 2, 8, dtype=torch.float32)), 'previous must be'),
    (dict(out=z(2, 2, 9)), 'out must be'),
    (dict(previous=line[:36].view(2, 2, 9), out=line[4:].view(2, 2, 9)), 'previous itself'),
    (dict(k=z(2, 9, 3, 64)), 'multiple of 3'),
    (dict(lse=line[:36].view(2, 6, 3), q=z(2, 3, 6, 64), out=line[4:].view(2, 2, 9)), 'apart from lse'),
    (dict(out=z(1, 2, 9, dtype=torch.float32).expand(2, 2, 9)), 'expanded view'),
    (dict(q=floats.view(BF16).view(2, 3, 8, 64), out=floats[:36].view(2, 2, 9)), 'apart from lse and the other'),
])
def test_attention_weights_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        weights(**over)


@pytest.mark.parametrize('args,match', [
    ((z(2, 3, 9, dtype=torch.float32), 4), 'device tensors'),
    ((z(2, 3, 9), 4), 'float32'),
    ((z(2, 9, dtype=torch.float32), 4), 'float32'),
    ((z(2, 3, 9, dtype=torch.float32), 0), 'keep > 0'),
    ((z(2, 3, 9, dtype=torch.float32), 4, 3, 2), 'sink'),
    ((z(2, 3, 9, dtype=torch.float32), 4, -1, 2), 'sink'),
])
def test_select_rows_refuses(args, match):
    from slimkv_amd import cache_ops
    with pytest.raises(ValueError, match=match):
        cache_ops.select_rows(*args[:2], **dict(zip(('sink', 'recent'), args[2:])))


def compact(**over):
    from slimkv_amd import cache_ops
    a = dict(rows=z(2, 2, 4, dtype=torch.int32), counts=z(2, dtype=torch.int32), k=z(2, 9, 2, 64), v=z(2, 9, 2, 64))
    a.update(over)
    return cache_ops.compact_rows(a.pop('rows'), a.pop('counts'), **a)


cache = z(2 * 9 * 2 * 64)


@pytest.mark.parametrize('over,match', [
    (dict(), 'device tensors'),
    (dict(rows=z(2, 2, 4, dtype=torch.int64)), 'rows must be int32'),
    (dict(counts=z(3, dtype=torch.int32)), 'rows must be int32'),
    (dict(rows=z(2, 3, 4, dtype=torch.int32)), '1 or 2 heads'),
    (dict(weights=z(2, 1, 9, dtype=torch.float32)), 'weights must be'),
    (dict(in_place=True, out_k=z(2, 4, 2, 64)), 'no outputs'),
    (dict(in_place=True, k=z(1, 9, 2, 64).expand(2, 9, 2, 64)), 'expanded'),
    (dict(in_place=True, k=cache.view(2, 9, 2, 64), v=cache.view(2, 9, 2, 64)), 'two tensors'),
    (dict(out_k=z(2, 4, 2, 32)), 'outputs must be'),
    (dict(k=cache.view(2, 9, 2, 64), out_k=cache[:1024].view(2, 4, 2, 64)), 'apart from the cache'),
    (dict(out_v=z(1, 4, 2, 64).expand(2, 4, 2, 64)), 'no expanded'),
])
def test_compact_rows_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        compact(**over)


def test_the_c_entry_points_refuse_bad_sizes():
    """Calls through the C interface that end before a launch."""
    from slimkv_amd import _lib
    lib, ref = _lib.lib(), ctypes.byref
    a = _lib.TreeAttentionArgs()
    assert lib.slimkv_tree_attention(ref(a), None, 0, None) < 0
    a.q, a.draft_k, a.draft_v, a.out = 4096, 4096, 4096, 4096
    a.batch, a.drafted, a.heads, a.kv_heads, a.head_dim, a.scale = 1, 1, 8, 2, 128, 1.0
    need = lib.slimkv_tree_attention_workspace(ref(a))
    assert need > 0
    assert lib.slimkv_tree_attention(ref(a), 4096, need - 1, None) == -3
    assert lib.slimkv_tree_attention(ref(a), None, need, None) == -3
    for field, value, code in (('head_dim', 96, -2), ('dtype', 2, -2), ('drafted', 1025, -1), ('heads', 9, -1),
                               ('scale', 0.0, -1), ('scale', float('inf'), -1), ('scale', 1e-60, -1), ('scale', float('nan'), -1),
                               ('batch', -1, -1), ('q', 4098, -1), ('draft_k', 0, -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert lib.slimkv_tree_attention(ref(a), 4096, need, None) == code, field
        setattr(a, field, old)
    a.cache.keys = 5
    assert lib.slimkv_tree_attention(ref(a), 4096, need, None) == -1          # null cache
    a.cache.k, a.cache.v, a.cache.table = 4096, 4096, 4096
    a.cache.block_size, a.cache.num_blocks, a.cache.t_cols = 2, 4, 2
    assert lib.slimkv_tree_attention(ref(a), 4096, need, None) == -1          # rows past the table
    assert b'block table' in lib.slimkv_last_error()
    a.cache.table, a.cache.k_sn = None, 100
    assert lib.slimkv_tree_attention(ref(a), 4096, need, None) == -1
    assert b'16-byte' in lib.slimkv_last_error()
    w = _lib.AttentionWeightsArgs()
    assert lib.slimkv_attention_weights(ref(w), None, 0, None) < 0
    w = _lib.AttentionWeightsArgs(batch=1, queries=1, heads=2, kv_heads=1, head_dim=64)
    for scale in (0.0, float('inf'), 1e-60, float('nan')):
        w.scale = scale
        assert lib.slimkv_attention_weights(ref(w), None, 0, None) == -1 and b'scale' in lib.slimkv_last_error()
    s = _lib.SelectRowsArgs()
    s.batch, s.heads, s.keys, s.keep, s.sink = 1, 1, 10, 4, 5
    assert lib.slimkv_select_rows(ref(s), None, 0, None) == -1
    c = _lib.CompactRowsArgs()
    assert lib.slimkv_compact_rows(ref(c), None) == -2


def test_torch_operators_shapes():
    import slimkv_amd.torch_ops  # noqa: F401
    with FakeTensorMode():
        q = torch.empty(2, 3, 8, 64, dtype=BF16, device='cuda')
        d = torch.empty(2, 3, 2, 64, dtype=BF16, device='cuda')
        pages, table = torch.empty(6, 4, 2, 2, 64, dtype=BF16, device='cuda'), torch.empty(2, 3, dtype=torch.int64, device='cuda')
        out, lse = torch.ops.slimkv.tree_attention(q, d, d, 1.0, None, None, pages, table, None, None, None, None)
        assert out.shape == q.shape and out.dtype == BF16 and lse.shape == (2, 8, 3) and lse.dtype == torch.float32
        w = torch.ops.slimkv.attention_weights(q, lse, 1.0, None, pages, table, None, None, True, None, None)
        assert w.shape == (2, 2, 12) and w.dtype == torch.float32
        rows, counts = torch.ops.slimkv.select_rows(w, 5, None, 1, 2)
        assert rows.shape == (2, 2, 5) and rows.dtype == torch.int32 and counts.shape == (2,)
        k, v, kept = torch.ops.slimkv.compact_rows(rows, counts, None, None, pages, table, w, None)
        assert k.shape == v.shape == (2, 5, 2, 64) and k.dtype == BF16 and kept.shape == (2, 2, 5)


def test_oracle_tree_by_hand():
    """One head of width 1: the cache's row 0 and the tokens the mask names."""
    q, one = np.ones((1, 2, 1, 1)), np.zeros((1, 1, 1, 1))
    dk, dv = np.log(np.array([2.0, 5.0])).reshape(1, 2, 1, 1), np.array([4.0, 10.0]).reshape(1, 2, 1, 1)
    mask = np.array([[False, False], [True, False]])
    out, lse, *_ = oc.tree_attention(q, one, one + 1, [1], dk, dv, mask, 1.0)
    assert np.allclose(out.ravel(), [1.0, (1 + 2 * 4) / 3]) and np.allclose(lse.ravel(), [0.0, np.log(3)])
    out, lse, *_ = oc.tree_attention(q, one, one + 1, [0], dk, dv, mask, 1.0)
    assert out[0, 0, 0, 0] == 0 and np.isneginf(lse[0, 0, 0]) and out[0, 1, 0, 0] == 4


def test_oracle_weights_and_rows_by_hand():
    q, k = np.ones((1, 2, 1, 1)), np.log(np.array([1.0, 3.0, 4.0])).reshape(1, 3, 1, 1)
    lse = np.log(np.array([4.0, 8.0])).reshape(1, 1, 2)
    w, *_ = oc.attention_weights(q, lse, k, [3], 1.0)
    assert np.allclose(w.ravel(), [1 / 4 + 1 / 8, 3 / 4 + 3 / 8, 4 / 8])
    rows, counts = oc.select_rows(np.array([[[5.0, 1, 9, 9, np.nan, 0, 2]]]), 4, [7], 1, 1)
    assert rows.tolist() == [[[0, 2, 3, 6]]] and counts.tolist() == [4]
    rows, counts = oc.select_rows(np.array([[[0.0, 1, 1, 1, 0, 0]]]), 2, [5], 0, 0)
    assert rows.tolist() == [[[1, 2]]]
    rows, counts = oc.select_rows(np.array([[[0.0, 1, 1]]]), 4, [2], 1, 1)
    assert rows.tolist() == [[[0, 1, -1, -1]]] and counts.tolist() == [2]


def operator_calls():
    """Each operator with one of its tensors replaced: (name, argument, call of the replacement)."""
    lse, line = z(2, 8, 3, dtype=torch.float32), z(2, 2, 9, dtype=torch.float32)
    rows = (z(2, 3, 8, 64), z(2, 3, 2, 64), z(2, 9, 2, 64))
    calls = [('tree', x, rows[i], lambda t, x=x: tree(**{x: t})) for x, i in
             (('q', 0), ('draft_k', 1), ('draft_v', 1), ('k', 2), ('v', 2), ('out', 0))]
    calls += [('tree', 'lse', lse, lambda t: tree(lse=t)),
              ('tree', 'pages', PAGED['pages'], lambda t: tree(**dict(PAGED, pages=t)))]
    calls += [('weights', x, t0, lambda t, x=x: weights(**{x: t})) for x, t0 in
              (('q', rows[0]), ('lse', lse), ('k', rows[2]), ('previous', line), ('out', line))]
    from slimkv_amd import cache_ops
    calls += [('select', 'weights', line, lambda t: cache_ops.select_rows(t, 4))]
    calls += [('compact', x, t0, lambda t, x=x: compact(**{x: t})) for x, t0 in
              (('k', rows[2]), ('v', rows[2]), ('weights', line), ('out_k', z(2, 4, 2, 64)), ('out_v', z(2, 4, 2, 64)))]
    return calls


@pytest.mark.parametrize('call', operator_calls(), ids=lambda c: f'{c[0]}-{c[1]}')
def test_tangents_and_negative_views_are_refused(call):
    _, _, t, run = call
    with pytest.raises(ValueError, match='negative'):
        run(torch._neg_view(t))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match='tangent'):
            run(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with torch.no_grad(), pytest.raises(ValueError, match='tangent'):
            run(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match='device tensors'):
            run(t)


def test_overlap_is_that_of_the_elements():
    """Random views of one buffer, interleaved, nested and expanded ones among them, against the bytes they name."""
    import random
    from slimkv_amd.cache_ops import _overlap
    rng, seen = random.Random(5), [0, 0]
    room = torch.zeros(128, dtype=torch.float32)
    for _ in range(4000):
        views, named = [], []
        for dtype in rng.choices((torch.float32, torch.bfloat16), k=2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
            step = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12)) for _ in shape]
            at, size = rng.randint(0, 20), dtype.itemsize
            views.append(torch.as_strided(room.view(dtype), shape, step, at))
            named.append({(at + sum(i * s for i, s in zip(index, step))) * size + byte
                          for index in np.ndindex(*shape) for byte in range(size)})
        meets = bool(named[0] & named[1])
        assert _overlap(*views) == meets, [(x.dtype, x.shape, x.stride(), x.storage_offset()) for x in views]
        seen[meets] += 1
    assert min(seen) > 500


def test_interleaved_views_are_taken():
    """K and V, or q and the output, as halves of one tensor: refused for nothing but the device."""
    both, qo = z(2, 4, 2, 2, 64), z(2, 3, 8, 2, 64)
    with pytest.raises(ValueError, match='device tensors'):
        compact(out_k=both[:, :, 0], out_v=both[:, :, 1])
    with pytest.raises(ValueError, match='device tensors'):
        tree(q=qo[:, :, :, 0], out=qo[:, :, :, 1])
    with pytest.raises(ValueError, match='apart'):
        tree(q=qo[:, :, :, 0], out=qo.view(2, 3, 8, 128)[..., 32:96])
    wide = z(2, 2, 2, 9, dtype=torch.float32)
    with pytest.raises(ValueError, match='device tensors'):
        weights(previous=wide[:, :, 0], out=wide[:, :, 1])


moved = z(4 * 2 * 4 * 2 * 64)


@pytest.mark.parametrize('out', ['out_k', 'out_v'])
@pytest.mark.parametrize('over', [
    dict(rows=moved.view(torch.int32)[:16].view(2, 2, 4)),
    dict(counts=moved.view(torch.int32)[500:502]),
    dict(weights=moved.view(torch.float32)[100:136].view(2, 2, 9)),
    dict(PAGED, table=moved.view(torch.int64)[:6].view(2, 3)),
    dict(k=moved[1000:3304].view(2, 9, 2, 64)),
], ids=['rows', 'counts', 'weights', 'table', 'k'])
def test_compact_rows_refuses_outputs_over_its_inputs(out, over):
    with pytest.raises(ValueError, match='apart from the cache and the other inputs'):
        compact(**over, **{out: moved[:1024].view(2, 4, 2, 64)})


def test_views_that_overlap_themselves():
    """Never taken for plain where two indices name one element; ordinary, permuted, sliced and empty views pass."""
    from slimkv_amd.cache_ops import _folded
    import random
    rng, room, seen = random.Random(6), torch.zeros(128), 0
    for _ in range(3000):
        shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
        step = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12)) for _ in shape]
        t = torch.as_strided(room, shape, step)
        named = [sum(i * s for i, s in zip(index, step)) for index in np.ndindex(*shape)]
        if len(set(named)) < len(named):
            assert _folded(t), (shape, step)
            seen += 1
    assert seen > 500
    for t in (z(2, 3, 4), z(2, 3, 4).transpose(0, 2), z(2, 6, 8)[:, ::2, :4], z(2, 3, 4)[:, :0], z(4, 2, 8, 64)[:, 0],
              z(1, 3, 4).as_strided((1, 3, 4), (0, 4, 1)), torch.zeros(())):
        assert not _folded(t)


windows = dict(size=(2, 4, 2, 64), stride=(512, 64, 64, 1))          # row 1 of head 0 is row 0 of head 1


@pytest.mark.parametrize('run', [
    lambda: tree(out=z(4000).as_strided((2, 3, 8, 64), (1536, 64, 64, 1))),
    lambda: weights(out=z(100, dtype=torch.float32).as_strided((2, 2, 9), (18, 8, 1))),
    lambda: compact(out_k=z(4000).as_strided(**windows)),
    lambda: compact(out_v=z(4000).as_strided(**windows)),
    lambda: compact(in_place=True, k=z(4000).as_strided((2, 9, 2, 64), (1152, 64, 64, 1))),
    lambda: compact(in_place=True, v=z(4000).as_strided((2, 9, 2, 64), (1152, 64, 64, 1))),
    lambda: compact(in_place=True, weights=z(100, dtype=torch.float32).as_strided((2, 2, 9), (18, 8, 1))),
    lambda: compact(**dict(PAGED, pages=z(9000).as_strided((6, 4, 2, 2, 64), (512, 128, 64, 64, 1))), in_place=True),
])
def test_tensors_written_that_overlap_themselves_are_refused(run):
    with pytest.raises(ValueError, match='expanded'):
        run()


def test_in_place_refuses_what_shares_memory():
    """Sequences on the same pages; K and V, weights or index tensors in each other's memory.  The halves of one tensor
    are apart."""
    room = z(6000)
    f, i = room.view(torch.float32), room.view(torch.int32)
    k = room[:2304].view(2, 9, 2, 64)
    for over, match in (
            (dict(PAGED, table=z(1, 3, dtype=torch.int64).expand(2, 3)), 'table'),
            (dict(PAGED, table=z(2, 1, dtype=torch.int64).expand(2, 3)), 'table'),
            (dict(PAGED, table=z(9, dtype=torch.int64).as_strided((2, 3), (2, 1))), 'table'),
            (dict(k=k, v=room[128:2432].view(2, 9, 2, 64)), 'two tensors'),
            (dict(k=k, weights=f[1000:1036].view(2, 2, 9)), 'share no memory'),
            (dict(k=k, rows=i[1000:1016].view(2, 2, 4)), 'share no memory'),
            (dict(v=k, counts=i[1151:1153]), 'share no memory'),
            (dict(PAGED, pages=room[:2048].view(2, 4, 2, 2, 64), table=room.view(torch.int64)[500:506].view(2, 3)),
             'share no memory'),
            (dict(rows=i[:16].view(2, 2, 4), weights=f[8:44].view(2, 2, 9)), 'share no memory')):
        with pytest.raises(ValueError, match=match):
            compact(in_place=True, **over)
    both = z(2, 9, 2, 2, 64)
    for over in (dict(k=both[:, :, 0], v=both[:, :, 1]), dict(k=both[..., 0, :], v=both[..., 1, :]), PAGED,
                 dict(k=k, v=room[2304:4608].view(2, 9, 2, 64), weights=f[2304:2340].view(2, 2, 9))):
        with pytest.raises(ValueError, match='device tensors'):
            compact(in_place=True, **over)


def test_the_c_entry_refuses_shared_rows_in_place():
    from slimkv_amd import _lib
    sound = dict(k=4096, v=8192, k_sb=1152, k_sn=128, k_sh=64, v_sb=1152, v_sn=128, v_sh=64, keys=9)
    paged = dict(sound, table=4096, t_sb=3, t_cols=3, num_blocks=6, block_size=3)
    for cache, over in ((dict(sound, k_sb=0), {}), (dict(sound, v_sh=0), {}), (dict(sound, v=4096), {}),
                        (dict(paged, t_sb=0), {}), (sound, dict(w_sb=0)), (sound, dict(w_sh=0))):
        a = dict(rows=4096, r_sb=8, r_sh=4, counts=4096, weights=4096, w_sb=18, w_sh=9, weight_heads=2, weight_keys=9, batch=2,
                 kv_heads=2, head_dim=64, keep=4, in_place=1)
        a.update(over)
        call = _lib.CompactRowsArgs(cache=_lib.CacheRows(**cache), **a)
        assert _lib.lib().slimkv_compact_rows(ctypes.byref(call), None) == -1, (cache, over)
        assert b'of its own' in _lib.lib().slimkv_last_error()


@pytest.mark.parametrize('over', [dict(sink=2 ** 62, recent=2 ** 62), dict(sink=2 ** 63 - 1, recent=1), dict(batch=2, heads=2 ** 63 - 1),
                                  dict(batch=2 ** 32, heads=2 ** 32)])
def test_row_selection_sizes_whose_sum_or_product_wraps(over):
    from slimkv_amd import _lib
    a = _lib.SelectRowsArgs(**{**dict(batch=1, heads=1, keys=10, keep=4), **over})
    assert _lib.lib().slimkv_select_rows_workspace(ctypes.byref(a)) == 0
    assert b'select rows' in _lib.lib().slimkv_last_error()


def test_calls_past_what_one_launch_holds_are_refused():
    """Threads of a grid dimension are counted in 32 bits: refused before anything is launched."""
    from slimkv_amd import _lib
    lib, ref = _lib.lib(), ctypes.byref
    rows = dict(k=4096, v=8192, k_sb=0, k_sn=128, k_sh=64, v_sb=0, v_sn=128, v_sh=64)
    tree = _lib.TreeAttentionArgs(cache=_lib.CacheRows(**rows, keys=9), q=4096, draft_k=4096, draft_v=4096, out=4096, batch=4096,
                                  drafted=1024, heads=64, kv_heads=8, head_dim=128, scale=1.0, dk_sn=1024, dv_sn=1024, dk_sh=128,
                                  dv_sh=128)
    for s in ('q_sb', 'q_sl', 'q_sh', 'o_sb', 'o_sl', 'o_sh', 'dk_sb', 'dv_sb'):
        setattr(tree, s, 128)
    tree.cache.k_sn = tree.cache.v_sn = 1024
    weights = _lib.AttentionWeightsArgs(cache=_lib.CacheRows(**rows, keys=33 * 128), q=4096, lse=4096, out=4096, batch=65535,
                                        queries=1, heads=8, kv_heads=8, head_dim=64, scale=1.0)
    select = _lib.SelectRowsArgs(weights=4096, rows=4096, counts=4096, batch=1 << 22, heads=1, keys=10, keep=4)
    long_select = _lib.SelectRowsArgs(weights=4096, rows=4096, counts=4096, batch=1 << 23, heads=1, keys=1 << 16, keep=4)
    compact = _lib.CompactRowsArgs(cache=_lib.CacheRows(**rows, keys=9), rows=4096, counts=4096, out_k=4096, out_v=4096, batch=1,
                                   kv_heads=16, head_dim=64, keep=1 << 25)
    for code in (lib.slimkv_tree_attention(ref(tree), 4096, 1 << 40, None),
                 lib.slimkv_attention_weights(ref(weights), None, 0, None),
                 lib.slimkv_select_rows(ref(select), None, 0, None), lib.slimkv_select_rows(ref(long_select), None, 0, None),
                 lib.slimkv_compact_rows(ref(compact), None)):
        assert code == -1, lib.slimkv_last_error()
        assert b'too many rows' in lib.slimkv_last_error()


def test_trees_of_one_run_ask_for_no_workspace():
    """Past half as many blocks of 128 query rows as two workgroups a CU (256 CUs) an item lies in one run: no partial
    results, however many blocks there are."""
    from slimkv_amd import _lib
    a = _lib.TreeAttentionArgs(q=4096, batch=1, drafted=1024, kv_heads=1, head_dim=128, scale=1.0)
    need = {}
    for a.heads in (1, 4, 16, 32, 33, 64, 128, 256):
        need[a.heads] = _lib.lib().slimkv_tree_attention_workspace(ctypes.byref(a))
    assert need[1] == need[4] == need[16] == need[32] == 512 * 2 * 128 * 130 * 4
    assert all(need[heads] == 16 for heads in (33, 64, 128, 256))


@pytest.mark.parametrize('numbers,message', [
    ((16, None), 'cache operator ABI none, expected 1'),
    ((16, 7), 'cache operator ABI 7, expected 1'),
    ((9, None), 'ABI 9, expected 16'),
    ((None, None), 'ABI none, expected 16'),
], ids=['before the cache operators', 'another number', 'older', 'another library'])
def test_an_override_library_of_another_interface_is_named(numbers, message, tmp_path, monkeypatch):
    if shutil.which('gcc') is None:
        pytest.skip('gcc not available')
    from slimkv_amd import _lib
    monkeypatch.setattr(_lib, 'ABI_VERSION', 16)
    monkeypatch.setattr(_lib, 'CACHE_ABI_VERSION', 1)
    (tmp_path / 'old.c').write_text('int unrelated;\n' + '\n'.join(
        f'int {name}(void) {{ return {n}; }}' for name, n in zip(('slimkv_abi_version', 'slimkv_cache_abi_version'), numbers)
        if n is not None))
    path = tmp_path / 'old.so'
    subprocess.run(['gcc', '-shared', '-fPIC', str(tmp_path / 'old.c'), '-o', str(path)], check=True)
    monkeypatch.setenv('SLIMKV_HIP_LIBRARY', str(path))
    with pytest.raises(ImportError, match=message):
        _lib.lib.__wrapped__()
