"""Attention over a cache for drafted tokens, and eviction from it by attention weight, as timed cases.

Three operators that a serving loop runs one after another over full-width K/V rows (dense tensors, or raw
pages [blocks, block, 2, Hkv, D] behind block tables):

* `tree`: every drafted token attends to the request's cached rows and to its ancestors among the drafted tokens;
* `weights`: the attention weight that each cached row gets from a step's or a window's queries, added to what it
  has gathered so far;
* `evict`: the rows that a smaller cache keeps by that weight (the first rows and the most recent ones always), and
  their K, V and weights moved together.

Layer shapes are this repository's (32 query / 8 KV heads and 40 / 8, head_dim 128) and a small one of 14 / 2 heads of
64.  `run` computes the operators from elementary torch operations in fp32 unless `own` is set, then with
slimkv_amd.cache_ops.
"""
import math
import random

import torch

own = False

DEV = 'cuda:0'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def listed():
    return [
        # One user's next token over a short chat, no draft: what a step costs at least.
        {'name': 'tree_one_token', 'kind': 'tree', 'batch': 1, 'draft': 1, 'heads': 32, 'kv_heads': 8, 'dim': 128,
         'keys': 517, 'ragged': False, 'block': 0, 'dtype': 'bf16', 'chain': True},
        # The single-token step of a serving batch: 16 requests of 8K to 32K tokens in pages.
        {'name': 'tree_token_b16_paged', 'kind': 'tree', 'batch': 16, 'draft': 1, 'heads': 32, 'kv_heads': 8,
         'dim': 128, 'keys': 32768, 'ragged': True, 'block': 16, 'dtype': 'bf16', 'chain': True},
        # The same batch verifying a tree of 26 drafted tokens a request.
        {'name': 'tree_26_b16_paged', 'kind': 'tree', 'batch': 16, 'draft': 26, 'heads': 32, 'kv_heads': 8,
         'dim': 128, 'keys': 32768, 'ragged': True, 'block': 16, 'dtype': 'bf16', 'chain': False},
        # One long document, a wide tree, half precision rows in one tensor.
        {'name': 'tree_63_long_fp16', 'kind': 'tree', 'batch': 1, 'draft': 63, 'heads': 40, 'kv_heads': 8,
         'dim': 128, 'keys': 131071, 'ragged': False, 'block': 0, 'dtype': 'fp16', 'chain': False},
        # A small model's chain of 5 guesses for 6 requests, pages of 48 rows.
        {'name': 'tree_chain_small_heads', 'kind': 'tree', 'batch': 6, 'draft': 5, 'heads': 14, 'kv_heads': 2,
         'dim': 64, 'keys': 4099, 'ragged': True, 'block': 48, 'dtype': 'bf16', 'chain': True},
        # After every token of a serving batch: its weights on the paged rows.
        {'name': 'weights_token_b16_paged', 'kind': 'weights', 'batch': 16, 'queries': 1, 'heads': 32, 'kv_heads': 8,
         'dim': 128, 'keys': 32768, 'ragged': True, 'block': 16, 'dtype': 'bf16'},
        # The end of a 32K-token prompt: its last 32 queries vote on all rows.
        {'name': 'weights_last32_b1', 'kind': 'weights', 'batch': 1, 'queries': 32, 'heads': 40, 'kv_heads': 8,
         'dim': 128, 'keys': 32771, 'ragged': False, 'block': 0, 'dtype': 'bf16'},
        # Whole prompt chunks of 2048 tokens, two users, the second with a shorter past.
        {'name': 'weights_chunk_b2_fp16', 'kind': 'weights', 'batch': 2, 'queries': 2048, 'heads': 32, 'kv_heads': 8,
         'dim': 128, 'keys': 10240, 'ragged': True, 'block': 0, 'dtype': 'fp16'},
        # A short chat cut back to 512 rows.
        {'name': 'evict_chat_b1', 'kind': 'evict', 'batch': 1, 'heads': 8, 'kv_heads': 8, 'dim': 128, 'keys': 1501,
         'keep': 512, 'sink': 4, 'recent': 64, 'ragged': False, 'block': 0, 'dtype': 'bf16'},
        # A paged batch of 8K to 32K tokens brought to 4096 rows a head each.
        {'name': 'evict_b16_paged', 'kind': 'evict', 'batch': 16, 'heads': 8, 'kv_heads': 8, 'dim': 128, 'keys': 32768,
         'keep': 4096, 'sink': 4, 'recent': 256, 'ragged': True, 'block': 16, 'dtype': 'bf16'},
        # A long document, one choice of rows for all heads.
        {'name': 'evict_long_shared_fp16', 'kind': 'evict', 'batch': 1, 'heads': 1, 'kv_heads': 8, 'dim': 128,
         'keys': 131072, 'keep': 16001, 'sink': 1, 'recent': 1024, 'ragged': False, 'block': 0, 'dtype': 'fp16'},
    ]


def _log(rng, lo, hi):
    hi = max(lo, hi)
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(['tree', 'tree', 'weights', 'evict'])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (40, 8, 128), (14, 2, 64)])
    batch = _log(rng, 1, 16)
    case = {'kind': kind, 'batch': batch, 'heads': heads, 'kv_heads': kv_heads, 'dim': dim,
            'ragged': rng.random() < 0.6, 'block': rng.choice([0, 0, 16, 16, 32, 48]),
            'dtype': rng.choice(['bf16', 'bf16', 'fp16'])}
    if kind == 'tree':
        keys = case['keys'] = _log(rng, 17, min(131072, 393216 // batch))
        case['draft'] = _log(rng, 1, min(64, 6000000 // (batch * keys)))
        case['chain'] = rng.random() < 0.3
    elif kind == 'weights':
        keys = case['keys'] = _log(rng, 65, min(131072, 393216 // batch))
        case['queries'] = _log(rng, 1, min(2048, keys, 20000000 // (batch * keys)))
    else:
        keys = case['keys'] = _log(rng, 300, min(131072, 393216 // batch))
        case['keep'] = _log(rng, 64, max(64, keys // 4))
        case['sink'] = rng.randint(0, 4)
        case['recent'] = rng.randint(0, case['keep'] // 2)
        case['heads'] = rng.choice([1, kv_heads, kv_heads])
    return case


def _lengths(case):
    """Rows a request has: all of them the full count, or spread from a quarter of it to all."""
    B, N = case['batch'], case['keys']
    if not case['ragged']:
        return [N] * B
    least = min(N, max(case.get('queries', 1), N // 4))
    return [N - (N - least) * b // max(B - 1, 1) for b in range(B)] if B > 1 else [(N + least + 1) // 2]


class _Draw:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.rng = random.Random(seed)

    def randn(self, *shape, dtype=torch.float32, gain=1.0):
        return (torch.randn(*shape, generator=self.gen, device=DEV) * gain).to(dtype)


def _cache(case, d):
    """The K/V rows a program holds: dense [B, N, Hkv, D] each, or pages with a table of scattered blocks.  Keys
    have channels of unequal size and a first row that every query finds, as a trained model's have."""
    B, N, H, D, dt = case['batch'], case['keys'], case['kv_heads'], case['dim'], DTYPES[case['dtype']]
    channel = torch.exp(d.randn(1, 1, H, D, gain=0.3))
    common = d.randn(1, 1, H, D)
    k = torch.empty(B, N, H, D, dtype=dt, device=DEV)
    v = torch.empty_like(k)
    for b in range(B):
        k[b:b + 1] = (d.randn(1, N, H, D) * channel).to(dt)
        v[b:b + 1] = d.randn(1, N, H, D, dtype=dt)
    k[:, :1] = (0.75 * common).to(dt)
    lengths = _lengths(case)
    d.rng.shuffle(lengths)
    s = {'lengths': torch.tensor(lengths, dtype=torch.int32, device=DEV), 'common': common}
    if not case['block']:
        s.update(k=k, v=v, ragged=case['ragged'])
        return s
    block = case['block']
    cols = (N + block - 1) // block
    order = torch.randperm(B * cols, generator=d.gen, device=DEV)
    pages = torch.zeros(B * cols, block, 2, H, D, dtype=dt, device=DEV)
    table = order.view(B, cols)
    for b in range(B):
        for kind, rows in enumerate((k, v)):
            padded = torch.zeros(cols * block, H, D, dtype=dt, device=DEV)
            padded[:N] = rows[b]
            pages[table[b], :, kind] = padded.view(cols, block, H, D)
    s.update(pages=pages, table=table.contiguous())
    return s


def _tree_mask(case, d):
    """Which drafted token sees which: itself and its ancestors; every token but the first hangs on an earlier one."""
    B, T = case['batch'], case['draft']
    if case['chain']:
        return None
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            if t:
                mask[b, t] = mask[b, max(0, t - 1 - int(d.rng.expovariate(0.25)))]
            mask[b, t, t] = True
    return mask.to(DEV)


def prepare(case, seed):
    d = _Draw(seed)
    s = {'case': case, 'scale': 1.0 / math.sqrt(case['dim']), 'status': torch.zeros(1, dtype=torch.int32, device=DEV)}
    s.update(_cache(case, d))
    B, H, D, dt = case['batch'], case['kv_heads'], case['dim'], DTYPES[case['dtype']]
    if case['kind'] == 'evict':
        N = case['keys']
        # what many steps gather: a few heavy rows, a long tail, rows never attended to
        w = torch.exp(d.randn(B, case['heads'], N, gain=2.0))
        s['weights'] = torch.where(d.randn(B, case['heads'], N) < -1.3, 0.0, w)
        return s
    G = case['heads'] // H
    L = case['draft'] if case['kind'] == 'tree' else case['queries']
    q = d.randn(B, L, H, G, D, gain=1.2) + s['common'][:, :, :, None]
    s['q'] = q.reshape(B, L, H * G, D).to(dt)
    if case['kind'] == 'tree':
        s['draft_k'] = d.randn(B, L, H, D, dtype=dt)
        s['draft_v'] = d.randn(B, L, H, D, dtype=dt)
        s['mask'] = _tree_mask(case, d)
        return s
    # the statistics that the queries' own attention left, and the weights of the steps before
    s['lse'] = torch.empty(B, H * G, L, device=DEV)
    for b in range(B):
        k, _ = _dense(s, b)
        s['lse'][b] = torch.logsumexp(_scores(s['q'][b], k, s['scale'], int(s['lengths'][b])), -1).reshape(H * G, L)
    s['previous'] = torch.exp(d.randn(B, H, case['keys'], gain=2.0))
    return s


def _dense(s, b):
    """One request's K and V rows [N, Hkv, D] in fp32."""
    if 'k' in s:
        return s['k'][b].float(), s['v'][b].float()
    rows = s['pages'][s['table'][b]].flatten(0, 1)[:s['case']['keys']].float()
    return rows[:, 0], rows[:, 1]


def _scores(q, k, scale, n):
    """Scores [Hkv, G, L, N] of one request's queries [L, Hq, D], the last one at the cache's last row."""
    L, N, H = q.shape[0], k.shape[0], k.shape[1]
    x = q.float().view(L, H, -1, q.shape[2]).permute(1, 2, 0, 3)
    sc = torch.matmul(x.reshape(H, -1, q.shape[2]), k.permute(1, 2, 0).contiguous()).view(H, -1, L, N) * scale
    seen = torch.arange(N, device=DEV) <= (n - L + torch.arange(L, device=DEV))[:, None]
    return sc.masked_fill(~seen, -math.inf)


def run(s):
    return {'tree': _run_tree, 'weights': _run_weights, 'evict': _run_evict}[s['case']['kind']](s)


def _cache_arguments(s):
    """The cache as slimkv_amd.cache_ops takes it (K alone where V is not read)."""
    if 'k' in s:
        return {'lengths': s['lengths'] if s['ragged'] else None}
    return {'pages': s['pages'], 'table': s['table'], 'lengths': s['lengths'], 'keys': s['case']['keys'],
            'status': s['status']}


def _run_tree(s):
    if own:
        from slimkv_amd import cache_ops
        return cache_ops.tree_attention(s['q'], s['draft_k'], s['draft_v'], s['scale'], s.get('k'), s.get('v'),
                                        mask=s['mask'], **_cache_arguments(s))
    case, dt = s['case'], s['q'].dtype
    B, T, H, D, N = case['batch'], case['draft'], case['kv_heads'], case['dim'], case['keys']
    mask = torch.ones(T, T, dtype=torch.bool, device=DEV).tril().expand(B, T, T) if s['mask'] is None else s['mask']
    out, lse = torch.empty_like(s['q']), torch.empty(B, case['heads'], T, device=DEV)
    for b in range(B):
        k, v = _dense(s, b)
        k, v = torch.cat([k, s['draft_k'][b].float()]), torch.cat([v, s['draft_v'][b].float()])
        x = s['q'][b].float().view(T, H, -1, D).permute(1, 2, 0, 3).reshape(H, -1, D)
        sc = torch.matmul(x, k.permute(1, 2, 0).contiguous()).view(H, -1, T, N + T) * s['scale']
        cached = (torch.arange(N, device=DEV) < s['lengths'][b]).expand(T, N)
        sc = sc.masked_fill(~torch.cat([cached, mask[b]], 1), -math.inf)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(H, -1, N + T), v.permute(1, 0, 2).contiguous()).view(H, -1, T, D) / total
        out[b] = o.permute(2, 0, 1, 3).reshape(T, -1, D).to(dt)
        lse[b] = (top + torch.log(total)).reshape(-1, T)
    return out, lse


def _run_weights(s):
    if own:
        from slimkv_amd import cache_ops
        return cache_ops.attention_weights(s['q'], s['lse'], s['scale'], s.get('k'), previous=s['previous'],
                                           **_cache_arguments(s))
    case = s['case']
    H, L = case['kv_heads'], case['queries']
    out = torch.empty_like(s['previous'])
    for b in range(case['batch']):
        k, _ = _dense(s, b)
        p = torch.exp(_scores(s['q'][b], k, s['scale'], s['lengths'][b]) - s['lse'][b].view(H, -1, L, 1))
        out[b] = s['previous'][b] + p.sum((1, 2))
    return out


def _run_evict(s):
    case = s['case']
    if own:
        from slimkv_amd import cache_ops
        rows, counts = cache_ops.select_rows(s['weights'], case['keep'], lengths=s['lengths'], sink=case['sink'],
                                             recent=case['recent'])
        place = {} if 'k' in s else {'pages': s['pages'], 'table': s['table']}
        k, v, w = cache_ops.compact_rows(rows, counts, s.get('k'), s.get('v'), weights=s['weights'], status=s['status'],
                                          **place)
        return rows, counts, k, v, w
    B, H, N, keep = case['batch'], case['heads'], case['keys'], case['keep']
    n = s['lengths'].long()[:, None]
    i = torch.arange(N, device=DEV)[None]
    held = (i < case['sink']) | (i >= n - case['recent'])
    rank = s['weights'].masked_fill(held[:, None], math.inf).masked_fill((i >= n)[:, None], -math.inf)
    rows = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    counts = n[:, 0].clamp(max=keep)
    live = (torch.arange(keep, device=DEV) < counts[:, None])[:, None]
    rows = torch.sort(rows.masked_fill(~live, N), dim=-1).values
    at = rows.clamp(max=N - 1)
    weights = torch.gather(s['weights'], 2, at).masked_fill(~live, 0.0)
    heads = torch.arange(case['kv_heads'], device=DEV)[None, None]
    at = at.expand(B, case['kv_heads'], keep).transpose(1, 2)
    request = torch.arange(B, device=DEV)[:, None, None]
    if 'k' in s:
        k, v = s['k'][request, at, heads], s['v'][request, at, heads]
    else:
        block = case['block']
        page = s['table'][request, at // block]
        k, v = (s['pages'][page, at % block, kind, heads] for kind in (0, 1))
    dead = ~live.transpose(1, 2)[..., None]
    rows = rows.masked_fill(~live, -1).to(torch.int32)
    return rows, counts.to(torch.int32), k.masked_fill(dead, 0), v.masked_fill(dead, 0), weights


def work(case):
    """Bytes that have to be read or written once and operations, for one pass."""
    e, B, H, D, N = 2, case['batch'], case['kv_heads'], case['dim'], case['keys']
    rows = sum(_lengths(case))
    table = 8 * B * -(-N // case['block']) if case['block'] else 0
    if case['kind'] == 'evict':
        kept = sum(min(n, case['keep']) for n in _lengths(case))
        choice = case['heads'] * (4 * rows + 8 * kept)
        return {'bytes': choice + 2 * 2 * e * D * H * kept + 4 * case['heads'] * kept, 'flops': case['heads'] * rows}
    Hq, L = case['heads'], case.get('draft') or case['queries']
    small = 4 * B * Hq * L + table
    if case['kind'] == 'tree':
        mask = 0 if case['chain'] else B * L * L
        return {'bytes': 2 * e * D * H * (rows + B * L) + 2 * e * B * L * Hq * D + small + mask,
                'flops': 4 * D * Hq * L * rows + 2 * D * Hq * B * L * (L + 1)}
    return {'bytes': e * D * H * rows + e * B * L * Hq * D + 8 * H * rows + small,
            'flops': 2 * D * Hq * (L * rows - B * L * (L - 1) // 2)}


def exact(case, seed):
    """`run`'s outputs from the definitions, in 64 bits, one request and KV head after another."""
    s = prepare(case, seed)
    B, H, N, kind = case['batch'], case['kv_heads'], case['keys'], case['kind']
    lengths = s['lengths'].tolist()

    def rows_of(b, h, which):
        """Rows [n, D] of one head as the cache holds them."""
        n = lengths[b]
        if 'k' in s:
            return s['v' if which else 'k'][b, :n, h]
        i = torch.arange(n, device=DEV)
        return s['pages'][s['table'][b, i // case['block']], i % case['block'], which, h]

    if kind == 'evict':
        Hs, keep = case['heads'], case['keep']
        rows = torch.full((B, Hs, keep), -1, dtype=torch.int32, device=DEV)
        k = torch.zeros(B, keep, H, case['dim'], dtype=DTYPES[case['dtype']], device=DEV)
        v, weights = torch.zeros_like(k), torch.zeros(B, Hs, keep, device=DEV)
        for b, n in enumerate(lengths):
            kept = min(n, keep)
            for h in range(Hs):
                w = s['weights'][b, h, :n].double()
                first, last = min(case['sink'], n), max(n - case['recent'], min(case['sink'], n))
                chosen = list(range(first)) + list(range(last, n))
                more = kept - len(chosen)
                if more < 0:
                    chosen, more = chosen[:kept], 0
                # the heaviest of the middle: all above the smallest kept weight, then its first equals
                middle = w[first:last]
                if more:
                    least = torch.topk(middle, more).values[-1]
                    above = torch.nonzero(middle > least)[:, 0]
                    equal = torch.nonzero(middle == least)[:, 0][:more - above.numel()]
                    chosen = torch.cat([torch.tensor(chosen, dtype=torch.long, device=DEV),
                                        above + first, equal + first])
                index = torch.as_tensor(chosen, dtype=torch.long, device=DEV).sort().values
                rows[b, h, :kept] = index.to(torch.int32)
                weights[b, h, :kept] = s['weights'][b, h, index]
                for kv in range(H) if Hs == 1 else [h]:
                    k[b, :kept, kv], v[b, :kept, kv] = rows_of(b, kv, 0)[index], rows_of(b, kv, 1)[index]
        counts = torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device=DEV)
        return rows, counts, k, v, weights
    G = case['heads'] // H
    if kind == 'weights':
        L, out = case['queries'], s['previous'].double()
        for b, n in enumerate(lengths):
            for h in range(H):
                keys = rows_of(b, h, 0).double().t().contiguous()
                for g in range(h * G, h * G + G):
                    x = torch.mm(s['q'][b, :, g].double(), keys) * s['scale']
                    p = torch.exp(x - s['lse'][b, g].double()[:, None])
                    out[b, h, :n] += torch.tril(p, n - L).sum(0)
        return out
    T = case['draft']
    out = torch.empty(B, T, case['heads'], case['dim'], dtype=torch.float64, device=DEV)
    lse = torch.empty(B, case['heads'], T, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lengths):
        sees = torch.ones(T, T, device=DEV).tril() > 0 if s['mask'] is None else s['mask'][b]
        for h in range(H):
            keys = rows_of(b, h, 0).double().t().contiguous()
            values = rows_of(b, h, 1).double()
            for g in range(h * G, h * G + G):
                x = s['q'][b, :, g].double()
                past = torch.mm(x, keys) * s['scale']
                tree = torch.mm(x, s['draft_k'][b, :, h].double().t().contiguous()) * s['scale']
                tree = torch.where(sees, tree, -math.inf)
                lse[b, g] = torch.logsumexp(torch.cat([past, tree], 1), 1)
                p_past, p_tree = torch.exp(past - lse[b, g][:, None]), torch.exp(tree - lse[b, g][:, None])
                out[b, :, g] = torch.mm(p_past, values) + torch.mm(p_tree, s['draft_v'][b, :, h].double())
    return out, lse
