"""Attention over a paged key/value cache, and what fills it: measured cases.

A server that answers several requests at once keeps their keys and values in
pages of one pool: a page holds ``page`` consecutive tokens of one request, and
a table names the pages of each request in order.  Three operators work on it:

  append  the Q|K|V product's new tokens: queries and keys rotated to their
          positions, keys and values written into the pages (bf16, or e4m3
          with one scale per key/value head);
  decode  attention of one new token per request over its cached tokens;
  prompt  attention of many new tokens per request (a prompt, a chunk of one, a
          few proposed tokens) over the cached tokens before and among them:
          causal, with a prefix that everything sees, a window, scores capped
          by a tanh.

Layouts: keys [pages, kv heads, page, head dim], values transposed, [pages, kv
heads, head dim, page]; columns (2i, 2i+1) of a query or key head are a rotated
pair; the new tokens of a request are its last ones, packed row after row.
Sizes: 8 query heads on one key/value head of 256 dims over prompts of 816
tokens are this repository's; the others are generic.
"""
import math

import torch

own = False

DEV = 'cuda'
BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn
THETA = 10000.0


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _case(kind, seqs, new, ctx, heads, kv_heads, dim, page, cache, name=None,
          prefix=0, window=0, softcap=0.0):
    """new / ctx: (least, most) new tokens and tokens before them."""
    c = {'kind': kind, 'seqs': seqs, 'new_min': new[0], 'new_max': new[1],
         'ctx_min': ctx[0], 'ctx_max': ctx[1], 'heads': heads,
         'kv_heads': kv_heads, 'dim': dim, 'page': page, 'cache': cache,
         'prefix': prefix, 'window': window, 'softcap': softcap}
    return {'name': name, **c} if name else c


def listed():
    return [
        # one robot's next text token behind three images and a prompt: the
        # call's latency
        _case('append', 1, (1, 1), (816, 816), 8, 1, 256, 64, 'bf16',
              'append 1 token'),
        # the next token of 128 requests, 8-bit cache with small pages
        _case('append', 128, (1, 1), (50, 600), 16, 4, 128, 16, 'e4m3',
              'append 128 tokens e4m3'),
        # a batch of long prompts of unequal lengths
        _case('append', 16, (700, 1300), (0, 0), 32, 8, 128, 32, 'e4m3',
              'append 16 prompts e4m3'),
        # one robot's next text token
        _case('decode', 1, (1, 1), (816, 816), 8, 1, 256, 64, 'bf16',
              'decode 1 x 817'),
        # a few requests, capped scores, a window that the longer ones pass
        _case('decode', 8, (1, 1), (1000, 8000), 16, 8, 256, 16, 'bf16',
              'decode 8 window cap', window=4096, softcap=50.0),
        # a busy server: lengths from one token to thousands
        _case('decode', 64, (1, 1), (0, 8191), 32, 8, 128, 32, 'bf16',
              'decode 64 ragged'),
        # long documents in an 8-bit cache
        _case('decode', 16, (1, 1), (30000, 32767), 32, 8, 128, 64, 'e4m3',
              'decode 16 x 32k e4m3'),
        # one very long request, one key/value head: only its length to split
        _case('decode', 1, (1, 1), (131071, 131071), 8, 1, 256, 128, 'bf16',
              'decode 1 x 128k'),
        # proposed tokens of 16 requests checked in one pass
        _case('prompt', 16, (5, 5), (500, 3000), 8, 1, 256, 64, 'bf16',
              'verify 16 x 5 tokens'),
        # one robot's prompt: 768 image tokens that see each other, then text
        _case('prompt', 1, (816, 816), (0, 0), 8, 1, 256, 64, 'bf16',
              'prompt 1 x 816 prefix', prefix=768),
        # prompts of unequal lengths in one batch
        _case('prompt', 4, (900, 4000), (0, 0), 32, 8, 128, 64, 'bf16',
              'prompt 4 ragged'),
        # the next chunk of four long documents, capped scores, 8-bit cache
        _case('prompt', 4, (512, 512), (14000, 16000), 32, 8, 128, 16, 'e4m3',
              'chunk 4 x 512 on 16k e4m3', softcap=30.0),
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c['kind'], [0.0, 0.0])
        m[0], m[1] = max(m[0], w['bytes']), max(m[1], w['flops'])
    kind = rng.choice(('append', 'decode', 'decode', 'prompt', 'prompt'))
    while True:
        dim = rng.choice((64, 128, 256))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 5, 8))
        page = rng.choice((16, 32, 64, 128))
        cache = rng.choice(('bf16', 'bf16', 'e4m3'))
        seqs = _log_int(rng, 1, 128 if kind != 'prompt' else 16)
        ctx = _log_int(rng, 1, 65536 if kind == 'decode' else 16384) - 1
        low = rng.choice((ctx, ctx // 2, 0))
        n = 1 if kind == 'decode' else _log_int(rng, 2 if kind == 'prompt' else 1, 4000)
        n_low = rng.choice((n, (n + 1) // 2, 1))
        prefix = rng.choice((0, 0, (ctx + n) // 2)) if kind == 'prompt' else 0
        window = rng.choice((0, 0, _log_int(rng, 16, 8192))) if kind != 'append' else 0
        cap = rng.choice((0.0, 0.0, 30.0, 50.0)) if kind != 'append' else 0.0
        c = _case(kind, seqs, (n_low, n), (low, ctx), heads, kv, dim, page,
                  cache, None, prefix, window, cap)
        w = work(c)
        # the plain form holds a padded batch and all its scores at once
        padded = seqs * (ctx + n) * kv * dim
        scores = 0 if kind == 'append' else seqs * heads * n * (ctx + n)
        if (w['bytes'] <= most[kind][0] and w['flops'] <= most[kind][1] and
                scores <= 2.2e9 and padded <= (1e8 if kind == 'append' else 6e8)):
            return c


def _spread(n, lo, hi, turn):
    """n whole numbers over [lo, hi], the ends among them, in mixed order."""
    return [lo + int(round((hi - lo) * ((((i + turn) * 7919) % n) / max(n - 1, 1))))
            for i in range(n)]


def _lengths(case):
    """Per request: new tokens, and tokens in the cache with them."""
    n = case['seqs']
    new = _spread(n, case['new_min'], case['new_max'], 0)
    ctx = _spread(n, case['ctx_min'], case['ctx_max'], 1)
    return new, [a + b for a, b in zip(new, ctx)]


def _visible(case, length, new):
    """(pairs of new token and visible token, tokens that any of them sees)."""
    pairs, first, last = 0, length, 0
    for p in range(length - new, length):
        hi = max(p + 1, min(case['prefix'], length))
        lo = max(0, p - case['window'] + 1) if case['window'] else 0
        pairs += hi - lo
        first, last = min(first, lo), max(last, hi)
    return pairs, last - first


def work(case):
    new, total = _lengths(case)
    h, kv, d = case['heads'], case['kv_heads'], case['dim']
    size = 2 if case['cache'] == 'bf16' else 1
    rows = sum(new)
    if case['kind'] == 'append':
        # the new rows in, rotated queries and the cache's entries out, the
        # rotations of the positions; 3 operations for each rotated value
        turns = min(rows, max(total)) * d * 4
        return {'bytes': rows * (h + 2 * kv) * d * 2 + rows * h * d * 2 +
                rows * 2 * kv * d * size + turns,
                'flops': rows * (h + kv) * d * 3}
    seen = [_visible(case, t, n) for t, n in zip(total, new)]
    return {'bytes': 2 * rows * h * d * 2 + sum(s[1] for s in seen) * 2 * kv * d * size,
            'flops': 4 * h * d * sum(s[0] for s in seen)}


# ---------------------------------------------------------------------------
# What a caller has in hand
# ---------------------------------------------------------------------------
def _rope_table(n, dim):
    """fp32 [n, dim / 2, 2]: cosine and sine, angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack((a.cos(), a.sin()), -1).float().contiguous()


def _normal(shape, g):
    """Normal bf16 values, made in pieces of the first dim."""
    out = torch.empty(shape, dtype=BF16, device=DEV)
    for part in out.split(max(1, shape[0] // 8)):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    return out


def prepare(case, seed):
    new, total = _lengths(case)
    h, kv, d, page = case['heads'], case['kv_heads'], case['dim'], case['page']
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [(t + page - 1) // page for t in total]
    n_pages = sum(pages) + 1
    order = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.zeros(len(pages), max(pages), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    k = _normal((n_pages, kv, page, d), g)
    v = _normal((n_pages, kv, d, page), g)
    s = {'kind': case['kind'], 'heads': h, 'window': case['window'],
         'softcap': case['softcap'], 'max_new': max(new),
         'max_len': max(total), 'page_table': table,
         'kv_len': torch.tensor(total, dtype=torch.int32, device=DEV),
         'k_scale': None, 'v_scale': None, 'prefix_len': None, 'q_start': None}
    if case['cache'] == 'e4m3':
        # scales near the largest normal value over e4m3's largest; the cast
        # makes NaN of what is beyond, so clamp
        u = torch.rand(2, kv, generator=g, device=DEV) * 0.4 + 0.8
        s['k_scale'], s['v_scale'] = (u * (6.0 / 448.0)).unbind(0)
        k = (k / s['k_scale'].view(-1, 1, 1)).clamp_(-448, 448).to(F8).view(torch.uint8)
        v = (v / s['v_scale'].view(-1, 1, 1)).clamp_(-448, 448).to(F8).view(torch.uint8)
    s['k'], s['v'] = k, v
    if case['prefix']:
        s['prefix_len'] = torch.tensor([min(case['prefix'], t) for t in total],
                                       dtype=torch.int32, device=DEV)
    if max(new) > 1:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s['q_start'] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    rows = sum(new)
    if case['kind'] == 'append':
        s['qkv'] = _normal((rows, (h + 2 * kv) * d), g)
        s['rope'] = _rope_table(max(total), d)
        s['q_out'] = torch.empty(rows, h * d, dtype=BF16, device=DEV)
    else:
        # queries whose products with a key spread over several units
        s['q'] = _normal((rows, h, d), g) * 2
    if own:
        from fluxvla_amd import kernels as K
        s['cache'] = K.PagedKV(k, v, s['k_scale'], s['v_scale'])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    if s['kind'] == 'append':
        q = _append_own(s) if own else _append(s)
        if s['k_scale'] is not None:                   # the same bytes, by their type
            return {'q': q, 'k': s['k'].view(F8), 'v': s['v'].view(F8)}
        return {'q': q, 'k': s['k'], 'v': s['v']}
    return _attention_own(s) if own else _attention(s)


def _append_own(s):
    from fluxvla_amd import kernels as K
    return K.paged_append(s['qkv'], s['cache'], s['rope'], s['page_table'],
                          s['kv_len'], s['heads'], q_out=s['q_out'],
                          q_start=s['q_start'])


def _attention_own(s):
    from fluxvla_amd import kernels as K
    return K.paged_attention(s['q'], s['cache'], s['page_table'], s['kv_len'],
                             q_start=s['q_start'], max_q=s['max_new'],
                             prefix_len=s['prefix_len'], window=s['window'],
                             softcap=s['softcap'])


def _rows(s, n_rows):
    """Per new row: its request, its place among the request's new rows, and
    its position."""
    n = s['kv_len'].shape[0]
    row = torch.arange(n_rows, device=DEV)
    if s['q_start'] is None:
        return row, torch.zeros_like(row), s['kv_len'].long() - 1
    start = s['q_start'].long()
    b = torch.searchsorted(start[1:].contiguous(), row, right=True).clamp_max(n - 1)
    i = row - start[b]
    return b, i, s['kv_len'].long()[b] - (start[b + 1] - start[b]) + i


def _rotate(x, rope):
    """x [rows, heads, dim] fp32, rope [rows, dim / 2, 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, n = rope[:, None, :, 0], rope[:, None, :, 1]
    return torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)


def _store(x, scale):
    """What the cache holds of x [rows, kv heads, dim] fp32."""
    if scale is None:
        return x.to(BF16)
    return (x / scale[:, None]).clamp(-448.0, 448.0).to(F8).view(torch.uint8)


def _append(s):
    k_cache, v_cache = s['k'], s['v']
    _, kv, page, d = k_cache.shape
    h, qkv = s['heads'], s['qkv']
    b, _, pos = _rows(s, qkv.shape[0])
    x = qkv.float().view(-1, h + 2 * kv, d)
    rope = s['rope'][pos]
    where = s['page_table'].long()[b, pos // page]
    k_cache[where, :, pos % page] = _store(_rotate(x[:, h:h + kv], rope), s['k_scale'])
    v_cache[where, :, :, pos % page] = _store(x[:, h + kv:], s['v_scale'])
    s['q_out'].copy_(_rotate(x[:, :h], rope).flatten(1))
    return s['q_out']


def _gathered(x, table, scale):
    """Pages of every request, [seqs, kv heads, ...] in 32 bits."""
    x = x[table.long()]
    x = x.float() if scale is None else x.view(F8).float() * scale.view(-1, 1, 1)
    return x.transpose(1, 2)


def _attention(s):
    q, n_seqs = s['q'], s['kv_len'].shape[0]
    rows, h, d = q.shape
    kv = s['k'].shape[1]
    g, t, most = h // kv, s['max_new'], s['max_len']
    k = _gathered(s['k'], s['page_table'], s['k_scale']).flatten(2, 3)[:, :, :most]
    v = _gathered(s['v'], s['page_table'], s['v_scale']).transpose(2, 3).flatten(3)[..., :most]
    b, i, pos = _rows(s, rows)
    # queries padded to [seqs, new tokens], a key/value head's rows together
    qp = torch.zeros(n_seqs, t, kv, g, d, device=DEV)
    qp[b, i] = q.float().view(rows, kv, g, d)
    qp = qp.permute(0, 2, 3, 1, 4).reshape(n_seqs, kv, g * t, d)
    at = torch.full((n_seqs, t), -1, dtype=torch.long, device=DEV)
    at[b, i] = pos
    key = torch.arange(most, device=DEV)
    seen = key <= at[..., None]
    if s['prefix_len'] is not None:
        seen |= (key < s['prefix_len'][:, None, None]) & (at[..., None] >= 0)
    seen &= key < s['kv_len'][:, None, None]
    if s['window']:
        seen &= key > at[..., None] - s['window']
    score = torch.matmul(qp, k.transpose(2, 3)) * d ** -0.5
    if s['softcap']:
        score = torch.tanh(score / s['softcap']) * s['softcap']
    score = score.view(n_seqs, kv, g, t, most).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).view(n_seqs, kv, g * t, most)
    o = torch.matmul(p, v.transpose(2, 3)).view(n_seqs, kv, g, t, d)
    return o.permute(0, 3, 1, 2, 4)[b, i].reshape(rows, h, d).to(BF16)


# ---------------------------------------------------------------------------
# The operators' definition in 64 bits, one request after another
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    new, total = _lengths(case)
    h, kv, d, page = case['heads'], case['kv_heads'], case['dim'], case['page']
    table = s['page_table'].tolist()
    scales = [torch.ones(kv, device=DEV) if x is None else x
              for x in (s['k_scale'], s['v_scale'])]
    ks, vs = (x.double() for x in scales)
    if case['kind'] == 'append':
        if case['cache'] == 'e4m3':
            kc, vc = s['k'].view(F8).double(), s['v'].view(F8).double()
        else:
            kc, vc = s['k'].double(), s['v'].double()
        out, row = [], 0
        for b, (n, t) in enumerate(zip(new, total)):
            x = s['qkv'][row:row + n].double().view(n, h + 2 * kv, d)
            row += n
            z = torch.view_as_complex(x[:, :h + kv].reshape(n, h + kv, d // 2, 2).contiguous())
            turn = torch.view_as_complex(s['rope'][t - n:t].double())
            z = torch.view_as_real(z * turn[:, None]).reshape(n, h + kv, d)
            out.append(z[:, :h].reshape(n, h * d))
            kn, vn = z[:, h:], x[:, h + kv:]
            if case['cache'] == 'e4m3':
                kn = (kn / ks[:, None]).clamp(-448, 448)
                vn = (vn / vs[:, None]).clamp(-448, 448)
            p = t - n
            while p < t:                               # page by page
                q = min(t, (p // page + 1) * page)
                slot, pg = p % page, table[b][p // page]
                m = slice(p - (t - n), q - (t - n))
                kc[pg, :, slot:slot + q - p] = kn[m].transpose(0, 1)
                vc[pg, :, :, slot:slot + q - p] = vn[m].permute(1, 2, 0)
                p = q
        return {'q': torch.cat(out), 'k': kc, 'v': vc}
    out, row = [], 0
    for b, (n, t) in enumerate(zip(new, total)):
        use = s['page_table'][b, :(t + page - 1) // page].long()
        k, v = s['k'][use], s['v'][use]
        if case['cache'] == 'e4m3':
            k, v = k.view(F8), v.view(F8)
        k = (k.double() * ks.view(-1, 1, 1)).permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :t]
        v = (v.double() * vs.view(-1, 1, 1)).permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :t]
        q = s['q'][row:row + n].double()
        row += n
        at = torch.arange(t - n, t, device=DEV)[:, None]
        key = torch.arange(t, device=DEV)[None]
        hide = (key > at) & (key >= case['prefix'])
        if case['window']:
            hide |= at - key >= case['window']
        o = torch.empty(n, h, d, dtype=torch.float64, device=DEV)
        for j in range(h):
            c = j // (h // kv)
            a = (q[:, j] @ k[c].t()) / math.sqrt(d)
            if case['softcap']:
                a = case['softcap'] * torch.tanh(a / case['softcap'])
            a = torch.softmax(a.masked_fill(hide, -math.inf), -1)
            o[:, j] = a @ v[c]
        out.append(o)
    return torch.cat(out)
