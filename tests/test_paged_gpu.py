"""fvx_paged_append and fvx_paged_attention against a plain 64-bit
implementation on the host: types, head layouts, lengths from one token on,
page sizes, masks, strides, empty rows, missing pages, graphs and streams.

Tolerances.  Append: fp32 products and sum (3 roundings of 2^-24 of the
products' magnitudes), then half a step of the stored type, 2^-8 (bf16) or
2^-4 (e4m3, at least half its smallest step, 2^-10, in units of the scale).
Attention: with A = sum_j p_j |v_j|, the probabilities' rounding to bf16 moves
a sum by at most 2^-8 A, the output's by 2^-8 |o|; the scores' fp32 sums of
D <= 256 products (at most 256 * 2^-24 * sum |q k| scale < 2^-11 for the
values used here, sum |q k| scale <= 32) and the exponentials move each
probability by less than 2^-10 of itself in all: 2^-9 A with the
denominator's."""
import pytest
import torch

from fluxvla_amd import kernels as K
from tests.conftest import announce

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32)


def _pool(total, kv, d, page, e4m3, seed, spare=2, fill=None):
    """(k, v, k_scale, v_scale, page_table) on the host, pages in mixed order."""
    g = torch.Generator().manual_seed(seed)
    need = [(t + page - 1) // page for t in total]
    n = sum(need) + spare
    table = torch.full((len(total), max(need + [1]) + 1), -1, dtype=torch.int32)
    order, at = torch.randperm(n, generator=g).int(), 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    k = torch.randn(n, kv, page, d, generator=g)
    v = torch.randn(n, kv, d, page, generator=g)
    ks = vs = None
    if e4m3:
        ks = torch.rand(kv, generator=g) * 0.01 + 0.01
        vs = torch.rand(kv, generator=g) * 0.01 + 0.01
        k = (k / ks.view(-1, 1, 1)).clamp(-448, 448).to(F8).view(torch.uint8)
        v = (v / vs.view(-1, 1, 1)).clamp(-448, 448).to(F8).view(torch.uint8)
    else:
        k, v = k.bfloat16(), v.bfloat16()
    if fill is not None:                     # what no token has written yet
        kw, vw = torch.ones(n, page, dtype=torch.bool), None
        for b, t in enumerate(total):
            for p in range(t):
                kw[table[b, p // page], p % page] = False
        k.transpose(1, 2)[kw] = fill
        v.permute(0, 3, 1, 2)[kw] = fill
    return k, v, ks, vs, table


def _values(x, scale):
    if scale is None:
        return x.double()
    return x.view(F8).double() * scale.double().view(-1, 1, 1)


def _reference(q, k, v, ks, vs, table, lens, new, window=0, softcap=0.0,
               prefix=None, scale=None):
    """(o, sum_j p_j |v_j|) in 64 bits; None rows stay NaN."""
    kd, vd = _values(k, ks), _values(v, vs)
    rows, heads, d = q.shape
    n_pages, kv, page, _ = k.shape
    out = torch.zeros(rows, heads, d, dtype=torch.float64)
    mag = torch.zeros_like(out)
    row = 0
    for b, (t, n) in enumerate(zip(lens, new)):
        cap = table.shape[1] * page
        ids = table[b].tolist()
        kk, vv, ok = [], [], []
        for j in range(min(max(t, 0), cap)):
            pg = ids[j // page]
            ok.append(0 <= pg < n_pages)
            pg = pg if ok[-1] else 0
            kk.append(kd[pg, :, j % page])
            vv.append(vd[pg, :, :, j % page])
        for i in range(n):
            pos = t - n + i
            keys = [j for j in range(len(kk)) if ok[j] and pos >= 0 and
                    (j <= pos or (prefix is not None and j < prefix[b])) and
                    (not window or j > pos - window)]
            if keys:
                kt = torch.stack([kk[j] for j in keys])
                vt = torch.stack([vv[j] for j in keys])
                for h in range(heads):
                    c = h // (heads // kv)
                    s = kt[:, c] @ q[row, h].double() * (d ** -0.5 if scale is None else scale)
                    if softcap:
                        s = softcap * torch.tanh(s / softcap)
                    p = torch.softmax(s, 0)
                    out[row, h] = p @ vt[:, c]
                    mag[row, h] = p @ vt[:, c].abs()
            row += 1
    return out, mag


def _close(got, want, mag):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all())
    err = (got - want).abs()
    tol = 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -9 * mag
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())


def _attend(cuda, lens, new, heads=8, kv=1, d=128, page=16, e4m3=False, seed=1,
            fill=None, edit=None, single=None, ldq=None, max_q=None, **kw):
    """Runs one batch and checks it; returns the output."""
    k, v, ks, vs, table = _pool([max(t, 0) for t in lens], kv, d, page, e4m3, seed, fill=fill)
    if edit is not None:
        edit(table, k, v)
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(new)
    q = torch.randn(rows, heads, d, generator=g).bfloat16()
    prefix = kw.pop('prefix', None)
    want, mag = _reference(q, k, v, ks, vs, table, lens, new, prefix=prefix, **kw)
    cache = K.PagedKV(k.to(cuda), v.to(cuda), None if ks is None else ks.to(cuda),
                      None if vs is None else vs.to(cuda))
    qd = q.to(cuda)
    if ldq:
        buf = torch.zeros(rows, ldq, dtype=torch.bfloat16, device=cuda)
        buf[:, :heads * d] = qd.view(rows, -1)
        qd = buf[:, :heads * d].unflatten(1, (heads, d))
    single = all(n == 1 for n in new) if single is None else single
    out = K.paged_attention(
        qd, cache, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
        q_start=None if single else _starts(new).to(cuda),
        max_q=max(new) if max_q is None else max_q,
        prefix_len=None if prefix is None else torch.tensor(prefix, dtype=torch.int32,
                                                            device=cuda), **kw)
    torch.cuda.synchronize()
    _close(out, want, mag)
    return out


# ---------------------------------------------------------------------------
# Attention of single tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('heads,kv,page', [(8, 1, 16), (4, 4, 64), (10, 2, 32), (16, 1, 128)])
def test_single_tokens(cuda, d, e4m3, heads, kv, page):
    announce(f'paged decode d={d} e4m3={e4m3} heads={heads}/{kv} page={page}')
    _attend(cuda, [1, 700, 33, 64, 129, 2], [1] * 6, heads, kv, d, page, e4m3)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kw', [{'window': 1}, {'window': 37}, {'window': 500},
                                {'softcap': 5.0}, {'softcap': 30.0, 'window': 64},
                                {'scale': 0.3}, {'prefix': [9, 50, 400, 0]}])
def test_single_tokens_masks(cuda, e4m3, kw):
    announce(f'paged decode e4m3={e4m3} {kw}')
    _attend(cuda, [1, 31, 300, 130], [1] * 4, 8, 2, 64, 16, e4m3, **kw)


@pytest.mark.parametrize('heads', [17, 24, 40])
def test_more_than_16_heads_of_one(cuda, heads):
    announce(f'paged decode heads={heads}')
    _attend(cuda, [5, 300], [1, 1], heads, 1, 64, 16)


@pytest.mark.parametrize('page', [16, 1024])
def test_long_sequence_is_split_and_joined(cuda, page):
    announce(f'paged decode long page={page}')
    _attend(cuda, [20011, 3], [1, 1], 2, 1, 64, page)


def test_many_sequences(cuda):
    # more sequences than threads of a workgroup, none and one among them
    lens = [(i * 37) % 90 + 1 for i in range(700)]
    announce('paged decode 700 sequences')
    _attend(cuda, lens, [1] * 700, 2, 1, 64, 16)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('fill', [float('nan'), float('inf')])
def test_unwritten_slots_do_not_matter(cuda, e4m3, fill):
    announce(f'paged decode unwritten slots {fill} e4m3={e4m3}')
    bits = 0x7f if e4m3 else fill                 # e4m3's NaN
    _attend(cuda, [1, 17, 65, 200], [1] * 4, 8, 1, 128, 64, e4m3, fill=bits)


def test_rows_that_see_nothing_are_zero(cuda):
    announce('paged decode empty rows')
    out = _attend(cuda, [0, 40, -3], [1, 1, 1], 8, 1, 64, 16)
    assert (out[0] == 0).all() and (out[2] == 0).all()


def test_missing_pages_are_not_seen(cuda):
    def edit(table, k, v):
        table[0, 1], table[1, 0], table[2, :] = -1, 10 ** 6, -7
    announce('paged decode missing pages')
    out = _attend(cuda, [60, 60, 20], [1, 1, 1], 8, 1, 64, 16, edit=edit)
    assert (out[2] == 0).all()


def test_lengths_past_the_table(cuda):
    # 3 pages of 16 in the table: keys 48 and later are not there
    announce('paged decode lengths past the table')
    k, v, _, _, table = _pool([48], 1, 64, 16, False, 3)
    table = table[:, :3].contiguous()
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    for n in (49, 100, 2 ** 31 - 1):
        out = K.paged_attention(q.to(cuda), K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda),
                                torch.tensor([n], dtype=torch.int32, device=cuda))
        want, mag = _reference(q, k, v, None, None, table, [min(n, 1000)], [1])
        _close(out, want, mag)


# ---------------------------------------------------------------------------
# Attention of several tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('heads,kv,page', [(8, 1, 64), (6, 2, 16), (4, 4, 32)])
def test_several_tokens(cuda, d, e4m3, heads, kv, page):
    announce(f'paged prompt d={d} e4m3={e4m3} heads={heads}/{kv} page={page}')
    _attend(cuda, [150, 5, 64, 200], [150, 5, 1, 37], heads, kv, d, page, e4m3)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kw', [{'window': 1}, {'window': 20}, {'softcap': 5.0},
                                {'prefix': [60, 0, 200]}, {'prefix': [1000, 3, 10]},
                                {'prefix': [60, 90, 90], 'window': 50, 'softcap': 20.0}])
@pytest.mark.parametrize('d', [64, 256])
def test_several_tokens_masks(cuda, d, e4m3, kw):
    announce(f'paged prompt masks d={d} e4m3={e4m3} {kw}')
    _attend(cuda, [130, 99, 257], [130, 40, 19], 4, 2, d, 32, e4m3, **kw)


@pytest.mark.parametrize('new', [[3, 3], [1, 0], [0, 2], [2, 70]])
@pytest.mark.parametrize('max_q', [0, 1, 2, 500])
def test_max_q_is_only_a_hint(cuda, new, max_q):
    announce(f'paged prompt new={new} max_q={max_q}')
    _attend(cuda, [90, 75], new, 8, 1, 64, 16, single=False, max_q=max_q)


def test_equal_prompts_need_no_workspace(cuda):
    # more problems than CUs, none of few rows: nothing to join
    announce('paged prompt without workspace')
    _attend(cuda, [20 + i for i in range(16)], [20] * 16, 16, 16, 64, 16)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kw', [{}, {'window': 9000}, {'window': 300}])
def test_one_workgroup_walks_a_long_sequence(cuda, e4m3, kw):
    # so many sequences that keys are not split: one workgroup goes through
    # 20000 keys, page ids in runs, a page missing in the last run
    def edit(table, k, v):
        table[0, 1230] = -1
    announce(f'paged prompt long walk e4m3={e4m3} {kw}')
    lens = [20000] + [i % 7 + 1 for i in range(1, 800)]
    _attend(cuda, lens, [20] + [1] * 799, 1, 1, 64, 16, e4m3, edit=edit, single=False, **kw)


def test_workgroups_walk_more_pages_than_they_hold(cuda):
    # 64 sequences over the same 4375 pages of 16 tokens: 547 blocks of keys
    # for each workgroup of the single-token kernel
    announce('paged decode long walk over shared pages')
    n, d, seqs = 70000, 64, 64
    k, v, _, _, table = _pool([n], 1, d, 16, False, 12)
    q = torch.randn(seqs, 2, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    lens = [n - 13 * i for i in range(seqs)]
    out = K.paged_attention(q.to(cuda), K.PagedKV(k.to(cuda), v.to(cuda)),
                            table.repeat(seqs, 1).to(cuda),
                            torch.tensor(lens, dtype=torch.int32, device=cuda))
    use = table[0, :n // 16].long()
    kk = k[use, 0].double().reshape(-1, d)
    vv = v[use, 0].double().transpose(1, 2).reshape(-1, d)
    for b in (0, 31, 63):
        p = torch.softmax(q[b].double() @ kk[:lens[b]].t() * d ** -0.5, -1)
        _close(out[b], p @ vv[:lens[b]], p @ vv[:lens[b]].abs())


@pytest.mark.parametrize('new', [[1, 1], [40, 7]])
@pytest.mark.parametrize('scale', [-0.2, 0.0])
@pytest.mark.parametrize('softcap', [0.0, 10.0])
def test_negative_and_zero_scales(cuda, new, scale, softcap):
    announce(f'paged scale={scale} softcap={softcap} new={new}')
    _attend(cuda, [80, 40], new, 4, 2, 64, 16, scale=scale, softcap=softcap,
            fill=float('nan'))


@pytest.mark.parametrize('new', [[1, 1], [3, 5], [40, 7]])
@pytest.mark.parametrize('softcap', [0.01, 1024.0])
def test_extreme_caps(cuda, new, softcap):
    # scores lose 3 * 2^-24 * 1024 * log2(e) * ln(2) = 2e-4 < 2^-10 to a cap of 1024
    announce(f'paged softcap={softcap} new={new}')
    _attend(cuda, [80, 40], new, 4, 2, 64, 16, softcap=softcap)


@pytest.mark.parametrize('most', [1, 4, 60])
@pytest.mark.parametrize('kw', [{'window': 33}, {'prefix': True}, {'softcap': 20.0}])
def test_more_sequences_than_lanes(cuda, most, kw):
    announce(f'paged 70 sequences most={most} {kw}')
    new = [1] * 70 if most == 1 else [i % (most + 1) for i in range(70)]
    lens = [n + (11 * i) % 190 for i, n in enumerate(new)]
    kw = dict(kw)
    if 'prefix' in kw:
        kw['prefix'] = [7 * i % 150 for i in range(70)]
    _attend(cuda, lens, new, 4, 2, 64, 16, **kw)


def test_overlapping_starts_of_many_sequences(cuda):
    # starts that run backwards: rows of several sequences, in any of their
    # values, and nothing outside the rows
    announce('paged overlapping starts')
    cache = K.PagedKV(torch.zeros(4, 1, 16, 64, dtype=torch.bfloat16, device=cuda),
                      torch.ones(4, 1, 64, 16, dtype=torch.bfloat16, device=cuda))
    n, rows = 200, 300
    starts = torch.tensor([0, 250] * (n // 2) + [0], dtype=torch.int32, device=cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda).repeat(n, 1)
    lens = torch.full((n,), 60, dtype=torch.int32, device=cuda)
    full = torch.full((rows + 2, 2, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    q = torch.ones(rows, 2, 64, dtype=torch.bfloat16, device=cuda)
    for most in (0, 8, 250):
        K.paged_attention(q, cache, table, lens, out=full[1:-1], q_start=starts, max_q=most)
        torch.cuda.synchronize()
        out = full.float()
        assert (out[0] == 7).all() and (out[251:] == 7).all()
        # the rows before a sequence's start see nothing, the others ones
        assert (((out[1:251] - 1).abs() <= 2 ** -7) | (out[1:251] == 0) | (out[1:251] == 7)).all()


def test_two_graphs_of_different_calls(cuda):
    announce('paged two graphs')
    k, v, _, _, table = _pool([900, 700], 1, 64, 16, False, 14)
    cache, t = K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda)
    lens = torch.tensor([900, 700], dtype=torch.int32, device=cuda)
    starts = _starts([30, 2]).to(cuda)
    g = torch.Generator().manual_seed(6)
    q1 = torch.randn(2, 8, 64, generator=g).bfloat16().to(cuda)
    q2 = torch.randn(32, 8, 64, generator=g).bfloat16().to(cuda)

    def one():
        return K.paged_attention(q1, cache, t, lens)

    def many():
        return K.paged_attention(q2, cache, t, lens, q_start=starts, max_q=30)

    one(), many()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (one, many):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for n in ([900, 700], [17, 650], [1, 0], [900, 32]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for gr in (graphs[0], graphs[1], graphs[0]):
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], one()) and torch.equal(outs[1], many())


def test_empty_calls(cuda):
    announce('paged empty calls')
    cache = K.PagedKV.empty(2, 16, 1, 64, cuda)
    table = torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    out = K.paged_attention(torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=cuda), cache, table,
                            none)
    assert out.shape == (0, 4, 64)
    # rows, but no sequence: they stay
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=cuda)
    out = torch.full_like(q, 5.0)
    start = torch.zeros(1, dtype=torch.int32, device=cuda)
    K.paged_attention(q, cache, table, none, out=out, q_start=start)
    assert (out == 5.0).all()
    # a table without pages: nothing to see, nowhere to write
    table = torch.zeros(2, 0, dtype=torch.int32, device=cuda)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=cuda)
    assert (K.paged_attention(q[:2], cache, table, lens) == 0).all()
    before = cache.k.clone()
    got = K.paged_append(torch.ones(2, 6 * 64, dtype=torch.bfloat16, device=cuda), cache,
                         K.rope_table(4, 64, device=cuda), table, lens, 4)
    assert torch.isfinite(got.float()).all() and torch.equal(cache.k.view(torch.int16),
                                                             before.view(torch.int16))


def test_workspace_bytes_are_enough(cuda):
    announce('paged workspace bytes')
    for new in ([1, 1], [5, 3], [200, 1]):
        lens = [900, 300]
        k, v, _, _, table = _pool(lens, 1, 64, 16, False, 13)
        cache, t = K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda)
        q = torch.randn(sum(new), 8, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(cuda)
        ln = torch.tensor(lens, dtype=torch.int32, device=cuda)
        st = None if max(new) == 1 else _starts(new).to(cuda)
        n = K.paged_attention_workspace_bytes(q, cache, t, st, max(new))
        ws = torch.full((n + 64,), 0x55, dtype=torch.uint8, device=cuda)
        got = K.paged_attention(q, cache, t, ln, q_start=st, max_q=max(new), workspace=ws[:n])
        assert torch.equal(got, K.paged_attention(q, cache, t, ln, q_start=st, max_q=max(new)))
        assert (ws[n:] == 0x55).all()


def test_more_new_tokens_than_length(cuda):
    # the first rows lie before the sequence's start: they see nothing
    announce('paged prompt rows before the start')
    out = _attend(cuda, [3, 20], [10, 20], 4, 1, 64, 16)
    assert (out[:7] == 0).all()


@pytest.mark.parametrize('n', [1, 40])
def test_rows_behind_the_last_sequence_stay(cuda, n):
    announce(f'paged prompt trailing rows n={n}')
    k, v, _, _, table = _pool([50], 1, 64, 16, False, 5)
    q = torch.randn(n + 3, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = torch.full((n + 3, 4, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    K.paged_attention(q.to(cuda), K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda),
                      torch.tensor([50], dtype=torch.int32, device=cuda), out=out,
                      q_start=torch.tensor([0, n], dtype=torch.int32, device=cuda))
    want, mag = _reference(q[:n], k, v, None, None, table, [50], [n])
    _close(out[:n], want, mag)
    assert (out[n:] == 7.0).all()


@pytest.mark.parametrize('starts', [[0, 60, 20], [-5, 3, 6], [4, 4, 90], [9, 2, 5]])
def test_bad_starts_stay_inside(cuda, starts):
    # not in order, negative, past the rows: clamped, rows of no sequence stay
    announce(f'paged prompt starts {starts}')
    rows = 30
    k, v, _, _, table = _pool([64, 64], 1, 64, 16, False, 6)
    q = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = torch.full((rows, 4, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    K.paged_attention(q.to(cuda), K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda),
                      torch.tensor([64, 64], dtype=torch.int32, device=cuda), out=out,
                      q_start=torch.tensor(starts, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    clamp = [min(max(s, 0), rows) for s in starts]
    taken = set()
    for a, b in zip(clamp, clamp[1:]):
        taken |= set(range(a, max(a, b)))
    stay = [r for r in range(rows) if r not in taken]
    assert (out[stay] == 7.0).all() and torch.isfinite(out.float()).all()


@pytest.mark.parametrize('new', [[1, 1, 1], [30, 2, 9]])
def test_strided_queries(cuda, new):
    announce(f'paged strided new={new}')
    _attend(cuda, [80, 40, 9], new, 4, 2, 64, 16, ldq=800)


def test_output_may_be_a_view_and_the_queries(cuda):
    announce('paged output views')
    k, v, _, _, table = _pool([70, 300], 2, 64, 16, False, 7)
    cache = K.PagedKV(k.to(cuda), v.to(cuda))
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    lens = torch.tensor([70, 300], dtype=torch.int32, device=cuda)
    want, mag = _reference(q, k, v, None, None, table, [70, 300], [1, 1])
    buf = torch.full((2, 512), 3.0, dtype=torch.bfloat16, device=cuda)
    K.paged_attention(q.to(cuda), cache, table.to(cuda), lens,
                      out=buf[:, 128:384].unflatten(1, (4, 64)))
    _close(buf[:, 128:384].reshape(2, 4, 64), want, mag)
    assert (buf[:, :128] == 3).all() and (buf[:, 384:] == 3).all()


def test_the_largest_scores_do_not_overflow(cuda):
    announce('paged large scores')
    k, v, _, _, table = _pool([100], 1, 64, 16, False, 8)
    q = torch.full((1, 2, 64), 300.0).bfloat16()
    k[table[0, 2], 0, 5] = 100.0                  # one key takes it all
    out = K.paged_attention(q.to(cuda), K.PagedKV(k.to(cuda), v.to(cuda)), table.to(cuda),
                            torch.tensor([100], dtype=torch.int32, device=cuda))
    want = v[table[0, 2], 0, :, 5]
    assert torch.equal(out.cpu()[0], want.expand(2, 64))


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def _append_check(cuda, lens, new, heads=8, kv=1, d=128, page=16, e4m3=False, seed=1,
                  positions=None, single=None, edit=None, rows_extra=0, in_place=False,
                  max_pos=None):
    k, v, ks, vs, table = _pool([max(t, 0) for t in lens], kv, d, page, e4m3, seed)
    if edit is not None:
        edit(table)
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(new) + rows_extra
    qkv = (torch.randn(rows, (heads + 2 * kv) * d, generator=g) * 2).bfloat16()
    rope = K.rope_table(max_pos or max(max(lens), 1), d)
    single = all(n == 1 for n in new) if single is None else single
    cache = K.PagedKV(k.to(cuda), v.to(cuda), None if ks is None else ks.to(cuda),
                      None if vs is None else vs.to(cuda))
    src = qkv.to(cuda)
    q_out = src[:, :heads * d] if in_place else torch.full(
        (rows, heads * d), 9.0, dtype=torch.bfloat16, device=cuda)
    got = K.paged_append(src, cache, rope.to(cuda), table.to(cuda),
                         torch.tensor(lens, dtype=torch.int32, device=cuda), heads,
                         q_out=q_out if heads else None,
                         q_start=None if single else _starts(new).to(cuda),
                         positions=None if positions is None else
                         torch.tensor(positions, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    kw, vw = k.clone(), v.clone()
    kd, vd = _values(cache.k.cpu(), ks), _values(cache.v.cpu(), vs)
    x = qkv.double().view(rows, heads + 2 * kv, d)
    q_want, q_mag = torch.full((rows, heads, d), 9.0).double(), torch.zeros(rows, heads, d).double()
    row = 0
    half = 2.0 ** -4 if e4m3 else 2.0 ** -8
    for b, (t, n) in enumerate(zip(lens, new)):
        for i in range(n):
            at = t - n + i
            pos = positions[row] if positions is not None else at
            if 0 <= pos < rope.shape[0]:
                c, s = rope[pos, :, 0].double(), rope[pos, :, 1].double()
                y, m = x[row].clone(), x[row].clone().abs()
                e, o = x[row][:, 0::2], x[row][:, 1::2]
                y[:, 0::2], y[:, 1::2] = e * c - o * s, o * c + e * s
                m[:, 0::2] = (e * c).abs() + (o * s).abs()
                m[:, 1::2] = (o * c).abs() + (e * s).abs()
                q_want[row], q_mag[row] = y[:heads], m[:heads]
                pg = int(table[b, at // page]) if 0 <= at < table.shape[1] * page else -1
                if 0 <= pg < k.shape[0]:
                    nk, mk, nv = y[heads:heads + kv], m[heads:heads + kv], x[row, heads + kv:]
                    gk, gv = kd[pg, :, at % page], vd[pg, :, :, at % page]
                    sk = torch.ones(kv, 1) if ks is None else ks.view(-1, 1)
                    sv = torch.ones(kv, 1) if vs is None else vs.view(-1, 1)
                    if e4m3:
                        nk = (nk / sk).clamp(-448, 448) * sk
                        nv = (nv / sv).clamp(-448, 448) * sv
                    low = 2.0 ** -10 if e4m3 else 0.0
                    assert ((gk - nk).abs() <= half * nk.abs() + low * sk + 2.0 ** -21 * mk).all()
                    if e4m3:
                        assert ((gv - nv).abs() <= half * nv.abs() + low * sv +
                                2.0 ** -21 * nv.abs()).all()
                    else:
                        assert torch.equal(gv, nv)
                    kw[pg, :, at % page] = cache.k.cpu()[pg, :, at % page]
                    vw[pg, :, :, at % page] = cache.v.cpu()[pg, :, :, at % page]
            elif in_place:
                q_want[row] = x[row, :heads]
            row += 1
    if in_place:
        q_want[row:] = x[row:, :heads]
    # every other slot as it was
    assert torch.equal(cache.k.cpu().view(torch.uint8), kw.view(torch.uint8))
    assert torch.equal(cache.v.cpu().view(torch.uint8), vw.view(torch.uint8))
    if heads:
        err = (got.double().cpu().view(rows, heads, d) - q_want).abs()
        assert (err <= 2.0 ** -8 * q_want.abs() + 2.0 ** -21 * q_mag).all()


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('heads,kv,page', [(8, 1, 64), (6, 2, 16), (4, 4, 32)])
def test_append_tokens(cuda, d, e4m3, heads, kv, page):
    announce(f'paged append d={d} e4m3={e4m3} heads={heads}/{kv} page={page}')
    _append_check(cuda, [1, 16, 17, 100, 64], [1] * 5, heads, kv, d, page, e4m3)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('lens,new', [([150, 5, 70, 200], [150, 5, 1, 37]),
                                      ([3000], [2981]), ([17, 9, 40, 90], [3, 0, 0, 8])])
def test_append_prompts(cuda, d, e4m3, lens, new):
    announce(f'paged append prompts d={d} e4m3={e4m3} {lens} {new}')
    _append_check(cuda, lens, new, 10, 2, d, 32, e4m3)


def test_append_large_prompt_rows(cuda):
    announce('paged append 64-row workgroups')
    _append_check(cuda, [900, 333, 64, 1, 700], [900, 300, 64, 1, 77], 10, 1, 64, 16)


@pytest.mark.parametrize('e4m3', [False, True])
def test_append_keys_and_values_only(cuda, e4m3):
    announce(f'paged append no queries e4m3={e4m3}')
    _append_check(cuda, [50, 30], [20, 30], 0, 2, 64, 16, e4m3)


def test_append_in_place_queries(cuda):
    announce('paged append in place')
    _append_check(cuda, [50, 30], [20, 30], 4, 2, 64, 16, in_place=True)


def test_append_positions(cuda):
    # positions of their own; two outside the table: those rows stay
    announce('paged append positions')
    _append_check(cuda, [50, 30], [3, 2], 4, 2, 64, 16, positions=[7, 7, -1, 60, 0], max_pos=60)


def test_append_missing_pages_and_trailing_rows(cuda):
    def edit(table):
        table[0, 1], table[1, 0] = -1, 10 ** 6
    announce('paged append missing pages')
    _append_check(cuda, [60, 20], [50, 20], 4, 1, 64, 16, edit=edit, rows_extra=5)


def test_append_rows_before_the_start(cuda):
    announce('paged append rows before the start')
    _append_check(cuda, [3, 0, -4, 20], [5, 1, 2, 4], 4, 1, 64, 16)


def test_append_many_sequences(cuda):
    announce('paged append 1500 sequences')
    lens = [(i * 37) % 50 + 2 for i in range(1500)]
    _append_check(cuda, lens, [i % 3 for i in range(1500)], 2, 1, 64, 16)


def test_append_rounds_like_separate_operations(cuda):
    # two products and a sum, each in fp32, then one rounding: bit for bit
    announce('paged append rounding')
    qkv = torch.randn(500, 4 * 128, generator=torch.Generator().manual_seed(6)).bfloat16().to(cuda)
    cache = K.PagedKV.empty(32, 16, 1, 128, cuda)
    rope = K.rope_table(500, 128, device=cuda)
    lens = torch.tensor([500], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 500], dtype=torch.int32, device=cuda)
    q = K.paged_append(qkv, cache, rope, torch.arange(32, dtype=torch.int32, device=cuda)[None],
                       lens, 2, q_start=starts)
    x = qkv.float().view(500, 4, 128)
    a, b, c, s = x[..., 0::2], x[..., 1::2], rope[:, None, :, 0], rope[:, None, :, 1]
    want = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2).bfloat16()
    assert torch.equal(q, want[:, :2].flatten(1))
    assert torch.equal(cache.k[:, 0].flatten(0, 1)[:500], want[:, 2])


def test_append_e4m3_saturates(cuda):
    announce('paged append saturation')
    k = torch.zeros(1, 1, 16, 64, dtype=torch.uint8, device=cuda)
    v = torch.zeros(1, 1, 64, 16, dtype=torch.uint8, device=cuda)
    one = torch.full((1,), 0.5, device=cuda)
    cache = K.PagedKV(k, v, one, one)
    qkv = torch.zeros(1, 128, dtype=torch.bfloat16)
    big = torch.tensor([1e30, -1e30, 300.0, float('nan'), float('inf'), 0.0009765625, 224.0, 1.0])
    qkv[0, 64:72] = big.bfloat16()
    qkv[0, 0:8:2] = torch.tensor([1e30, -300.0, float('nan'), 1.0]).bfloat16()
    K.paged_append(qkv.to(cuda), cache, K.rope_table(4, 64, device=cuda),
                   torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                   torch.ones(1, dtype=torch.int32, device=cuda), 0)
    got = cache.v.view(F8).float().cpu()[0, 0, :8, 0]
    assert got[:3].tolist() == [448.0, -448.0, 448.0] and torch.isnan(got[3])
    # 2^-10 / 0.5 = 2^-9, the smallest step
    assert got[4:].tolist() == [448.0, 2.0 ** -9, 448.0, 2.0]
    gk = cache.k.view(F8).float().cpu()[0, 0, 0, :8]
    assert gk[0] == 448.0 and gk[2] == -448.0 and torch.isnan(gk[4]) and gk[6] == 2.0


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def _rot(x, rope, pos):
    c, s = rope[pos, :, 0].double()[:, None], rope[pos, :, 1].double()[:, None]
    y = torch.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., 1::2] * c + x[..., 0::2] * s
    return y


@pytest.mark.parametrize('e4m3', [False, True])
def test_prompt_then_tokens_in_a_graph(cuda, e4m3):
    """Two requests' prompts, then single tokens by replaying one captured
    step (append, attention, next lengths) with eager work in between, against
    attention over all tokens so far in 64 bits from what the cache holds."""
    announce(f'paged decoding loop e4m3={e4m3}')
    heads, kv, d, page, steps = 8, 2, 64, 16, 5
    g = torch.Generator().manual_seed(3)
    new = [37, 16]
    scale = torch.full((kv,), 0.02, device=cuda) if e4m3 else None
    cache = K.PagedKV.empty(8, page, kv, d, cuda, scale, scale)
    table = torch.tensor([[5, 2, 7, -1], [0, 4, 1, 3]], dtype=torch.int32, device=cuda)
    rope = K.rope_table(64, d, device=cuda)
    lens = torch.tensor(new, dtype=torch.int32, device=cuda)
    width = (heads + 2 * kv) * d
    qkv = torch.randn(sum(new), width, generator=g).bfloat16().to(cuda)
    starts = _starts(new).to(cuda)

    def check(q, out, lens_now, n):
        ks = None if scale is None else scale.cpu()
        want, mag = _reference(q.cpu().view(-1, heads, d), cache.k.cpu(), cache.v.cpu(), ks, ks,
                               table.cpu(), lens_now, n)
        _close(out, want, mag)

    q = K.paged_append(qkv, cache, rope, table, lens, heads, q_start=starts)
    out = K.paged_attention(q.view(-1, heads, d), cache, table, lens, q_start=starts,
                            max_q=max(new))
    check(q, out, new, new)
    want = _rot(qkv.cpu().double().view(-1, heads + 2 * kv, d)[:, :heads], rope.cpu(),
                list(range(37)) + list(range(16)))
    assert (q.cpu().double().view(-1, heads, d) - want).abs().max() <= 2.0 ** -8 * want.abs().max()

    step_in = torch.zeros(2, width, dtype=torch.bfloat16, device=cuda)
    step_out = torch.empty(2, heads, d, dtype=torch.bfloat16, device=cuda)
    step_q = torch.empty(2, heads * d, dtype=torch.bfloat16, device=cuda)

    def step():
        lens.add_(1)
        K.paged_append(step_in, cache, rope, table, lens, heads, q_out=step_q)
        K.paged_attention(step_q.view(2, heads, d), cache, table, lens, out=step_out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):             # warm-up outside the capture
        lens.sub_(1)
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens.copy_(torch.tensor(new, dtype=torch.int32))
    for t in range(1, steps + 1):
        step_in.copy_(torch.randn(2, width, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        now = [n + t for n in new]
        assert lens.tolist() == now
        check(step_q, step_out, now, [1, 1])
        eager = K.paged_attention(step_q.view(2, heads, d), cache, table, lens)
        assert torch.equal(eager, step_out)


def test_two_streams_at_once(cuda):
    announce('paged two streams')
    k, v, _, _, table = _pool([4000, 3000], 1, 128, 16, False, 9)
    cache = K.PagedKV(k.to(cuda), v.to(cuda))
    t = table.to(cuda)
    lens = torch.tensor([4000, 3000], dtype=torch.int32, device=cuda)
    qs = [torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(i)).bfloat16().to(cuda)
          for i in range(2)]
    want = [K.paged_attention(q, cache, t, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(K.paged_attention(qs[i], cache, t, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_workspace_contents_do_not_matter(cuda):
    announce('paged workspace')
    k, v, _, _, table = _pool([2000], 1, 64, 16, False, 10)
    cache = K.PagedKV(k.to(cuda), v.to(cuda))
    q = torch.randn(1, 8, 64, generator=torch.Generator().manual_seed(4)).bfloat16().to(cuda)
    lens = torch.tensor([2000], dtype=torch.int32, device=cuda)
    want = K.paged_attention(q, cache, table.to(cuda), lens)
    ws = torch.full((64 << 20,), 0xff, dtype=torch.uint8, device=cuda)
    for _ in range(2):
        assert torch.equal(K.paged_attention(q, cache, table.to(cuda), lens, workspace=ws), want)
    with pytest.raises(RuntimeError, match='workspace'):
        K.paged_attention(q, cache, table.to(cuda), lens, workspace=ws[:1024])


def test_python_refusals(cuda):
    announce('paged refusals')
    k, v, ks, vs, table = _pool([40, 20], 2, 64, 16, True, 11)
    kd, vd, t = k.to(cuda), v.to(cuda), table.to(cuda)
    with pytest.raises(ValueError, match='k_scale'):
        K.PagedKV(kd, vd)
    with pytest.raises(ValueError, match='v must be'):
        K.PagedKV(kd, vd[:, :1].contiguous(), ks.to(cuda), vs.to(cuda))
    with pytest.raises(ValueError, match='contiguous'):
        K.PagedKV(kd, vd[..., :8], ks.to(cuda), vs.to(cuda))
    cache = K.PagedKV(kd, vd, ks.to(cuda), vs.to(cuda))
    lens = torch.tensor([40, 20], dtype=torch.int32, device=cuda)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=cuda)
    for args, kw, text in [
            ((q.float(), cache, t, lens), {}, 'q must be'),
            ((q[:, :3], cache, t, lens), {}, 'multiple'),
            ((q[:1], cache, t, lens), {}, 'q_start'),
            ((q, cache, t.long(), lens), {}, 'page_table'),
            ((q, cache, t, lens[:1]), {}, 'kv_len'),
            ((q, cache, t, lens.cpu()), {}, 'kv_len'),
            ((q, cache, t, lens), {'q_start': lens}, 'q_start'),
            ((q, cache, t, lens), {'out': q[:1]}, 'out'),
            ((q, cache, t, lens), {'window': -1}, 'window'),
            ((q, cache, t, lens), {'softcap': -2.0}, 'softcap'),
            ((q, cache, t, lens), {'prefix_len': lens[:1]}, 'prefix_len')]:
        with pytest.raises(ValueError, match=text):
            K.paged_attention(*args, **kw)
    qkv = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=cuda)
    rope = K.rope_table(40, 64, device=cuda)
    for args, kw, text in [
            ((qkv, cache, rope, t, lens, 5), {}, 'qkv'),
            ((qkv, cache, rope[:, :16].contiguous(), t, lens, 4), {}, 'rope'),
            ((qkv, cache, rope.bfloat16(), t, lens, 4), {}, 'rope'),
            ((qkv, cache, rope, t, lens, 4), {'q_out': q[:1]}, 'q_out'),
            ((qkv, cache, rope, t, lens, 4), {'positions': lens[:1]}, 'positions')]:
        with pytest.raises(ValueError, match=text):
            K.paged_append(*args, **kw)


def test_pools_past_4_gib(cuda):
    """Pages whose byte offsets pass 32 bits."""
    announce('paged large pool')
    n, page, d = 140000, 64, 256                   # 4.6 GB each of k and v
    cache = K.PagedKV.empty(n, page, 1, d, cuda)
    ids = [n - 1, 3, 131072]
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    rope = K.rope_table(192, d, device=cuda)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(170, 10 * d, generator=g).bfloat16().to(cuda)
    lens = torch.tensor([170], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 170], dtype=torch.int32, device=cuda)
    q = K.paged_append(qkv, cache, rope, table, lens, 8, q_start=starts).view(-1, 8, d)
    out = K.paged_attention(q[-1:], cache, table, lens)
    full = K.paged_attention(q, cache, table, lens, q_start=starts)
    small = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want, mag = _reference(q.cpu(), cache.k[ids].cpu(), cache.v[ids].cpu(), None, None, small,
                           [170], [170])
    _close(out, want[-1:], mag[-1:])
    _close(full, want, mag)
