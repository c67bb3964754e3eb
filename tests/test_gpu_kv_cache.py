"""The 8-bit KV cache's operators against plain float64 computations, at the sizes
and masks where they can go wrong.

Written codes, scales and read values are exact: every step of the formula is (a
power-of-two scale, one rounding to e4m3, one to the dense type), so they are compared
for equality.  Attention's tolerance counts its roundings, per output value:

* a score is a sum of D products of a 22-bit (fp32) or exact (bf16) q and an exact
  code, added in at most D / 8 tensor-core steps that may each drop 2^-23 of the sum of
  magnitudes B = scale * sum |q| |k|: an error of at most e = B (2^-21 + D / 8 * 2^-23);
* a weight's relative error is d = e plus 2^-21 for the exponential and the exponent's
  own rounding, 2^-23 times the largest |score| in units of log2 (and 2^-12 where
  the weights are one fp16 value: bf16 rows);
* the log of the softmax's sum moves by d and the sum's own additions, and is rounded once;
* numerator and denominator each move by d, and their sums add 2^-22 a step over at
  most n / 16 + 8 steps, all relative to the largest |v|;
* the output's own rounding is half a step of its type.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
NAN = float('nan')


@pytest.fixture(scope='module', autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.fail('CUDA device required for -m gpu tests')


# ----------------------------------------------------------- plain references
def least_scale(amax):
    """The least power of two in [2^-48, 2^48] at which amax is at most 448."""
    out = torch.empty_like(amax)
    for i, a in enumerate(amax.tolist()):
        e = -48
        while e < 48 and a > 448.0 * 2.0 ** e:
            e += 1
        out[i] = 2.0 ** e
    return out


def grid(x):
    """float64 magnitudes of at most 448 to the nearest e4m3 value, ties to even; NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def plain_write(code, scale, x, table, old, new):
    """What a write leaves, in float64: code [pages, heads, page, dim], scale [pages, heads]."""
    code, scale, x = code.clone(), scale.clone(), x.double().cpu()
    page, row = code.shape[2], 0
    x = torch.where(x.abs() <= 448.0 * 2.0 ** 48, x, NAN)
    for b, (a, n) in enumerate(zip(old, new)):
        for t in range(a, a + n):
            if t > a and t % page:
                continue
            p, lo, hi = table[b][t // page], t, min(a + n, (t // page + 1) * page)
            rows = x[row + lo - a:row + hi - a].transpose(0, 1)
            need = least_scale(rows.abs().nan_to_num(0.0).amax((1, 2)))
            keep = lo % page
            if keep:
                need = torch.maximum(need, scale[p])
                again = grid(code[p, :, :keep] * (scale[p] / need)[:, None, None])
                code[p, :, :keep] = torch.where((need > scale[p])[:, None, None], again, code[p, :, :keep])
            scale[p] = need
            code[p, :, keep:keep + hi - lo] = grid(rows / need[:, None, None])
        row += n
    return code, scale


def gather(code, scale, pages, tokens):
    x = code[pages].double() * scale[pages].double()[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, code.shape[1], code.shape[3])[:tokens]


def plain_attention(q, cache, table, lens, counts, causal, scale=None):
    """out, lse and the tolerances of both, all float64."""
    dt, heads, dim = q.dtype, q.shape[1], q.shape[2]
    kv = cache.kv_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    outs, lses, tols, lse_tols = [], [], [], []
    row = 0
    for b, (t, n) in enumerate(zip(lens, counts)):
        ids = table[b][:-(-t // cache.page)]
        k = gather(cache.k, cache.k_scale, ids, t).repeat_interleave(heads // kv, 1)
        v = gather(cache.v, cache.v_scale, ids, t).repeat_interleave(heads // kv, 1)
        x = q[row:row + n].double()
        row += n
        s = torch.einsum('nhd,thd->nht', x, k) * scale
        see = torch.ones(n, t, dtype=torch.bool, device=q.device)
        if causal:
            see = torch.arange(t, device=q.device)[None] < (t - n + 1 + torch.arange(n, device=q.device))[:, None]
        s = s.masked_fill(~see[:, None], -math.inf)
        lse = torch.logsumexp(s, -1) if t else torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
        p = torch.where(see[:, None], torch.exp(s - lse[..., None]), 0.0)
        p = torch.where((~see.any(1))[:, None, None], 0.0, p)
        out = torch.einsum('nht,thd->nhd', p, torch.where(p.sum((0, 1))[:, None, None] != 0, v, 0.0))
        outs.append(out)
        lses.append(lse)
        if t:
            size = torch.einsum('nhd,thd->nht', x.abs(), k.abs().nan_to_num(0.0)).amax(-1, keepdim=True) * abs(scale)
            most = s.masked_fill(~see[:, None], 0.0).nan_to_num(0.0).abs().amax(-1, keepdim=True) * 1.45 + 60
            err = size * (2.0 ** -21 + dim / 8 * 2.0 ** -23) + 2.0 ** -21 + most * 2.0 ** -23
            if dt == torch.bfloat16:
                err = err + 2.0 ** -12
            lse_tols.append((err + (t / 16 + 8) * 2.0 ** -22).squeeze(-1) + lse.abs() * 2.0 ** -23)
            err = 2 * err + (t / 16 + 8) * 2.0 ** -22
            tols.append(err * v.abs().nan_to_num(0.0).amax() + torch.finfo(dt).eps / 2 * out.abs())
        else:
            tols.append(torch.zeros_like(out))
            lse_tols.append(torch.zeros_like(lse))
    return torch.cat(outs), torch.cat(lses), torch.cat(tols), torch.cat(lse_tols)


def check_attention(cache, q, table, lens, counts, causal, **kw):
    dev = q.device
    starts = kw.pop('starts', None)
    out, lse = cache.attention(q, table, torch.tensor(lens, dtype=torch.int32, device=dev), starts=starts, causal=causal,
                               return_lse=True, **kw)
    want, want_lse, tol, lse_tol = plain_attention(q, cache, table.tolist(), lens, counts, causal, kw.get('scale'))
    off = (out[:len(want)].double() - want).abs()
    bad = ~(off <= tol) & ~(out[:len(want)].isnan() & want.isnan())
    assert not bad.any(), (off - tol)[bad].max()
    none = want_lse == -math.inf
    assert torch.equal(lse[:len(want)] == -math.inf, none)
    assert (out[:len(want)][none] == 0).all()
    near = ~none & ~want_lse.isnan()
    assert ((lse[:len(want)].double() - want_lse).abs() <= lse_tol)[near].all()
    cache.check()
    return out, lse


# ------------------------------------------------------------------ set-up
def filled(pages, kv, page, dim, seed, dev='cuda'):
    """A cache with ordinary contents in every page."""
    from rapidtinyrec_b200.kv_cache import KvCache8
    g = torch.Generator().manual_seed(seed)
    cache = KvCache8.allocate(pages, kv, page, dim, dev)
    for code, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        scale.copy_(torch.exp2(torch.randint(-9, -5, (pages, kv), generator=g).float()))
        code.copy_((torch.randn(pages, kv, page, dim, generator=g) * 80).clamp(-448, 448).to(F8))
    return cache


def tables(total, page, pages, seed, width=None, dev='cuda'):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    need = [-(-t // page) for t in total]
    rows = torch.full((len(total), width or max(1, *need)), 0, dtype=torch.int32)
    for b, n in enumerate(need):
        rows[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return rows.to(dev)


def cuts(counts, dev='cuda', first=0):
    out = [first]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=dev)


def ints(x, dev='cuda'):
    return torch.tensor(x, dtype=torch.int32, device=dev)


SHAPES = [(12, 2, 128), (14, 2, 64), (28, 4, 128), (4, 4, 64), (8, 1, 128), (9, 1, 64)]
DTYPES = [torch.float32, torch.bfloat16]


# ------------------------------------------------------------ write and read
@pytest.mark.parametrize('page', [16, 32, 64, 128])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('dtype', DTYPES)
def test_write_gives_the_formulas_codes_and_scales(page, dim, dtype):
    old = [0, 0, 1, page - 1, page, page + 5, 0, 3]
    new = [1, 2 * page + 3, 0, 2, page, page - 6, 0, 2 * page]
    total = [a + n for a, n in zip(old, new)]
    pages, kv = sum(-(-t // page) for t in total) + 2, 3
    cache = filled(pages, kv, page, dim, seed=page + dim)
    table = tables(total, page, pages, seed=1)
    g = torch.Generator().manual_seed(2)
    rows = sum(new)
    k = torch.randn(rows, kv, dim, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, kv, 1), generator=g).float())
    v = torch.randn(rows, kv, dim, generator=g)
    k, v = k.to(dtype).cuda(), v.to(dtype).cuda()
    want = [plain_write(c.double().cpu(), s.double().cpu(), x, table.tolist(), old, new)
            for c, s, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v))]
    cache.write(k, v, table, ints(total), starts=cuts(new))
    for (code, scale), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(s.double().cpu(), scale)
        assert torch.equal(c.double().cpu(), code)
    # a second time: the same pages, the same result
    cache.write(k, v, table, ints(total), starts=cuts(new))
    assert torch.equal(cache.k.double().cpu(), want[0][0]) and torch.equal(cache.v_scale.double().cpu(), want[1][1])
    # and back: every value times a power of two is exact in float32, one rounding in bf16
    got = cache.read(rows, table, ints(total), starts=cuts(new), dtype=dtype)
    for x, code, scale in ((got[0], cache.k, cache.k_scale), (got[1], cache.v, cache.v_scale)):
        at = 0
        for b, (a, n) in enumerate(zip(old, new)):
            ref = gather(code, scale, table[b].tolist(), a + n)[a:]
            assert torch.equal(x[at:at + n].double(), ref.to(dtype).double())
            at += n
    cache.check()


def test_write_takes_extreme_values():
    from rapidtinyrec_b200.kv_cache import KvCache8
    big = 448.0 * 2.0 ** 48
    cache = KvCache8.allocate(8, 1, 16, 64)
    rows = torch.zeros(6 * 16, 1, 64, device='cuda')
    rows[0, 0, :4] = torch.tensor([NAN, math.inf, -math.inf, 1.0])                 # page 0: scale of the 1.0
    rows[16, 0, :3] = torch.tensor([big, -big, math.nextafter(big, math.inf) * 1.001])  # page 1: the largest scale
    rows[32, 0, :3] = torch.tensor([1e-40, 2.0 ** -57, 1e-14])                       # page 2: below the least scale
    rows[48] = 0                                                                      # page 3: nothing but zeros
    rows[64, 0, :2] = torch.tensor([448.0, 17.0])                                    # page 4: 448 exactly
    rows[80, 0, :3] = torch.tensor([448.0001, 17.0, 1.0625])                         # page 5: a little more; ties to even
    table = ints([[0, 1, 2, 3, 4, 5]])
    want = plain_write(torch.zeros(8, 1, 16, 64, dtype=torch.float64), torch.ones(8, 1, dtype=torch.float64), rows,
                       table.tolist(), [0], [96])
    cache.write(rows, rows, table, ints([96]))
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert torch.equal(s.double().cpu(), want[1])
        torch.testing.assert_close(c.double().cpu(), want[0], rtol=0, atol=0, equal_nan=True)
    assert cache.k_scale[1].item() == 2.0 ** 48 and cache.k_scale[2].item() == 2.0 ** -48 and cache.k_scale[4].item() == 1
    cache.check()


def test_tokens_written_one_by_one_match_the_formula_at_every_step():
    page, kv, dim, n = 16, 2, 64, 37
    cache = filled(4, kv, page, dim, seed=3)
    table = ints([[2, 0, 3]])
    g = torch.Generator().manual_seed(4)
    x = torch.randn(n, kv, dim, generator=g) * torch.exp2(torch.linspace(-4, 6, n))[:, None, None]  # scales grow
    code, scale = cache.k.double().cpu(), cache.k_scale.double().cpu()
    for t in range(n):
        code, scale = plain_write(code, scale, x[t:t + 1], table.tolist(), [t], [1])
        cache.write(x[t:t + 1].cuda(), x[t:t + 1].cuda(), table, ints([t + 1]))
        assert torch.equal(cache.k.double().cpu(), code) and torch.equal(cache.k_scale.double().cpu(), scale), t
    assert torch.equal(cache.v.view(torch.uint8)[2, :, :, :], cache.k.view(torch.uint8)[2])


def test_scales_from_elsewhere_are_kept_and_divided_by():
    """An old scale that is no power of two: codes are x / scale, rounded once."""
    cache = filled(2, 1, 16, 64, seed=5)
    cache.k_scale.fill_(0.3)
    cache.v_scale.fill_(0.3)
    table, x = ints([[1]]), torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(6)).cuda()
    cache.write(x, x, table, ints([6]))
    want = (x[0, 0] / cache.k_scale[1, 0]).to(F8)  # float32 division, one rounding
    assert cache.k_scale[1, 0].item() == torch.tensor(0.3).item()
    assert torch.equal(cache.k[1, 0, 5].float(), want.float())


def test_an_old_scale_that_is_none_is_reported_and_its_page_left():
    from rapidtinyrec_b200._native import NativeError
    for bad in (0.0, -1.0, NAN, math.inf):
        cache = filled(2, 2, 16, 64, seed=7)
        cache.k_scale[1, 1] = bad
        before = cache.k.view(torch.uint8).clone()
        x = torch.ones(1, 2, 64, device='cuda')
        cache.write(x, x, ints([[1]]), ints([4]))
        with pytest.raises(NativeError, match='scale'):
            cache.check()
        cache.check()
        assert torch.equal(cache.k.view(torch.uint8)[1, 1], before[1, 1])
        assert not torch.equal(cache.k.view(torch.uint8)[1, 0], before[1, 0])


def test_strides_of_rows_and_of_the_cache():
    """Rows cut out of a fused projection, outputs inside larger tensors, the heads of one layer."""
    page, dim, kv, layers = 32, 128, 2, 3
    whole = filled(9, kv * layers, page, dim, seed=8)
    total = [40, 33, 64]
    table = tables(total, page, 9, seed=9, width=5)[:, :2]  # table rows further apart than their width
    g = torch.Generator().manual_seed(10)
    fused = torch.randn(sum(total), 8 + 2 * kv, dim, generator=g).bfloat16().cuda()
    before = whole.k.view(torch.uint8).clone()
    one = whole.heads(kv, kv)
    one.write(fused[:, 8:8 + kv], fused[:, 8 + kv:], table, ints(total), starts=cuts(total))
    assert torch.equal(whole.k.view(torch.uint8)[:, :kv], before[:, :kv])
    assert torch.equal(whole.k.view(torch.uint8)[:, 2 * kv:], before[:, 2 * kv:])
    from rapidtinyrec_b200.kv_cache import KvCache8
    own = KvCache8(one.k.contiguous(), one.v.contiguous(), one.k_scale.contiguous(), one.v_scale.contiguous())
    big = torch.full((sum(total), 2, 2 * kv, dim), 7.0, device='cuda')
    one.read(sum(total), table, ints(total), starts=cuts(total), out=(big[:, 0, :kv], big[:, 1, kv:]))
    k, v = own.read(sum(total), table, ints(total), starts=cuts(total))
    assert torch.equal(big[:, 0, :kv], k) and torch.equal(big[:, 1, kv:], v)
    assert (big[:, 0, kv:] == 7).all() and (big[:, 1, :kv] == 7).all()
    # heads-first rows [kv, rows, dim], as the prefix arena holds them
    first = fused[:, 8:8 + kv].transpose(0, 1).contiguous().transpose(0, 1)
    own.write(first, first, table, ints(total), starts=cuts(total))
    one.write(fused[:, 8:8 + kv], fused[:, 8:8 + kv], table, ints(total), starts=cuts(total))
    assert torch.equal(own.v.view(torch.uint8), one.v.contiguous().view(torch.uint8))
    q = fused[:, :8]
    out, _ = check_attention(one, q, table, total, total, True, starts=cuts(total))
    assert torch.equal(out, own.attention(q.contiguous(), table, ints(total), starts=cuts(total)))
    # an odd address is copied, not refused
    shifted = torch.empty(q.numel() + 1, dtype=q.dtype, device='cuda')[1:].view(q.shape).copy_(q)
    assert torch.equal(one.attention(shifted, table, ints(total), starts=cuts(total)), out)


def test_a_cache_with_its_heads_outermost():
    from rapidtinyrec_b200.kv_cache import KvCache8
    a = filled(40, 3, 32, 64, seed=85)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (a.k, a.v)]
    assert turned[0].stride(1) > turned[0].stride(0)
    b = KvCache8(*turned, a.k_scale.clone(), a.v_scale.clone())
    counts, lens = [3, 40, 1], [90, 500, 33]
    table = tables(lens, 32, 40, seed=86)
    x = torch.randn(44, 3, 64, device='cuda')
    for cache in (a, b):
        cache.write(x, 2 * x, table, ints(lens), starts=cuts(counts))
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)
    for one, two in zip(*(c.read(44, table, ints(lens), starts=cuts(counts)) for c in (a, b))):
        assert torch.equal(one, two)
    for dtype in DTYPES:
        q = torch.randn(44, 12, 64, device='cuda').to(dtype)
        out, _ = check_attention(b, q, table, lens, counts, True, starts=cuts(counts))
        assert torch.equal(out, a.attention(q, table, ints(lens), starts=cuts(counts)))
    cut = b.heads(1, 2)
    q = torch.randn(1500, 12, 64, device='cuda')
    check_attention(cut, q, table[1:2], [500], [1500], False)


# --------------------------------------------------------------- attention
@pytest.mark.parametrize('heads,kv,dim', SHAPES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('page', [16, 64])
def test_one_token_a_sequence(heads, kv, dim, dtype, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 128, 300, 0, 257]
    pages = sum(-(-t // page) for t in lens) + 1
    cache = filled(pages, kv, page, dim, seed=heads + dim)
    table = tables(lens, page, pages, seed=11)
    q = 2 * torch.randn(len(lens), heads, dim, generator=torch.Generator().manual_seed(12))
    check_attention(cache, q.to(dtype).cuda(), table, lens, [1] * len(lens), True)


@pytest.mark.parametrize('heads,kv,dim', SHAPES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
def test_ragged_rows(heads, kv, dim, dtype, causal):
    """New rows of different numbers: none, one, more than the sequence holds (rows that see
    nothing), tiles that end inside a sequence."""
    page = 32
    counts = [3, 0, 1, 40, 17, 5, 64, 2]
    lens = [3, 50, 0, 45, 400, 2, 64, 129]  # the sixth: 5 rows of a sequence of 2
    pages = sum(-(-t // page) for t in lens) + 1
    cache = filled(pages, kv, page, dim, seed=heads + dim + 1)
    table = tables(lens, page, pages, seed=13)
    q = 2 * torch.randn(sum(counts), heads, dim, generator=torch.Generator().manual_seed(14))
    check_attention(cache, q.to(dtype).cuda(), table, lens, counts, causal, starts=cuts(counts))


@pytest.mark.parametrize('dtype', DTYPES)
def test_many_short_sequences(dtype):
    counts = [b % 3 for b in range(300)]
    lens = [(7 * b) % 40 + 2 for b in range(300)]
    cache = filled(900, 2, 16, 64, seed=43)
    table = tables(lens, 16, 900, seed=44)
    q = torch.randn(sum(counts), 6, 64, generator=torch.Generator().manual_seed(45)).to(dtype).cuda()
    check_attention(cache, q, table, lens, counts, True, starts=cuts(counts))
    x = q[:, :2].contiguous()
    old = [t - n for t, n in zip(lens, counts)]
    want = [plain_write(c.double().cpu(), s.double().cpu(), x, table.tolist(), old, counts)
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    cache.write(x, x, table, ints(lens), starts=cuts(counts))
    for (code, scale), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(s.double().cpu(), scale) and torch.equal(c.double().cpu(), code)
    back = cache.read(len(x), table, ints(lens), starts=cuts(counts))
    for r, c, s in zip(back, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        want = torch.cat([gather(c, s, table[b].tolist(), lens[b])[old[b]:] for b in range(len(lens))])
        assert torch.equal(r.double(), want)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tokens', [2047, 2048, 2049, 6000])
def test_long_sequences_split_over_blocks(dtype, tokens):
    cache = filled(64, 2, 128, 128, seed=15)
    table = tables([tokens, 100], 128, 64, seed=16)
    q = torch.randn(2, 12, 128, generator=torch.Generator().manual_seed(17)).to(dtype).cuda()
    check_attention(cache, q, table, [tokens, 100], [1, 1], True)
    check_attention(cache, q, table, [tokens, 0], [1, 1], True)


@pytest.mark.parametrize('dtype', DTYPES)
def test_long_rows_of_several_tokens(dtype):
    cache = filled(64, 2, 128, 64, seed=18)
    table = tables([5000, 2100], 128, 64, seed=19)
    counts = [150, 33]
    q = torch.randn(183, 14, 64, generator=torch.Generator().manual_seed(20)).to(dtype).cuda()
    for causal in (True, False):
        check_attention(cache, q, table, [5000, 2100], counts, causal, starts=cuts(counts))


def test_sizes_of_queries_and_scales():
    """Tiny and huge queries, pages whose scales differ by 2^60, a softmax scale of its own."""
    cache = filled(8, 2, 16, 64, seed=21)
    table = tables([100], 16, 8, seed=22)
    g = torch.Generator().manual_seed(23)
    for size in (1e-30, 1e-6, 1.0, 30.0):
        q = (torch.randn(5, 4, 64, generator=g) * size).cuda()
        check_attention(cache, q, table, [100], [5], True)
        check_attention(cache, q, table, [100], [5], False, scale=0.02)
    q = torch.randn(5, 4, 64, generator=g).cuda()
    cache.v_scale.copy_(torch.exp2(torch.randint(-30, 30, (8, 2), generator=g).float()))
    check_attention(cache, q, table, [100], [5], True)
    cache.v_scale.copy_(torch.rand(8, 2, generator=g) + 0.1)  # no powers of two
    cache.k_scale.copy_(torch.rand(8, 2, generator=g) * 0.01 + 0.001)
    check_attention(cache, q, table, [100], [5], True)
    check_attention(cache, torch.zeros_like(q), table, [100], [5], True)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('counts', [[20], [150]])
def test_nan_stays_with_the_rows_that_see_it(dtype, counts):
    n = counts[0]
    cache = filled(12, 1, 16, 64, seed=24)
    table = tables([160], 16, 12, seed=25)
    code = cache.v.view(torch.uint8)
    last = table.tolist()[0]
    code[last[-1]] = 0x7f            # tokens 144 .. 159 of V: behind the sequence's last (lens 158) and its last ones
    cache.k.view(torch.uint8)[last[-1], :, 13:] = 0xff  # K of tokens 157 ..
    code[last[-1], :, :13] = 0x10
    code[last[-1], 0, 12, 5] = 0xff  # V of token 156, dimension 5
    q = torch.randn(n, 6, 64, generator=torch.Generator().manual_seed(26)).to(dtype).cuda()
    out = cache.attention(q, table, ints([158]), starts=cuts(counts))
    nan = out.isnan()
    assert not nan[:n - 2].any()                       # rows at tokens up to 155
    assert nan[n - 2, :, 5].all() and nan[n - 2].sum() == 6  # the row at token 156: dimension 5 alone
    assert nan[n - 1].all()                            # the row at token 157 sees a NaN score
    clean = cache.attention(q[:n - 2], table, ints([156]), starts=cuts([n - 2]))
    check_attention(cache, q[:n - 2], table, [156], [n - 2], True, starts=cuts([n - 2]))
    assert torch.allclose(out[:n - 2].float(), clean.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
    # a query that is NaN or infinite spoils its own row alone
    q[1, 2, 3], q[4, 0, 0] = NAN, math.inf
    nan = cache.attention(q[:n - 2], table, ints([156])).isnan()
    want = torch.zeros_like(nan)
    want[1, 2] = want[4, 0] = True
    assert torch.equal(nan, want)


# ------------------------------------------------------------- 128-row tiles
# Sizes at which the tiles of 128 rows are expected to be the faster ones by a wide margin:
# some thousand rows a KV head over more than a thousand keys.
TILED = [(12, 2, 128), (14, 2, 64)]


@pytest.mark.parametrize('heads,kv,dim', TILED)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
def test_tiles_of_128_rows(heads, kv, dim, dtype, causal):
    """Ragged sequences, some with more rows than tokens or none; one longer than a block's keys."""
    counts = [700, 0, 1, 300, 129, 1400]
    lens = [1300, 900, 0, 120, 9000, 1500]
    pages = sum(-(-t // 64) for t in lens) + 1
    cache = filled(pages, kv, 64, dim, seed=heads + dim + 2)
    table = tables(lens, 64, pages, seed=46)
    g = torch.Generator().manual_seed(47)
    q = (2 * torch.randn(sum(counts), heads, dim, generator=g)).to(dtype).cuda()
    check_attention(cache, q, table, lens, counts, causal, starts=cuts(counts))
    for scale in (0.0, -0.05):
        check_attention(cache, q[:1400], table[:1], lens[:1], [1400], causal, scale=scale)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tokens', [1100, 9000])
def test_tiles_of_an_own_length(dtype, tokens):
    """Rows of one sequence, scales 2^60 apart and no powers of two, tiny and huge queries."""
    cache = filled(80, 2, 128, 128, seed=48)
    table = tables([tokens], 128, 80, seed=49)
    g = torch.Generator().manual_seed(50)
    cache.v_scale.copy_(torch.exp2(torch.randint(-30, 30, (80, 2), generator=g).float()))
    cache.k_scale.copy_(torch.rand(80, 2, generator=g) * 0.01 + 0.001)
    for size in (1e-30, 1.0, 30.0):
        q = (torch.randn(1000, 12, 128, generator=g) * size).to(dtype).cuda()
        check_attention(cache, q, table, [tokens], [1000], True)


@pytest.mark.parametrize('dtype', DTYPES)
def test_tiles_keep_nan_with_the_rows_that_see_it(dtype):
    n, tokens, page = 1000, 1300, 32
    cache = filled(50, 1, page, 64, seed=51)
    table = tables([tokens], page, 50, seed=52)
    pages = table.tolist()[0]
    q = torch.randn(n, 14, 64, generator=torch.Generator().manual_seed(53)).to(dtype).cuda()
    before = cache.attention(q, table, ints([tokens]))
    code = cache.v.view(torch.uint8)
    code[pages[1100 // page], 0, 1100 % page, 5] = 0xff       # V of token 1100, dimension 5
    cache.k.view(torch.uint8)[pages[1250 // page], 0, 1250 % page, 7] = 0x7f  # K of token 1250
    code[pages[-1], 0, tokens % page:] = 0x7f                 # behind the last token
    cache.k.view(torch.uint8)[pages[-1], 0, tokens % page:] = 0x7f
    cache.v_scale[pages[1280 // page]] = 0.0                  # tokens 1280 ..
    out = cache.attention(q, table, ints([tokens]))
    nan = out.isnan()
    first = tokens - n  # the token of row 0
    assert not nan[:1100 - first].any() and torch.equal(out[:1100 - first], before[:1100 - first])
    some = nan[1100 - first:1250 - first]
    assert some[:, :, 5].all() and some.sum() == some.shape[0] * 14
    assert nan[1250 - first:].all()
    # the row at token 1279 sees all but the page without a scale; what it sees has the NaN
    ok = torch.ones(64, dtype=torch.bool)
    ok[5] = False
    assert torch.equal(out[1100 - first:1250 - first][..., ok], before[1100 - first:1250 - first][..., ok])
    # queries that are NaN or infinite spoil their own rows alone
    q[1, 2, 3], q[130, 0, 0] = NAN, math.inf
    nan = cache.attention(q[:700], table, ints([1000])).isnan()
    want = torch.zeros_like(nan)
    want[1, 2] = want[130, 0] = True
    assert torch.equal(nan, want)
    # a page number outside the cache, in the last page: the rows before it are whole
    from rapidtinyrec_b200._native import NativeError
    table[0, 1000 // page - 1] = 50
    out = cache.attention(q[:700], table, ints([1000]))
    with pytest.raises(NativeError, match='page'):
        cache.check()
    behind = (1000 // page - 1) * page - (1000 - 700)  # the first row that sees it
    assert out[behind:].isnan().all() and not out[131:behind].isnan().any()


# ------------------------------------------------------------- 256-row tiles
# bf16, head_dim 128: enough rows to fill the GPU with blocks of 256, some of them split along
# the keys and joined (more than 148 blocks or more than 16,384 keys).
def tails(cache, q, table, lens, starts=None):
    """Whether the call is one of 256-row tiles with split ones: 4 bytes for each of their rows beside
    the sums' 8 + 4 * head_dim."""
    from rapidtinyrec_b200 import _native
    b = _native.KvBatchC(table.data_ptr(), lens.data_ptr(), None if starts is None else starts.data_ptr(), table.shape[1],
                         table.shape[1], table.shape[0], q.shape[0])
    need = ctypes.c_int64()
    assert _native.load().rtr_kv_attention_workspace(ctypes.byref(cache._c), ctypes.byref(b), _native.RTR_DTYPE_BF16,
                                                     q.shape[1], 0, ctypes.byref(need)) == 0
    return need.value % 520 != 0


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('page', [16, 128])
def test_tiles_of_256_rows(causal, page):
    """Ragged sequences as in the test of 128 rows: whole blocks, and split ones at the end."""
    counts = [500, 0, 1, 300, 129, 400]
    lens = [1300, 900, 0, 120, 9000, 1500]
    pages = sum(-(-t // page) for t in lens) + 1
    cache = filled(pages, 4, page, 128, seed=page + 60)
    table = tables(lens, page, pages, seed=61)
    g = torch.Generator().manual_seed(62)
    q = (2 * torch.randn(sum(counts), 28, 128, generator=g)).bfloat16().cuda()
    assert tails(cache, q, table, ints(lens), cuts(counts))
    check_attention(cache, q, table, lens, counts, causal, starts=cuts(counts))
    # rows in front of and behind the sequences', in a tensor of NaN
    starts = cuts(counts, first=3)
    wide = torch.cat((q[:3], q, q[:5]))
    out = torch.full_like(wide, NAN)
    cache.attention(wide, table, ints(lens), starts=starts, causal=causal, out=out)
    assert out[:3].isnan().all() and out[-5:].isnan().all() and not out[3:-5].isnan().any()


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('rows', [1300, 1290])
def test_tiles_of_256_rows_without_starts(causal, rows):
    """Whole blocks only; the last block has both of its tiles, or one."""
    cache = filled(40, 4, 64, 128, seed=63)
    table = tables([2000], 64, 40, seed=64)
    q = (2 * torch.randn(rows, 28, 128, generator=torch.Generator().manual_seed(65))).bfloat16().cuda()
    for scale in (None, 0.0, -0.05):
        out, _ = check_attention(cache, q, table, [2000], [rows], causal, **({} if scale is None else dict(scale=scale)))
    # again, on another stream and from a captured graph
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        assert torch.equal(cache.attention(q, table, ints([2000]), causal=causal, scale=-0.05), out)
    torch.cuda.synchronize()
    lens, given = ints([2000]), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(q, table, lens, causal=causal, scale=-0.05, out=given)
    for _ in range(2):
        given.fill_(NAN)
        graph.replay()
        assert torch.equal(given, out)


@pytest.mark.parametrize('heads,kv,rows', [(16, 16, 2300), (40, 1, 900), (300, 1, 130)])
def test_tiles_of_256_rows_of_other_groups(heads, kv, rows):
    """One head a group, more than a tile's half and more than a tile; q, K and V slices of larger
    tensors."""
    whole = filled(50, kv + 3, 32, 128, seed=72)
    cache = whole.heads(2, kv)
    table = tables([1300], 32, 50, seed=73)
    g = torch.Generator().manual_seed(74)
    fused = torch.randn(rows, heads + 5, 128, generator=g).bfloat16().cuda()
    q = fused[:, 3:3 + heads]
    out, _ = check_attention(cache, q, table, [1300], [rows], True)
    assert torch.equal(cache.attention(q.contiguous(), table, ints([1300])), out)
    check_attention(cache, q, table, [1300], [rows], False, scale=0.3)


@pytest.mark.parametrize('size', [1e-30, 1.0, 30.0])
def test_tiles_of_256_rows_over_many_keys(size):
    """More keys than one block takes; scales 2^60 apart and no powers of two, tiny and huge
    queries; rows that see nothing of the last stretches; a row that sees a single key."""
    cache = filled(140, 4, 128, 128, seed=66)
    g = torch.Generator().manual_seed(67)
    cache.v_scale.copy_(torch.exp2(torch.randint(-30, 30, (140, 4), generator=g).float()))
    cache.k_scale.copy_(torch.rand(140, 4, generator=g) * 0.01 + 0.001)
    table = tables([17000], 128, 140, seed=68)
    q = (torch.randn(400, 28, 128, generator=g) * size).bfloat16().cuda()
    assert tails(cache, q, table, ints([17000]))
    check_attention(cache, q, table, [17000], [400], True)
    if size == 1.0:
        for length in (400, 399, 1, 0, 129):  # of a table row for many more
            check_attention(cache, q, table, [length], [400], True)
            check_attention(cache, q, table, [length], [400], False)


@pytest.mark.parametrize('n,tokens,heads,kv,page', [(1300, 2000, 28, 4, 32), (1000, 17000, 12, 2, 128)])
def test_tiles_of_256_rows_keep_nan_with_the_rows_that_see_it(n, tokens, heads, kv, page):
    """Rows that do not see a NaN stay as they are up to when their maximum was taken: every
    fp16 weight may round otherwise, 2^-11 of it each time (V is at most 448 * 2^-6 = 7), then the
    output's bf16."""
    from rapidtinyrec_b200._native import NativeError
    pages = -(-tokens // page)
    cache = filled(pages, kv, page, 128, seed=69)
    table = tables([tokens], page, pages, seed=70)
    ids = table.tolist()[0]
    q = torch.randn(n, heads, 128, generator=torch.Generator().manual_seed(71)).bfloat16().cuda()
    before = cache.attention(q, table, ints([tokens]))

    def same(a, b):
        return ((a.float() - b.float()).abs() <= 7 * 2.0 ** -10 + 1e-5 + b.float().abs() * 2.0 ** -8).all()

    t0 = tokens - n  # the token of row 0
    v_at, k_at, bad = tokens - 200, tokens - 150, (tokens - 40) // page * page
    cache.v.view(torch.uint8)[ids[v_at // page], :, v_at % page, 5] = 0xff
    out = cache.attention(q, table, ints([tokens]))
    nan = out.isnan()
    want = torch.zeros_like(nan)
    want[v_at - t0:, :, 5] = True
    assert torch.equal(nan, want) and same(out[~want], before[~want])
    cache.k.view(torch.uint8)[ids[k_at // page], :, k_at % page, 7] = 0x7f
    nan = cache.attention(q, table, ints([tokens])).isnan()
    want[k_at - t0:] = True
    assert torch.equal(nan, want)
    # behind the last token nothing counts
    last = tokens % page
    if last:
        cache.v.view(torch.uint8)[ids[-1], :, last:] = 0x7f
        cache.k.view(torch.uint8)[ids[-1], :, last:] = 0x7f
    assert torch.equal(cache.attention(q, table, ints([tokens])).isnan(), want)
    # a query with a NaN or an infinite value spoils its own row
    q[1, 2, 3], q[130, 0, 0], q[40] = NAN, math.inf, -math.inf
    nan = cache.attention(q, table, ints([tokens])).isnan()
    want[1, 2] = want[130, 0] = want[40] = True
    assert torch.equal(nan, want)
    # a page without a scale, then one outside the cache: the rows that see it
    cache.v_scale[ids[bad // page]] = 0.0
    want[bad - t0:] = True
    assert torch.equal(cache.attention(q, table, ints([tokens])).isnan(), want)
    first = (t0 + 600) // page * page
    table[0, first // page] = pages
    want[first - t0:] = True
    assert torch.equal(cache.attention(q, table, ints([tokens])).isnan(), want)
    with pytest.raises(NativeError, match='page'):
        cache.check()
    # a length that the table cannot hold
    assert cache.attention(q, table, ints([pages * page + 1])).isnan().all()
    with pytest.raises(NativeError, match='length'):
        cache.check()


# ------------------------------------------- keys that outweigh all others together
# One row, stretches of one cluster, stretches joined by a kernel; tiles of 128 and 256 rows.
OUTWEIGHED = [(torch.float32, 12, 2, 128, 1, 700), (torch.float32, 14, 2, 64, 3, 3000), (torch.float32, 12, 2, 128, 2, 20000),
              (torch.bfloat16, 12, 2, 128, 1, 700), (torch.bfloat16, 14, 2, 64, 3, 3000), (torch.bfloat16, 12, 2, 128, 2, 20000),
              (torch.float32, 12, 2, 128, 1000, 2300), (torch.float32, 14, 2, 64, 1000, 2300),
              (torch.bfloat16, 14, 2, 64, 1000, 2300), (torch.bfloat16, 28, 4, 128, 1300, 2000)]


@pytest.mark.parametrize('dtype,heads,kv,dim,rows,tokens', OUTWEIGHED)
@pytest.mark.parametrize('by', ['score', 'scale'])
def test_keys_beside_one_that_outweighs_them(dtype, heads, kv, dim, rows, tokens, by):
    """One key (or one page's V scale) outweighs all others by up to 2^26 (fp32: 2^32) and its V is 0: the
    output is what the others give.  All V are positive, so every error is relative to the output.

    Scores are one exact product: x = 45 in units of log2 at most, and the six roundings of its factors
    and of the exponent move a weight by 6 * 2^-24 * 64 * ln 2 < 2^-15.  A weight has 22 bits (2^-22;
    one fp16 value: 2^-12), or is off by half a step of the operand: 2^-40 of the largest of its 128 keys
    (fp32; the other tiles' weights are exact to 22 bits, and where one row's running maximum counts
    for all keys it is 2^-51) and 2^-35 of the row's largest (bf16).  Positive
    terms are added in at most tokens / 16 + 64 steps of 2^-22; the output's own rounding comes last.
    """
    page, most = 32, 32 if dtype == torch.float32 else 26
    pages = -(-tokens // page)
    cache = filled(pages, kv, page, dim, seed=80)
    g = torch.Generator().manual_seed(81)
    table = tables([tokens], page, pages, seed=82)
    ids = table.tolist()[0]
    cache.v.copy_((torch.randint(8, 449, cache.v.shape, generator=g).float()).to(F8))
    cache.v_scale.fill_(2.0 ** -7)
    cache.k_scale.fill_(2.0 ** -3)
    # log2 of the factor, for each row: eighths, which bf16 holds and 2^x does not make round numbers of
    more = torch.randint(8 * (most - 10), 8 * most, (rows, heads), generator=g).double() / 8
    for at in (0, tokens // 2, tokens - 1):
        v, vs = cache.v.clone(), cache.v_scale.clone()
        cache.k.zero_()
        q = torch.zeros(rows, heads, dim, device='cuda')
        if by == 'score':
            cache.k[ids[at // page], :, at % page, 0] = 8.0  # times 2^-3: the score is scale * q
            cache.v[ids[at // page], :, at % page] = 0.0
            q[..., 0] = more.float().cuda()
        else:
            cache.v[ids[at // page]] = 0.0
            cache.v_scale[ids[at // page]] = 1.3 * 2.0 ** (most - 8)  # and the others' weights no round numbers
        out, lse = cache.attention(q.to(dtype), table, ints([tokens]), causal=False, scale=math.log(2.0), return_lse=True)
        want, want_lse, _, _ = plain_attention(q.to(dtype).double(), cache, table.tolist(), [tokens], [rows], False, math.log(2.0))
        low = 2.0 ** (most - 40) * min(1.0, 256 / tokens) if dtype == torch.float32 else 2.0 ** (most - 35)
        rel = 2.0 ** -15 + (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -12) + low + (tokens / 16 + 64) * 2.0 ** -22
        off = (out.double() - want).abs() / want
        assert off.max() <= rel + torch.finfo(dtype).eps / 2, (at, off.max())
        assert (lse.double() - want_lse).abs().max() <= rel + want_lse.abs().max() * 2.0 ** -22
        cache.v.copy_(v)
        cache.v_scale.copy_(vs)
    cache.check()


@pytest.mark.parametrize('dtype,heads,kv,dim,rows,tokens', OUTWEIGHED)
@pytest.mark.parametrize('low', ['first', 'last'])
def test_scores_beyond_float_in_some_pages(dtype, heads, kv, dim, rows, tokens, low):
    """Most pages hold K so large that every score is minus infinity in float (2^75 * 448 * 2^48 * dim), the
    others zeros: the output is the mean of their V, whichever block has which.  Weights are equal and
    exact or one fp16 value (2^-12), their positive terms added in tokens / 16 + 64 steps of 2^-22."""
    page = 32
    pages = -(-tokens // page)
    cache = filled(pages, kv, page, dim, seed=87)
    g = torch.Generator().manual_seed(88)
    table = tables([tokens], page, pages, seed=89)
    ids = table.tolist()[0]
    cache.v.copy_((torch.randint(8, 449, cache.v.shape, generator=g).float()).to(F8))
    cache.v_scale.fill_(2.0 ** -7)
    cache.k.zero_()
    cut = pages * 17 // 20 if low == 'first' else pages * 3 // 20
    for p in ids[:cut] if low == 'first' else ids[cut:]:
        cache.k[p], cache.k_scale[p] = 448.0, 2.0 ** 48
    q = torch.full((rows, heads, dim), -2.0 ** 75, device='cuda').to(dtype)
    out, lse = cache.attention(q, table, ints([tokens]), causal=False, return_lse=True)
    v = gather(cache.v, cache.v_scale, ids, tokens)
    v = v[cut * page:] if low == 'first' else v[:cut * page]
    want = v.mean(0).repeat_interleave(heads // kv, 0)
    rel = (0.0 if dtype == torch.float32 else 2.0 ** -12) + (tokens / 16 + 64) * 2.0 ** -22
    off = ((out.double() - want).abs() / want).max()
    assert off <= rel + torch.finfo(dtype).eps / 2, off
    assert (lse.double() - math.log(len(v))).abs().max() <= rel + 2.0 ** -20
    # where no key is left that counts, 0 / 0
    cache.k.fill_(448.0)
    cache.k_scale.fill_(2.0 ** 48)
    assert cache.attention(q, table, ints([tokens]), causal=False).isnan().all()
    cache.check()


def test_bad_k_scales_make_their_rows_nan():
    cache = filled(4, 1, 16, 64, seed=54)
    table = ints([[0, 1], [2, 3]])
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(55)).cuda()
    for bad in (-1.0, NAN):
        cache.k_scale[1] = bad
        out = cache.attention(q, table, ints([20, 20]))
        assert out[0].isnan().all() and not out[1].isnan().any()
        assert not cache.attention(q, table, ints([16, 20])).isnan().any()
    cache.k_scale[1] = 0.0  # a page of equal scores
    check_attention(cache, q, table, [20, 20], [1, 1], True)
    check_attention(cache, q, table, [20, 20], [1, 1], True, scale=-0.3)


def test_bad_v_scales_make_their_rows_nan():
    cache = filled(4, 1, 16, 64, seed=27)
    table = ints([[0, 1], [2, 3]])
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(28)).cuda()
    for bad in (0.0, -1.0, NAN, math.inf, 2.0 ** 49):
        cache.v_scale[1] = bad
        out = cache.attention(q, table, ints([20, 20]))
        assert out[0].isnan().all() and not out[1].isnan().any()
        assert not cache.attention(q, table, ints([16, 20])).isnan().any()


# -------------------------------------------- rows, pages and lengths that do not fit
def test_what_a_table_holds_behind_a_length_is_not_used():
    cache = filled(40, 2, 16, 64, seed=56)
    lens = [20, 0, 33, 300]
    table = tables(lens, 16, 40, seed=57, width=70)
    need = torch.tensor([-(-t // 16) for t in lens], device='cuda')
    wild = torch.where(torch.arange(70, device='cuda') < need[:, None], table, -(1 << 30)).to(torch.int32)
    q = torch.randn(4, 4, 64, device='cuda')
    out, _ = check_attention(cache, q, table, lens, [1] * 4, True)
    assert torch.equal(cache.attention(q, wild, ints(lens)), out)
    assert torch.equal(cache.attention(q, wild[:, :19], ints(lens)), cache.attention(q, table[:, :19], ints(lens)))
    x = torch.randn(3, 2, 64, device='cuda')
    cache.write(x, x, wild[[0, 2, 3]], ints([20, 33, 300]))
    cache.read(3, wild[[0, 2, 3]], ints([20, 33, 300]))
    cache.check()


def test_rows_of_no_sequence_stay():
    cache = filled(8, 2, 16, 64, seed=29)
    table = tables([20, 30], 16, 8, seed=30)
    starts = ints([2, 5, 9])
    q = torch.randn(12, 4, 64, device='cuda')
    for width in (2, 400):  # one block a row tile, and split ones
        wide = torch.zeros(2, width, dtype=torch.int32, device='cuda')
        wide[:, :2] = table
        out = torch.full_like(q, 7.0)
        got = cache.attention(q, wide, ints([20, 30]), starts=starts, out=out)
        assert got is out and (out[:2] == 7).all() and (out[9:] == 7).all()
        want = plain_attention(q[2:9], cache, table.tolist(), [20, 30], [3, 4], True)
        assert ((out[2:9].double() - want[0]).abs() <= want[2]).all()
    k, v = (torch.full((12, 2, 64), 7.0, device='cuda') for _ in range(2))
    cache.read(12, table, ints([20, 30]), starts=starts, out=(k, v))
    assert (k[:2] == 7).all() and (k[9:] == 7).all() and (v[9:] == 7).all()
    assert torch.equal(k[2:5].double(), gather(cache.k, cache.k_scale, table[0].tolist(), 20)[17:])
    cache.check()


@pytest.mark.parametrize('fault', ['page low', 'page high', 'long', 'negative', 'too many rows', 'starts order',
                                   'starts beyond', 'starts negative'])
def test_what_does_not_fit_is_left_out_and_reported(fault):
    from rapidtinyrec_b200._native import NativeError
    cache = filled(8, 2, 16, 64, seed=31)
    table, lens, starts = ints([[0, 1], [2, 3], [4, 5]]), ints([20, 25, 32]), ints([0, 2, 4, 6])
    if fault == 'page low':
        table[1, 1] = -1
    elif fault == 'page high':
        table[1, 1] = 8
    elif fault == 'long':
        lens[1] = 33
    elif fault == 'negative':
        lens[1] = -1
    elif fault == 'too many rows':
        lens[1] = 1
    elif fault == 'starts order':
        starts[2] = 1
    elif fault == 'starts beyond':
        starts[3] = 7
    elif fault == 'starts negative':
        starts[0] = -1
    x = torch.randn(6, 2, 64, device='cuda')
    q = torch.randn(6, 4, 64, device='cuda')
    guard = cache.k.view(torch.uint8).clone()
    scales = cache.k_scale.clone()
    cache.write(x, x, table, lens, starts=starts)
    with pytest.raises(NativeError):
        cache.check()
    assert torch.equal(cache.k.view(torch.uint8)[6:], guard[6:]) and torch.equal(cache.k_scale[6:], scales[6:])
    if not fault.startswith('starts'):
        assert torch.equal(cache.k.view(torch.uint8)[3], guard[3])
    cache.read(6, table, lens, starts=starts)
    with pytest.raises(NativeError):
        cache.check()
    out = cache.attention(q, table, lens, starts=starts)
    if fault == 'too many rows':  # attention allows it: the rows before the sequence see nothing
        cache.check()
        assert (out[2] == 0).all() and not out[3].isnan().any()
    else:
        with pytest.raises(NativeError):
            cache.check()
        if not fault.startswith('starts'):
            assert out[2:4].isnan().all()
    if not fault.startswith('starts'):
        want = plain_attention(q[4:], cache, [[4, 5]], [32], [2], True)
        assert ((out[4:].double() - want[0]).abs() <= want[2]).all()


@pytest.mark.parametrize('starts,rows', [([0, 300, 100, 400], 400), ([5000, 5002, 5004, 5006], 10),
                                         ([0, 4, 400, 100], 400), ([0, 100, 200, 401], 400), ([-1, 100, 200, 400], 400),
                                         ([400, 300, 200, 100], 400), ([0, -(1 << 31), (1 << 31) - 1, 400], 400)])
@pytest.mark.parametrize('width', [25, 600])
def test_starts_that_do_not_fit_leave_out_the_whole_call(starts, rows, width):
    """Also where no work item, or more than one, would match a sequence; tables so wide that stretches
    are joined by a kernel."""
    from rapidtinyrec_b200._native import NativeError
    cache = filled(80, 2, 16, 128, seed=83)
    table = tables([400, 400, 400], 16, 80, seed=84, width=width)
    lens, bad = ints([400, 400, 400]), ints(starts)
    x = torch.randn(rows, 2, 128, device='cuda')
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    calls = [lambda: cache.write(x, x, table, lens, starts=bad)]
    outs = []
    for dtype in DTYPES:
        for heads in (2, 8, 64):
            q = torch.randn(rows, heads, 128, device='cuda').to(dtype)
            outs.append(torch.full_like(q, 7.0))
            calls.append(lambda q=q, out=outs[-1]: cache.attention(q, table, lens, starts=bad, out=out))
    outs += [torch.full_like(x, 7.0), torch.full_like(x, 7.0)]
    calls.append(lambda: cache.read(rows, table, lens, starts=bad, out=outs[-2:]))
    for call in calls:
        call()
        with pytest.raises(NativeError, match='row range'):
            cache.check()
    assert all((out == 7).all() for out in outs)
    for t, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        assert torch.equal(t.view(torch.uint8), was)
    # the next call, with starts that fit
    q = torch.randn(9, 8, 128, device='cuda')
    check_attention(cache, q, table, [400] * 3, [4, 0, 5], True, starts=ints([0, 4, 4, 9]))


def test_python_refuses_what_the_kernels_cannot_take():
    cache = filled(4, 2, 16, 64, seed=32)
    q, x = torch.randn(2, 4, 64, device='cuda'), torch.randn(2, 2, 64, device='cuda')
    table, lens = ints([[0], [1]]), ints([4, 4])
    for call in (lambda: cache.attention(q[:, :3], table, lens), lambda: cache.attention(q.half(), table, lens),
                 lambda: cache.attention(q.cpu(), table, lens), lambda: cache.attention(q[..., :32], table, lens),
                 lambda: cache.attention(q, table.long(), lens), lambda: cache.attention(q, table, lens[:1]),
                 lambda: cache.attention(q, table, lens.cpu()), lambda: cache.attention(q, table, lens, starts=ints([0, 2])),
                 lambda: cache.attention(q, table, lens, starts=cuts([1, 1]).cpu()),
                 lambda: cache.attention(q[:1].expand(3, 4, 64), table, lens), lambda: cache.attention(q, table, lens, out=q[:1]),
                 lambda: cache.write(x, x.bfloat16(), table, lens), lambda: cache.write(x, x[:1], table, lens),
                 lambda: cache.write(x[:, :1], x[:, :1], table, lens), lambda: cache.read(2, table, lens, dtype=torch.half),
                 lambda: cache.read(2, table, lens, out=(x, x[:, :1])), lambda: cache.heads(1, 2),
                 lambda: cache.read(3, table, lens)):
        with pytest.raises(ValueError):
            call()
    assert cache.attention(q[:0], table, lens).shape == (0, 4, 64)
    cache.write(x[:0], x[:0], table, lens)
    assert cache.read(0, table[:0], lens[:0])[0].shape == (0, 2, 64)
    cache.check()


def test_outputs_that_memory_cannot_hold():
    """The allocator's error comes as torch raises it, and the cache serves on."""
    cache = filled(4, 2, 16, 64, seed=91)
    with pytest.raises(torch.OutOfMemoryError):
        cache.read(1 << 30, ints([[0]]), ints([4]))  # 512 GiB each
    check_attention(cache, torch.randn(1, 4, 64, device='cuda'), ints([[1]]), [9], [1], True)


def test_one_tensor_is_not_both_outputs():
    cache = filled(4, 2, 16, 64, seed=92)
    x = torch.full((4, 2, 64), 7.0, device='cuda')
    with pytest.raises(ValueError, match='twice'):
        cache.read(4, ints([[0]]), ints([9]), out=(x, x))
    assert (x == 7).all()
    both = torch.empty(4, 2, 2, 64, device='cuda')  # side by side is fine
    k, v = cache.read(4, ints([[0]]), ints([9]), out=(both[:, 0], both[:, 1]))
    want = cache.read(4, ints([[0]]), ints([9]))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize('dtype,heads,kv,dim,rows,tokens', OUTWEIGHED)
def test_the_output_may_be_q(dtype, heads, kv, dim, rows, tokens):
    page = 32
    pages = -(-tokens // page)
    cache = filled(pages, kv, page, dim, seed=93)
    table = tables([tokens], page, pages, seed=94)
    q = torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(95)).to(dtype).cuda()
    for causal in (True, False):
        want, want_lse = cache.attention(q, table, ints([tokens]), causal=causal, return_lse=True)
        own = q.clone()
        out, lse = cache.attention(own, table, ints([tokens]), causal=causal, return_lse=True, out=own)
        assert out is own and torch.equal(own, want) and torch.equal(lse, want_lse)


def test_an_output_that_overlaps_q_is_refused():
    cache = filled(4, 2, 16, 64, seed=96)
    table, lens = ints([[0]]), ints([9])
    room = torch.randn(20, 4, 64, device='cuda')
    for q, out in ((room[:8], room[1:9]), (room[1:9], room[:8]), (room[::2][:8], room[:8]), (room[::2][:8], room[7:15]),
                   (room[:4].view(2, 8, 64)[:, :4], room[2:4]), (room[:1].expand(3, 4, 64), room[:3])):
        before = room.clone()
        with pytest.raises(ValueError, match='apart'):
            cache.attention(q, table, lens, out=out)
        assert torch.equal(room, before)
    for q, out in ((room[:8], room[8:16]), (room[8:16], room[:8]), (room.view(2, 40, 64)[:, :4], room[2:4]),
                   (room[:8:4], room[12:14])):
        want = cache.attention(q, table, lens)
        assert torch.equal(cache.attention(q, table, lens, out=out), want)


# -------------------------------------------------------- streams and graphs
def test_other_streams_and_captured_graphs():
    """Calls on a side stream; two graphs over one cache, replayed with other inputs."""
    cache = filled(40, 2, 64, 128, seed=33)
    table = tables([2400], 64, 40, seed=34)
    lens, g = ints([2000]), torch.Generator().manual_seed(35)
    q = torch.randn(3, 12, 128, generator=g).cuda()
    x = torch.randn(1, 2, 128, generator=g).bfloat16().cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = cache.attention(q, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(beside, cache.attention(q, table, lens))
    graphs, outs = [], []
    for rows in (3, 1):  # split over blocks: each graph has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.write(x, x, table, lens)
            outs.append(cache.attention(q[:rows], table, lens))
        graphs.append(graph)
    for t in (2001, 2002, 700):
        lens.fill_(t)
        q.copy_(torch.randn(3, 12, 128, generator=g))
        x.copy_(torch.randn(1, 2, 128, generator=g))
        for graph in graphs:
            graph.replay()
        for rows, out in zip((3, 1), outs):
            want = plain_attention(q[:rows], cache, table.tolist(), [t], [rows], True)
            assert ((out.double() - want[0]).abs() <= want[2]).all(), t
        got = cache.read(1, table, lens)[0]
        assert (got - x.float()).abs().max() <= x.abs().max().item() * 2.0 ** -4
    cache.check()


def test_check_waits_for_calls_on_other_streams():
    from rapidtinyrec_b200._native import NativeError
    cache = filled(4, 2, 16, 64, seed=90)
    q, lens = torch.randn(1, 4, 64, device='cuda'), ints([20])
    tables_ = ints([[0, 1]]), ints([[0, 4]])
    cache.attention(q, tables_[0], lens)
    cache.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # cycles, some 50 ms
        cache.attention(q, tables_[1], lens)
    with pytest.raises(NativeError, match='page'):
        cache.check()
    cache.check()


def test_calls_on_two_streams_at_once():
    cache = filled(80, 2, 64, 128, seed=36)
    table = tables([5000], 64, 80, seed=37)
    lens = ints([5000])
    qs = [torch.randn(2, 12, 128, device='cuda') for _ in range(2)]
    want = [cache.attention(q, table, lens) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attention(qs[i], table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_results_repeat_bit_for_bit():
    cache = filled(80, 4, 64, 128, seed=38)
    table = tables([5000], 64, 80, seed=39)
    q = torch.randn(300, 28, 128, device='cuda')
    a = cache.attention(q, table, ints([5000]))
    for _ in range(3):
        assert torch.equal(a, cache.attention(q, table, ints([5000])))


# ----------------------------------------------------------------- far offsets
def test_offsets_beyond_32_bits():
    """A cache of 4.6 GB of codes for each of K and V, used in its last pages."""
    from rapidtinyrec_b200.kv_cache import KvCache8
    pages, kv, page, dim = 70000, 4, 128, 128
    code = [torch.empty(pages, kv, page, dim, dtype=torch.uint8, device='cuda').view(F8) for _ in range(2)]
    scale = [torch.ones(pages, kv, device='cuda') for _ in range(2)]
    big = KvCache8(*code, *scale)
    small = KvCache8.allocate(3, kv, page, dim)
    far, near = ints([[pages - 1, 3, pages - 2]]), ints([[0, 1, 2]])
    x = torch.randn(300, kv, dim, device='cuda')
    big.write(x, x, far, ints([300]))
    small.write(x, x, near, ints([300]))
    for a, b in zip(big.read(300, far, ints([300])), small.read(300, near, ints([300]))):
        assert torch.equal(a, b)
    q = torch.randn(300, 8, dim, device='cuda')
    assert torch.equal(big.attention(q, far, ints([300])), small.attention(q, near, ints([300])))
    big.check()


# ---------------------------------------------------------------- all together
@pytest.mark.parametrize('dtype', DTYPES)
def test_prompts_then_tokens_as_a_server_runs_them(dtype):
    """Prompts of three users written and attended, then tokens one at a time: each step writes,
    attends and agrees with float64 attention over what the cache reads back; and with attention
    over the exact K and V within what 4-bit mantissas can hold."""
    page, heads, kv, dim = 32, 12, 2, 128
    g = torch.Generator().manual_seed(40)
    prompts, steps = [70, 1, 33], 9
    cache = filled(20, kv, page, dim, seed=41)
    table = tables([t + steps for t in prompts], page, 20, seed=42)
    make = lambda n, h: torch.randn(n, h, dim, generator=g).to(dtype).cuda()  # noqa: E731
    k, v, q = make(sum(prompts), kv), make(sum(prompts), kv), make(sum(prompts), heads)
    held = [list(t) for t in (k.split(prompts), v.split(prompts))]
    cache.write(k, v, table, ints(prompts), starts=cuts(prompts))
    check_attention(cache, q, table, prompts, prompts, True, starts=cuts(prompts))
    for step in range(1, steps + 1):
        k, v, q = make(3, kv), make(3, kv), make(3, heads)
        for part, x in zip(held, (k, v)):
            for b in range(3):
                part[b] = torch.cat([part[b], x[b:b + 1]])
        lens = [t + step for t in prompts]
        cache.write(k, v, table, ints(lens))
        out, _ = check_attention(cache, q, table, lens, [1] * 3, True)
        for b in range(3):
            kk, vv = (part[b].double().repeat_interleave(heads // kv, 1) for part in held)
            p = torch.softmax(torch.einsum('hd,thd->ht', q[b].double(), kk) / math.sqrt(dim), -1)
            full = torch.einsum('ht,thd->hd', p, vv)
            # rounding K by 2^-4 relative at most moves a score by 2^-4 sum |q| |k|; its typical
            # size is 2^-4 / sqrt(3) sqrt(sum q^2 k^2): a loose check that the pages are the right ones
            assert (out[b].double() - full).norm() / full.norm() < 0.25
    back = cache.read(sum(lens), table, ints(lens), starts=cuts(lens))
    want = torch.cat([t for t in held[0]]).float()
    assert ((back[0] - want).abs() <= want.abs() * 2.0 ** -4 + want.abs().max() * 2.0 ** -13).all()
    cache.check()
