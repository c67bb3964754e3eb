"""The 8-bit KV cache operators: what is measured, and their plain forms.

The cache holds e4m3 codes in pages, ``[pages, kv_heads, page, head_dim]``, with
one float32 scale for each page and head; a sequence finds its pages through a row
of a page table.  Three operators work on it:

* ``write``: new K and V rows are quantised into the pages of their sequences;
* ``read``: rows of the cache are read back as the values they stand for;
* ``attention``: softmax attention of new query rows over cached sequences.

Sequence ``b`` holds ``lens[b]`` tokens.  Row ``r`` of the new rows belongs to the
sequence with ``starts[b] <= r < starts[b + 1]`` (equal shares where ``starts`` is
None), and a sequence's n rows are its last n positions, or, in attention that is
not causal, rows beside the sequence that each see all of it.

Formulas, with c the code and s the scale of its page and head:

* the value of a code is ``c * s``;
* a page's scale is the least power of two, from 2^-48 to 2^48, at which the largest
  magnitude written to the page is at most 448; where the page holds older tokens of
  the sequence it is no less than the scale it had, and their codes are rounded again
  where it grew.  ``c = e4m3(x / s)``, to nearest even; NaN, infinities and magnitudes
  above 448 * 2^48 are NaN;
* ``out = sum_j p_j v_j`` with ``p = softmax_j(scale * q . k_j)`` over the visible j,
  and ``lse = log sum_j exp(scale * q . k_j)``; a row that sees nothing is 0, its lse
  minus infinity.

``run`` computes them in elementary torch operations, or, where ``own`` is true, by the
package's kernels.
"""
import math

import torch

own = False

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
CODE = torch.float8_e4m3fn
LARGEST = 448.0
LOW, HIGH = -48, 48


# ------------------------------------------------------------------- cases
def _case(name, op, dtype, heads, kv_heads, dim, page, seqs, old, new, causal=True, lse=False):
    return {'name': name, 'op': op, 'dtype': dtype, 'heads': heads, 'kv_heads': kv_heads, 'dim': dim, 'page': page,
            'seqs': seqs, 'old_lo': old[0], 'old_hi': old[1], 'new_lo': new[0], 'new_hi': new[1],
            'causal': causal, 'lse': lse}


def listed():
    return [
        # one user, one new token over a prompt of the 1.5B workload: latency counts
        _case('attn-token-1.5b', 'attention', 'fp32', 12, 2, 128, 64, 1, (237, 237), (1, 1)),
        # the 50 beams of one user over the shared prompt, for a merge with the beams' own tokens
        _case('attn-beams-7b', 'attention', 'bf16', 28, 4, 128, 64, 1, (719, 719), (50, 50), causal=False, lse=True),
        # a batch of users of different prompt lengths, one token each
        _case('attn-batch-0.5b', 'attention', 'fp32', 14, 2, 64, 16, 61, (30, 300), (1, 1)),
        # a large batch over long histories: bandwidth
        _case('attn-long-7b', 'attention', 'bf16', 28, 4, 128, 64, 24, (6000, 32001), (1, 1)),
        # one sequence of 128 Ki tokens: all of the GPU on one row
        _case('attn-one-128k-1.5b', 'attention', 'bf16', 12, 2, 128, 128, 1, (131071, 131071), (1, 1)),
        # histories that grew by some items since they were cached, fp32
        _case('attn-extend-1.5b', 'attention', 'fp32', 12, 2, 128, 32, 7, (90, 350), (3, 61)),
        # a long prompt's next chunk over what is cached: arithmetic
        _case('attn-chunk-7b', 'attention', 'bf16', 28, 4, 128, 128, 2, (4096, 6001), (700, 1024)),
        # one decode step's K and V of a batch
        _case('write-token-7b', 'write', 'bf16', 28, 4, 128, 16, 64, (600, 1024), (1, 1)),
        # the prompt of one user, every layer's heads at once (28 layers x 2 heads)
        _case('write-prompt-1.5b', 'write', 'fp32', 12, 56, 128, 64, 1, (0, 0), (350, 350)),
        # many prompts, some of them continued inside a page
        _case('write-prompts-7b', 'write', 'bf16', 28, 4, 128, 32, 96, (0, 200), (600, 2047)),
        # a short history read back
        _case('read-prompt-0.5b', 'read', 'fp32', 14, 2, 64, 16, 3, (100, 300), (100, 300)),
        # many histories read back
        _case('read-prompts-7b', 'read', 'bf16', 28, 4, 128, 64, 40, (1, 900), (2000, 4001)),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'attention', 'write', 'read'])
    dtype = rng.choice(['fp32', 'bf16'])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.randint(1, 8)
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    if op != 'attention':
        seqs = _log_int(rng, 1, 96)
        most = max(1, min(4096, (64 << 20) // (seqs * kv * dim)))  # tokens a sequence, for at most 64 Mi values
        new = _log_int(rng, 1, most)
        old = rng.choice([0, _log_int(rng, 1, most)])
        return _case('', op, dtype, kv * group, kv, dim, page, seqs, (rng.randint(old // 3, old), old),
                     (max(1, new // rng.randint(1, 3)), new))
    kind = rng.choice(['token', 'rows', 'chunk'])
    causal = kind != 'rows'
    seqs = _log_int(rng, 1, {'token': 128, 'rows': 8, 'chunk': 8}[kind])
    most = {'token': min(131072, (96 << 20) // (seqs * kv * dim)), 'rows': 2000, 'chunk': 8192}[kind]
    old = _log_int(rng, 1, most)
    new = 1 if kind == 'token' else _log_int(rng, 2, 64 if kind == 'rows' else 1024)
    cap = (6 << 30) // (seqs * kv * group * dim)  # pairs of one head
    new = max(1, min(new, cap // (old + new)))
    lo = new if kind != 'chunk' else max(1, new // rng.randint(1, 4))
    return _case('', op, dtype, kv * group, kv, dim, page, seqs, (max(1, old // rng.choice([1, 2, 8])), old), (lo, new),
                 causal=causal, lse=kind == 'rows')


def _spread(lo, hi, count, step):
    """count lengths from lo to hi, the first of them hi."""
    return [hi - int(round((hi - lo) * ((b * step) % 1.0))) for b in range(count)]


def _lengths(case):
    """Tokens that each sequence holds before its new rows, and its new rows."""
    old = _spread(case['old_lo'], case['old_hi'], case['seqs'], 0.6180339887)
    new = _spread(case['new_lo'], case['new_hi'], case['seqs'], 0.7548776662)
    return old, new


def _totals(case):
    """Tokens that each sequence holds with its new rows (attention that is not causal: without them)."""
    old, new = _lengths(case)
    return [a + b if case['causal'] else a for a, b in zip(old, new)]


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    old, new = _lengths(case)
    total = _totals(case)
    heads, kv, dim, page = case['heads'], case['kv_heads'], case['dim'], case['page']
    rows = sum(new)
    if case['op'] == 'write':
        pages = sum(-(-(a + b) // page) - a // page for a, b in zip(old, new))
        return {'bytes': 2 * kv * (rows * dim * (size + 1) + pages * 4), 'flops': 4 * rows * kv * dim}
    if case['op'] == 'read':
        pages = sum(-(-(a + b) // page) - a // page for a, b in zip(old, new))
        return {'bytes': 2 * kv * (rows * dim * (size + 1) + pages * 4), 'flops': 2 * rows * kv * dim}
    pairs = sum(n * t - (n * (n - 1) // 2 if case['causal'] else 0) for n, t in zip(new, total))
    cached = 2 * kv * (sum(total) * dim + sum(-(-t // page) for t in total) * 4)
    return {'bytes': cached + rows * heads * (2 * dim * size + (4 if case['lse'] else 0)), 'flops': 4 * pairs * heads * dim}


# ------------------------------------------------------------------ inputs
def _encode(x):
    """Pages of float32 values as codes and scales."""
    scale = _least_scale(x.abs().amax((-1, -2)))
    return (x / scale[..., None, None]).to(CODE), scale


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dev, dtype = 'cuda', TYPES[case['dtype']]
    heads, kv, dim, page = case['heads'], case['kv_heads'], case['dim'], case['page']
    old, new = _lengths(case)
    total = _totals(case)
    rows = sum(new)
    used = [-(-t // page) for t in total]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(total), max(used), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n

    def values(*shape, gain):
        return torch.randn(*shape, generator=g, device=dev) * gain

    # some channels of K are much larger than the others, as rotary models have them
    channel = torch.ones(dim, device=dev)
    channel[dim // 4::dim // 2] = 5.0
    state = {'case': case, 'table': table, 'lens': torch.tensor(total, dtype=torch.int32, device=dev), 'rows': rows,
             'most': max(new), 'starts': None}
    if len(set(new)) > 1:
        cuts = [0]
        for n in new:
            cuts.append(cuts[-1] + n)
        state['starts'] = torch.tensor(cuts, dtype=torch.int32, device=dev)
    spread = torch.exp(0.5 * torch.randn(pages, kv, 1, 1, generator=g, device=dev))
    state['k'], state['k_scale'] = _encode(values(pages, kv, page, dim, gain=channel * spread))
    state['v'], state['v_scale'] = _encode(values(pages, kv, page, dim, gain=spread))
    if case['op'] != 'read':
        # the rows of a fused projection: q, k and v side by side
        own_kv = kv if case['op'] == 'write' else 0
        both = values(rows, (heads if case['op'] == 'attention' else 0) + 2 * own_kv, dim, gain=1.0).to(dtype)
        if case['op'] == 'attention':
            state['q'] = both
        else:
            state['new_k'] = both[:, :kv].mul_(channel.to(dtype))
            state['new_v'] = both[:, kv:]
    return state


# ------------------------------------------------------------- plain forms
def _least_scale(amax):
    """The least power of two, from 2^LOW to 2^HIGH, at which amax is at most 448 (= 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    x = torch.where(m <= LARGEST / 512, e - 9, e - 8).clamp(LOW, HIGH)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, x, LOW))


def _rows(state):
    """For each new row its sequence and its place among the sequence's new rows, and each sequence's count."""
    lens, rows = state['lens'], state['rows']
    each = torch.arange(rows, device=lens.device)
    if state['starts'] is None:
        n = rows // lens.numel()
        return each // n, each % n, torch.full_like(lens, n)
    starts = state['starts']
    seq = torch.searchsorted(starts[1:], each, right=True)
    return seq, each - starts[seq], starts[1:] - starts[:-1]


def _plain_write(state):
    page, lens, table = state['case']['page'], state['lens'], state['table']
    seq, _, count = _rows(state)
    first = torch.cumsum(count, 0) - count
    begin = lens - count
    slots = (state['most'] + page - 2) // page + 1
    nth = (begin // page)[:, None] + torch.arange(slots, device=lens.device)  # [seqs, slots]
    valid = nth * page < lens[:, None]
    pid = table.gather(1, nth.clamp(max=table.shape[1] - 1).long())
    pos = nth[:, :, None] * page + torch.arange(page, device=lens.device)  # [seqs, slots, page]
    fresh = (pos >= begin[:, None, None]) & (pos < lens[:, None, None])
    row = (first[:, None, None] + pos - begin[:, None, None]).clamp(0, state['rows'] - 1)
    kept = pos < begin[:, None, None]
    pid, pick = pid[valid].long(), (row[valid], fresh[valid], kept[valid])
    for code, scale, new in ((state['k'], state['k_scale'], state['new_k']), (state['v'], state['v_scale'], state['new_v'])):
        row_, fresh_, kept_ = pick
        x = new[row_].float().transpose(1, 2)  # [pages, heads, page, dim]
        x = torch.where(x.abs() <= LARGEST * 2.0 ** HIGH, x, torch.nan)
        size = torch.where(fresh_[:, None, :, None], x.abs().nan_to_num(0.0), 0.0).amax((-1, -2))
        had = scale[pid]
        some = kept_[:, :1]
        now = torch.where(some, torch.maximum(had, _least_scale(size)), _least_scale(size))
        was = code[pid]
        again = (was.float() * had[..., None, None] / now[..., None, None]).to(CODE)
        again = torch.where((now > had)[..., None, None], again.view(torch.uint8), was.view(torch.uint8))
        put = torch.where(fresh_[:, None, :, None], (x / now[..., None, None]).to(CODE).view(torch.uint8),
                          torch.where(kept_[:, None, :, None], again, was.view(torch.uint8)))
        code.view(torch.uint8)[pid] = put
        scale[pid] = now
    return {'k': state['k'], 'v': state['v'], 'k_scale': state['k_scale'], 'v_scale': state['v_scale']}


def _plain_read(state):
    page, lens = state['case']['page'], state['lens']
    seq, place, count = _rows(state)
    pos = lens[seq] - count[seq] + place
    pid = state['table'][seq, pos // page].long()
    dtype = TYPES[state['case']['dtype']]
    return {'k': (state['k'][pid, :, pos % page].float() * state['k_scale'][pid][..., None]).to(dtype),
            'v': (state['v'][pid, :, pos % page].float() * state['v_scale'][pid][..., None]).to(dtype)}


def _dense(code, scale, table):
    """The pages of a table's rows as [seqs, heads, tokens, dim]."""
    t = table.long()
    x = code[t].float().mul_(scale[t][..., None, None])  # [seqs, slots, heads, page, dim]
    return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _plain_attention(state):
    case, lens = state['case'], state['lens']
    kv, dim, group = case['kv_heads'], case['dim'], case['heads'] // case['kv_heads']
    seq, place, count = _rows(state)
    n, seqs = state['most'], lens.numel()
    k = _dense(state['k'], state['k_scale'], state['table'])
    v = _dense(state['v'], state['v_scale'], state['table'])
    tokens = k.shape[2]
    q = torch.zeros(seqs, n, case['heads'], dim, device=k.device)
    q[seq, place] = state['q'].float()
    q = q.view(seqs, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * n, dim)
    s = torch.matmul(q, k.transpose(2, 3)).view(seqs, kv, group, n, tokens).mul_(1 / math.sqrt(dim))
    last = lens[:, None] - (count[:, None] - 1 - torch.arange(n, device=k.device) if case['causal'] else 0)
    seen = torch.arange(tokens, device=k.device) < last[:, :, None]  # [seqs, n, tokens]
    s.masked_fill_(~seen[:, None, None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    sums = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, kv, group * n, tokens), v).view(seqs, kv, group, n, dim)
    o = o / torch.where(sums > 0, sums, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, n, case['heads'], dim)[seq, place].to(TYPES[case['dtype']])
    if not case['lse']:
        return {'out': o}
    lse = (top + torch.log(sums)).view(seqs, kv, group, n).permute(0, 3, 1, 2).reshape(seqs, n, case['heads'])
    return {'out': o, 'lse': lse[seq, place]}


def run(state):
    case = state['case']
    if not own:
        return {'write': _plain_write, 'read': _plain_read, 'attention': _plain_attention}[case['op']](state)
    cache = state.get('cache')
    if cache is None:  # the handle that a program makes once for its cache
        from rapidtinyrec_b200.kv_cache import KvCache8
        cache = state['cache'] = KvCache8(state['k'], state['v'], state['k_scale'], state['v_scale'])
    if case['op'] == 'write':
        cache.write(state['new_k'], state['new_v'], state['table'], state['lens'], starts=state['starts'])
        return {'k': state['k'], 'v': state['v'], 'k_scale': state['k_scale'], 'v_scale': state['v_scale']}
    if case['op'] == 'read':
        k, v = cache.read(state['rows'], state['table'], state['lens'], starts=state['starts'], dtype=TYPES[case['dtype']])
        return {'k': k, 'v': v}
    got = cache.attention(state['q'], state['table'], state['lens'], starts=state['starts'], causal=case['causal'],
                          return_lse=case['lse'])
    return {'out': got[0], 'lse': got[1]} if case['lse'] else {'out': got}


# -------------------------------------------------------------- in 64 bits
def _grid(x):
    """float64 values of at most 448 rounded to the nearest e4m3 value (ties to even)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    page, dim, heads, kv = case['page'], case['dim'], case['heads'], case['kv_heads']
    old, new = _lengths(case)
    table, cuts = state['table'].tolist(), [0]
    for n in new:
        cuts.append(cuts[-1] + n)
    if case['op'] == 'write':
        out = {}
        for name in ('k', 'v'):
            code, scale, x = state[name].double(), state[name + '_scale'].double(), state['new_' + name].double()
            for b, (a, n) in enumerate(zip(old, new)):
                for j in range(a // page, -(-(a + n) // page)):
                    p, lo, hi = table[b][j], max(a, j * page), min(a + n, (j + 1) * page)
                    rows = x[cuts[b] + lo - a:cuts[b] + hi - a].transpose(0, 1)  # [heads, tokens, dim]
                    size = rows.abs().amax((1, 2))
                    need = torch.exp2(torch.ceil(torch.log2((size / LARGEST).clamp(min=2.0 ** LOW))).clamp(LOW, HIGH))
                    need = torch.where(need * LARGEST < size, 2 * need, need)  # where the logarithm was a little off
                    need = torch.where((need * LARGEST >= 2 * size) & (need > 2.0 ** LOW), need / 2, need)
                    keep = lo - j * page
                    if keep:
                        had = scale[p]
                        need = torch.maximum(need, had)
                        code[p, :, :keep] = _grid(code[p, :, :keep] * (had / need)[:, None, None])
                    scale[p] = need
                    code[p, :, keep:hi - j * page] = _grid(rows / need[:, None, None])
            out[name], out[name + '_scale'] = code, scale
        return out
    if case['op'] == 'read':
        out = {}
        for name in ('k', 'v'):
            parts = []
            for b, (a, n) in enumerate(zip(old, new)):
                ids = torch.tensor(table[b][:-(-(a + n) // page)], device='cuda')
                x = state[name][ids].double() * state[name + '_scale'][ids].double()[:, :, None, None]
                parts.append(x.transpose(1, 2).reshape(-1, kv, dim)[a:a + n])
            out[name] = torch.cat(parts)
        return out
    total = _totals(case)
    outs, lses = [], []
    for b, (n, t) in enumerate(zip(new, total)):
        ids = torch.tensor(table[b][:-(-t // page)], device='cuda')
        k, v = ((state[name][ids].double() * state[name + '_scale'][ids].double()[:, :, None, None]).transpose(1, 2)
                .reshape(-1, kv, dim)[:t] for name in ('k', 'v'))
        q = state['q'][cuts[b]:cuts[b + 1]].double().view(n, kv, heads // kv, dim)
        mask = None
        if case['causal']:
            mask = torch.arange(t, device='cuda')[None, :] > t - n + torch.arange(n, device='cuda')[:, None]
        o = torch.empty_like(q)
        lse = torch.empty(q.shape[:3], dtype=torch.float64, device='cuda')
        for h in range(kv):
            s = torch.einsum('ngd,td->ngt', q[:, h], k[:, h]) / math.sqrt(dim)
            if mask is not None:
                s.masked_fill_(mask[:, None], -torch.inf)
            lse[:, h] = torch.logsumexp(s, -1)
            o[:, h] = torch.einsum('ngt,td->ngd', torch.exp(s - lse[:, h, :, None]), v[:, h])
        outs.append(o.view(n, heads, dim))
        lses.append(lse.view(n, heads))
    return {'out': torch.cat(outs), 'lse': torch.cat(lses)} if case['lse'] else {'out': torch.cat(outs)}
