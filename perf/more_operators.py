"""The operators of decoding with beams over a paged cache: what is measured, and their plain forms.

* ``select``: from logits ``[items * n, vocab]`` and the running scores ``[items, n]`` the ``k``
  best continuations of each item, and its next beams;
* ``reorder``: the rows of the beams' states in the order of their parents, in place;
* ``pages``: pages given back and taken for sequences that shrink and grow, with the page table,
  row offsets, positions and slots of the new rows;
* ``rotary``: rotary positions applied to query and key rows.

Formulas:

* select: ``value(i, v) = logits[i, v] - log sum_u exp logits[i, u] + scores[i]`` where ``allowed``
  holds, minus infinity elsewhere; the k largest of an item's n * vocab values, equal ones in the
  order of ``i * vocab + v``.  The next beams are the first ``beams`` of them that do not end with ``eos``;
* reorder: row ``b * beams + i`` becomes what row ``b * beams + parents[b, i]`` was;
* pages: n tokens need ``ceil(n / page)`` pages.  Taking: the j-th page of a call, in the order of
  the sequences and of their pages, is ``free[count - 1 - j]``; giving back: page j of m goes to
  ``free[count + m - 1 - j]``.  Row r of sequence b stands at ``lens[b] + r - starts[b]``, and its slot is
  ``table[b, position // page] * page + position % page``;
* rotary: the pair ``(a, b)`` of frequency f becomes ``m (a cos t - b sin t, b cos t + a sin t)`` with
  ``t = position * f``; frequency i of R / 2 is ``theta^(-2 i / R)``.  ``linear`` divides it by the
  factor; ``ntk`` takes ``theta * factor^(R / (R - 2))``; ``bands`` divides what turns less than ``low`` times over
  the original length, leaves what turns more than ``high`` times and goes linearly in between.

``run`` computes them in elementary torch operations, or, where ``own`` is true, by the package's kernels.
"""
import math
import random

import torch

own = False

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}


# ------------------------------------------------------------------- cases
def _select(name, dtype, items, n, beams, vocab, allowed=False, eos=True):
    return {'name': name, 'op': 'select', 'dtype': dtype, 'items': items, 'n': n, 'beams': beams, 'vocab': vocab,
            'allowed': allowed, 'eos': eos}


def _reorder(name, dtype, items, beams, layers, kv_heads, dim, room, tokens):
    return {'name': name, 'op': 'reorder', 'dtype': dtype, 'items': items, 'beams': beams, 'layers': layers,
            'kv_heads': kv_heads, 'dim': dim, 'room': room, 'tokens': tokens}


def _pages(name, seqs, page, old, new, spare=0):
    return {'name': name, 'op': 'pages', 'seqs': seqs, 'page': page, 'old_lo': old[0], 'old_hi': old[1],
            'new_lo': new[0], 'new_hi': new[1], 'spare': spare}


def _rotary(name, dtype, seqs, old, new, heads, kv_heads, dim, part, interleaved=False, theta=1e6, scaling='none', factor=1.0,
            in_place=True, back=False):
    return {'name': name, 'op': 'rotary', 'dtype': dtype, 'seqs': seqs, 'old': old, 'new': new, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'part': part, 'interleaved': interleaved, 'theta': theta, 'scaling': scaling,
            'factor': factor, 'in_place': in_place, 'back': back}


def listed():
    return [
        # a few beams over the small test model's vocabulary: latency counts
        _select('select-tiny', 'fp32', 1, 4, 4, 8192),
        # one user's step: 50 beams over the whole vocabulary
        _select('select-1.5b', 'fp32', 1, 50, 50, 152704),
        # ten beams of sixteen requests over a smaller, odd vocabulary, each with its own list of allowed tokens
        _select('select-allowed', 'fp32', 16, 10, 10, 32003, allowed=True),
        # a batch of users: bandwidth
        _select('select-batch-7b', 'bf16', 32, 50, 50, 152832),
        # one user's own tokens of 50 beams, every layer's K and V, two of the four slots filled
        _reorder('reorder-1.5b', 'fp32', 1, 50, 28, 2, 128, 4, 2),
        # eight users' longer continuations
        _reorder('reorder-7b', 'bf16', 8, 50, 28, 4, 128, 24, 17),
        # one token more for each sequence of a batch
        _pages('pages-token', 64, 16, (600, 1024), (1, 1)),
        # the same for a large batch, as a captured step has it: more rows than there are tokens
        _pages('pages-token-many', 1900, 64, (1, 4000), (0, 1), spare=37),
        # many prompts end and as many come
        _pages('pages-prompts', 96, 32, (0, 0), (600, 2047)),
        # one token of one user
        _rotary('rotary-token-1.5b', 'fp32', 1, 237, 1, 12, 2, 128, 128),
        # a batch's tokens behind long histories: half of each head, neighbouring pairs, scaled
        _rotary('rotary-far', 'fp32', 61, 130000, 7, 14, 2, 64, 32, interleaved=True, theta=1e4, scaling='bands', factor=8.0,
                in_place=False),
        # a long prompt's chunks: bandwidth
        _rotary('rotary-chunk-7b', 'bf16', 9, 4096, 3001, 28, 4, 128, 128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['select', 'reorder', 'pages', 'rotary'])
    dtype = rng.choice(['fp32', 'bf16'])
    if op == 'select':
        n = rng.choice([1, rng.randint(2, 64), 50])
        vocab = _log_int(rng, 1000, 262144)
        items = _log_int(rng, 1, max(1, min(64, (120 << 20) // (n * vocab))))
        beams = n if n > 1 else rng.choice([1, rng.randint(2, 64)])
        return _select('', dtype, items, n, beams, vocab, allowed=rng.random() < 0.3, eos=rng.random() < 0.7)
    if op == 'reorder':
        items, beams = _log_int(rng, 1, 16), rng.choice([2, 4, 10, rng.randint(3, 64), 50])
        layers, kv, dim = rng.randint(1, 32), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        most = max(1, min(256, (96 << 20) // (items * beams * layers * 2 * kv * dim)))
        tokens = _log_int(rng, 1, most)
        return _reorder('', dtype, items, beams, layers, kv, dim, min(most, tokens + rng.randint(0, 9)), tokens)
    if op == 'pages':
        seqs, page = _log_int(rng, 1, 2048), rng.choice([16, 32, 64, 128])
        old = rng.choice([0, _log_int(rng, 1, 4096)])
        new = rng.choice([1, _log_int(rng, 1, max(1, min(4096, 150000 // seqs)))])
        return _pages('', seqs, page, (rng.randint(0, old), old), (rng.randint(0, new), new), spare=rng.choice([0, rng.randint(1, 99)]))
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.randint(1, 8)
    rows = _log_int(rng, 1, min(30000, (110 << 20) // ((heads + kv) * dim)))
    seqs = rng.randint(1, min(rows, 64))
    scaling = rng.choice(['none', 'none', 'linear', 'ntk', 'bands'])
    return _rotary('', dtype, seqs, _log_int(rng, 1, 1 << 20), max(1, rows // seqs), heads, kv, dim,
                   rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5, theta=rng.choice([1e4, 1e6]), scaling=scaling,
                   factor=1.0 if scaling == 'none' else rng.choice([2.0, 4.0, 8.0]), in_place=rng.random() < 0.5,
                   back=rng.random() < 0.25)


def _spread(lo, hi, count, step):
    """count lengths from lo to hi, the first of them hi."""
    return [hi - int(round((hi - lo) * ((b * step) % 1.0))) for b in range(count)]


def _lengths(case):
    """Tokens that each sequence keeps, and its new ones."""
    return (_spread(case['old_lo'], case['old_hi'], case['seqs'], 0.6180339887),
            _spread(case['new_lo'], case['new_hi'], case['seqs'], 0.7548776662))


def _most(case):
    """Candidates of an item: twice the beams, so that enough are left without those that end."""
    return 2 * case['beams']


def work(case):
    size = 4 if case.get('dtype') == 'fp32' else 2
    if case['op'] == 'select':
        values = case['items'] * case['n'] * case['vocab']
        out = 12 * case['items'] * (_most(case) + case['beams'])
        return {'bytes': values * (size + case['allowed']) + 4 * case['items'] * case['n'] + out, 'flops': 4 * values}
    if case['op'] == 'reorder':
        row = case['layers'] * 2 * case['kv_heads'] * case['tokens'] * case['dim'] * size
        kept, moved, read = 0, 0, 0
        for parents in _parents(case):
            stay = [i for i, p in enumerate(parents) if p == i]
            kept += len(stay)
            moved += len(parents) - len(stay)
            read += len({p for i, p in enumerate(parents) if p != i})
        return {'bytes': (moved + read) * row + 4 * (kept + moved), 'flops': 0}
    if case['op'] == 'pages':
        old, new = _lengths(case)
        page, rows = case['page'], sum(new)
        taken = sum(-(-(a + n) // page) - -(-a // page) for a, n in zip(old, new))
        partial = sum(1 for a, n in zip(old, new) if a % page and n)
        return {'bytes': case['seqs'] * 24 + 4 + taken * 16 + partial * 4 + (rows + case['spare']) * 12, 'flops': 4 * rows}
    rows = case['seqs'] * case['new']
    heads = case['heads'] + case['kv_heads']
    moved = case['part'] if case['in_place'] else case['dim']
    return {'bytes': rows * heads * 2 * moved * size + 4 * rows, 'flops': 3 * rows * heads * case['part']}


# ------------------------------------------------------------------ inputs
def _parents(case):
    """The beams' parents: few of the beams have most of the children, as in a search."""
    rng = random.Random(case['items'] * 1009 + case['beams'] * 31 + case['tokens'])
    some = max(1, (2 * case['beams']) // 3)
    return [[int(some * rng.random() ** 1.5) for _ in range(case['beams'])] for _ in range(case['items'])]


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _prepare_select(case, seed):
    g, dev = _generator(seed), 'cuda'
    items, n, vocab = case['items'], case['n'], case['vocab']
    dtype = TYPES[case['dtype']]
    # tokens that are likely after anything, and what each beam adds
    usual = 1.5 * torch.randn(vocab, generator=g, device=dev)
    logits = torch.cat([(usual + 2.0 * torch.randn(n, vocab, generator=g, device=dev)).to(dtype) for _ in range(items)])
    scores = -torch.cumsum(0.2 * torch.rand(items, n, generator=g, device=dev), 1) - 6.0 * torch.rand(items, 1, generator=g, device=dev)
    allowed = None
    if n > 4:
        scores[::3, -2:] = -torch.inf  # items with fewer live beams
    if case['allowed']:
        allowed = torch.rand(items * n, vocab, generator=g, device=dev) < torch.rand(items * n, 1, generator=g, device=dev) ** 4
        allowed[n // 2::2 * n] = False  # beams that have nothing to go on with
    return {'logits': logits, 'scores': scores, 'allowed': allowed, 'end': int(usual.argmax()) if case['eos'] else None}


def _prepare_reorder(case, seed):
    g, dev, dtype = _generator(seed), 'cuda', TYPES[case['dtype']]
    rows = case['items'] * case['beams']
    shape = (2, rows, case['kv_heads'], case['room'], case['dim'])
    states = [torch.randn(shape, generator=g, device=dev, dtype=dtype) for _ in range(case['layers'])]
    # the same number of moved rows whatever the seed: beams under other numbers
    parents = torch.tensor(_parents(case), dtype=torch.int32, device=dev)
    named = torch.rand(case['items'], case['beams'], generator=g, device=dev).argsort(1)
    parents = torch.empty_like(parents).scatter_(1, named, named.gather(1, parents.long()).to(torch.int32))
    return {'states': states, 'parents': parents}


def _prepare_pages(case, seed):
    g, dev = _generator(seed), 'cuda'
    old, new = _lengths(case)
    page = case['page']
    total = [a + n for a, n in zip(old, new)]
    used = [-(-t // page) for t in total]
    pages = sum(used) + 11
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case['seqs'], max(1, max(used)) + 2), -1, dtype=torch.int32, device=dev)
    ids = torch.arange(table.shape[1], device=dev)
    table[ids < torch.tensor(used, device=dev)[:, None]] = order[:sum(used)]
    free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
    free[:pages - sum(used)] = order[sum(used):]
    as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return {'table': table, 'held': as_ints(total), 'keep': as_ints(old), 'new': as_ints(new), 'free': free,
            'count': as_ints([pages - sum(used)]), 'pages': pages, 'rows': sum(new) + case['spare']}


def _prepare_rotary(case, seed):
    g, dev, dtype = _generator(seed), 'cuda', TYPES[case['dtype']]
    rows, heads, kv, dim = case['seqs'] * case['new'], case['heads'], case['kv_heads'], case['dim']
    # the rows of a fused projection: q, k and v side by side
    fused = torch.randn(rows, heads + 2 * kv, dim, generator=g, device=dev, dtype=dtype)
    first = torch.randint(case['old'] // 2, case['old'] + 1, (case['seqs'], 1), generator=g, device=dev)
    positions = (first + torch.arange(case['new'], device=dev)).reshape(-1).to(torch.int32)
    return {'q': fused[:, :heads], 'k': fused[:, heads:heads + kv], 'positions': positions}


def prepare(case, seed):
    made = {'select': _prepare_select, 'reorder': _prepare_reorder, 'pages': _prepare_pages, 'rotary': _prepare_rotary}
    return {'case': case, **made[case['op']](case, seed)}


# ------------------------------------------------------------- plain forms
def _plain_select(state):
    case, k = state['case'], _most(state['case'])
    x = state['logits'].double()
    top = x.amax(1, keepdim=True)
    value = x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True))) + state['scores'].view(-1, 1).double()
    if state['allowed'] is not None:
        value.masked_fill_(~state['allowed'], -torch.inf)
    value = value.masked_fill_(value.isnan(), -torch.inf).view(case['items'], -1)
    least = value.topk(k, dim=1).values[:, -1:]
    above, equal = value > least, value == least
    taken = above | (equal & (equal.cumsum(1) <= k - above.sum(1, keepdim=True)))
    place = taken.nonzero()[:, 1].view(case['items'], k)
    value, order = value.gather(1, place).sort(dim=1, descending=True, stable=True)
    place = place.gather(1, order)
    found = (place % case['vocab'], place // case['vocab'], value)
    end = -1 if state['end'] is None else state['end']
    on = (found[0] == end).to(torch.uint8).sort(dim=1, stable=True).indices[:, :case['beams']]
    types = (torch.int32, torch.int32, torch.float32)
    names = ('tokens', 'parents', 'scores')
    return {**{'all_' + a: v.to(t) for a, v, t in zip(names, found, types)},
            **{a: v.gather(1, on).to(t) for a, v, t in zip(names, found, types)}}


def _plain_reorder(state):
    parents, beams = state['parents'].long(), state['case']['beams']
    rows = (parents + beams * torch.arange(parents.shape[0], device=parents.device)[:, None]).view(-1)
    parts = [s[:, :, :, :state['case']['tokens']] for s in state['states']]
    [p.copy_(p.index_select(1, rows)) for p in parts]
    return state['states']


def _page_items(before, after, page, width):
    """(sequence, place) of the pages that tokens ``before`` .. ``after`` need beyond those of ``before``."""
    nth = torch.arange(width, device=before.device)
    return ((nth >= ((before + page - 1) // page)[:, None]) & (nth < ((after + page - 1) // page)[:, None])).nonzero(as_tuple=True)


def _plain_pages(state):
    page, table, free, count, keep, new = (state['case']['page'], state['table'], state['free'], state['count'], state['keep'],
                                           state['new'])
    seq, nth = _page_items(keep, state['held'], page, table.shape[1])
    back = torch.arange(seq.numel(), device=free.device)
    free[(count + seq.numel() - 1 - back).long()] = table[seq, nth]
    count += seq.numel()
    lens = keep + new
    seq, nth = _page_items(keep, lens, page, table.shape[1])
    table[seq, nth] = free[(count - 1 - torch.arange(seq.numel(), device=free.device)).long()]
    count -= seq.numel()
    starts = torch.cat([torch.zeros_like(count), new.cumsum(0).to(torch.int32)])
    row = torch.arange(state['rows'], device=free.device)
    there = row < starts[-1]
    of = torch.searchsorted(starts[1:], row.to(torch.int32), right=True).clamp(max=new.numel() - 1)
    position = torch.where(there, keep[of] + row - starts[of], -1)
    slot = torch.where(there, table[of, position.clamp(min=0) // page].long() * page + position % page, -1)
    return {'lens': lens, 'starts': starts, 'positions': position.to(torch.int32), 'slots': slot, 'table': table,
            'count': count, 'free': free}


def _frequencies(case, dev):
    part, theta = case['part'], case['theta']
    if case['scaling'] == 'ntk':
        theta *= case['factor'] ** (part / (part - 2))
    f = theta ** (-torch.arange(0, part, 2, dtype=torch.float64, device=dev) / part)
    if case['scaling'] == 'linear':
        f = f / case['factor']
    if case['scaling'] == 'bands':
        share = ((f * (_LENGTH / (2 * math.pi)) - _LOW) / (_HIGH - _LOW)).clamp(0, 1)
        f = f * (share + (1 - share) / case['factor'])
    return f


_LENGTH, _LOW, _HIGH = 8192, 1.0, 4.0  # of the bands


def _plain_rotary(state):
    case, part = state['case'], state['case']['part']
    angle = state['positions'].double()[:, None] * _frequencies(case, state['q'].device)
    angle = -angle if case['back'] else angle
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x):
        y = x.float()
        pairs = y[..., :part].unflatten(2, (-1, 2) if case['interleaved'] else (2, -1))
        a, b = pairs.unbind(-1 if case['interleaved'] else -2)
        a, b = a * cos - b * sin, b * cos + a * sin
        y = torch.cat([torch.stack((a, b), -1 if case['interleaved'] else -2).flatten(2), y[..., part:]], -1).to(x.dtype)
        return x.copy_(y) if case['in_place'] else y

    return {'q': turned(state['q']), 'k': turned(state['k'])}


# ------------------------------------------------------- the package's calls
def _own_select(state):
    search = state.get('search')
    if search is None:  # the handle that a program makes once
        from rapidtinyrec_b200.beam_search import BeamSearch
        search = state['search'] = BeamSearch(state['case']['beams'], eos=state['end'])
    step = search.select(state['logits'], state['scores'], allowed=state['allowed'])
    return {'all_tokens': step.all_tokens, 'all_parents': step.all_parents, 'all_scores': step.all_scores,
            'tokens': step.tokens, 'parents': step.parents, 'scores': step.scores}


def _own_reorder(state):
    search = state.get('search')
    if search is None:
        from rapidtinyrec_b200.beam_search import BeamSearch
        search = state['search'] = BeamSearch(state['case']['beams'])
    search.reorder(state['states'], state['parents'], dim=1, token_dim=3, tokens=state['case']['tokens'])
    return state['states']


def _own_pages(state):
    pool = state.get('pool')
    if pool is None:
        from rapidtinyrec_b200.page_pool import PagePool
        held = state['count'].item()
        pool = state['pool'] = PagePool(state['pages'], state['case']['page'], free=state['free'][:held])
    pool.release(state['table'], state['held'], state['keep'])
    got = pool.grow(state['table'], state['keep'], state['new'], rows=state['rows'])
    return {'lens': got.lens, 'starts': got.starts, 'positions': got.positions, 'slots': got.slots, 'table': state['table'],
            'count': pool.count, 'free': pool.free}


def _own_rotary(state):
    case, rotary = state['case'], state.get('rotary')
    if rotary is None:
        from rapidtinyrec_b200.rotary import Rotary
        more = {'length': _LENGTH, 'low': _LOW, 'high': _HIGH} if case['scaling'] == 'bands' else {}
        rotary = state['rotary'] = Rotary(case['dim'], rotary_dim=case['part'], theta=case['theta'], interleaved=case['interleaved'],
                                          scaling=None if case['scaling'] == 'none' else case['scaling'], factor=case['factor'], **more)
    out = (state['q'], state['k']) if case['in_place'] else None
    q, k = rotary.rotate(state['q'], state['k'], state['positions'], back=case['back'], out=out)
    return {'q': q, 'k': k}


def run(state):
    calls = ({'select': _own_select, 'reorder': _own_reorder, 'pages': _own_pages, 'rotary': _own_rotary} if own else
             {'select': _plain_select, 'reorder': _plain_reorder, 'pages': _plain_pages, 'rotary': _plain_rotary})
    return calls[state['case']['op']](state)


# -------------------------------------------------------------- in 64 bits
def _exact_select(case, state):
    values = [torch.log_softmax(x.double(), 1) + y.double()[:, None] for x, y in zip(state['logits'].split(case['n']), state['scores'])]
    if state['allowed'] is not None:
        values = [torch.where(a, v, -torch.inf) for a, v in zip(state['allowed'].split(case['n']), values)]
    values = [v.flatten().sort(descending=True, stable=True) for v in values]
    places = torch.stack([v.indices[:_most(case)] for v in values])
    best = torch.stack([v.values[:_most(case)] for v in values])
    ways = [[(p % case['vocab'], p // case['vocab'], v) for p, v in zip(*row) if p % case['vocab'] != state['end']][:case['beams']]
            for row in zip(places.tolist(), best.tolist())]
    return {'all_tokens': places % case['vocab'], 'all_parents': places // case['vocab'], 'all_scores': best,
            'tokens': torch.tensor([[w[0] for w in row] for row in ways]), 'parents': torch.tensor([[w[1] for w in row] for row in ways]),
            'scores': torch.tensor([[w[2] for w in row] for row in ways], dtype=torch.float64)}


def _exact_reorder(case, state):
    beams, t = case['beams'], case['tokens']
    rows = [b * beams + p for b, parents in enumerate(state['parents'].tolist()) for p in parents]
    return [torch.cat([torch.stack([s[:, r, :, :t] for r in rows], 1), s[:, :, :, t:]], 3).double() for s in state['states']]


def _exact_pages(case, state):
    page, old = case['page'], state['keep'].tolist()
    table, free = state['table'].tolist(), state['free'][:state['count'].item()].tolist()
    held, new = state['held'].tolist(), state['new'].tolist()
    for b in reversed(range(case['seqs'])):
        for j in reversed(range(-(-old[b] // page), -(-held[b] // page))):
            free.append(table[b][j])
    starts, positions, slots = [0], [], []
    for b in range(case['seqs']):
        for j in range(-(-old[b] // page), -(-(old[b] + new[b]) // page)):
            table[b][j] = free.pop()
        for t in range(old[b], old[b] + new[b]):
            positions.append(t)
            slots.append(table[b][t // page] * page + t % page)
        starts.append(len(slots))
    more = [-1] * (state['rows'] - len(slots))
    return {'lens': torch.tensor([a + n for a, n in zip(old, new)]), 'starts': torch.tensor(starts),
            'positions': torch.tensor(positions + more), 'slots': torch.tensor(slots + more), 'table': torch.tensor(table),
            'count': torch.tensor([len(free)]), 'free': None}


def _exact_rotary(case, state):
    part, theta, factor = case['part'], case['theta'], case['factor']
    if case['scaling'] == 'ntk':
        theta = theta * factor ** (part / (part - 2))
    steps = [math.exp(-math.log(theta) * 2 * i / part) / (factor if case['scaling'] == 'linear' else 1.0) for i in range(part // 2)]
    if case['scaling'] == 'bands':
        turns = [_LENGTH * f / (2 * math.pi) for f in steps]
        steps = [f if r >= _HIGH else f / factor if r <= _LOW else ((_HIGH - r) * f / factor + (r - _LOW) * f) / (_HIGH - _LOW)
                 for f, r in zip(steps, turns)]
    angle = state['positions'].double()[:, None, None] * torch.tensor(steps, dtype=torch.float64, device='cuda')
    turn = torch.polar(torch.ones_like(angle), angle)
    turn = turn.conj() if case['back'] else turn
    out = {}
    for name in ('q', 'k'):
        x = state[name].double()
        even, odd = (x[..., 0:part:2], x[..., 1:part:2]) if case['interleaved'] else (x[..., :part // 2], x[..., part // 2:part])
        z = torch.complex(even, odd) * turn
        y = x.clone()
        if case['interleaved']:
            y[..., 0:part:2], y[..., 1:part:2] = z.real, z.imag
        else:
            y[..., :part // 2], y[..., part // 2:part] = z.real, z.imag
        out[name] = y
    return out


def exact(case, seed):
    made = {'select': _exact_select, 'reorder': _exact_reorder, 'pages': _exact_pages, 'rotary': _exact_rotary}
    return made[case['op']](case, prepare(case, seed))
