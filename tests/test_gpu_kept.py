"""Kept prefixes: a user's prefilled K and V quantised into a store of 8-bit pages, later
requests without a prefill (``BeamEngine.keep_prefix`` / ``generate_kept``).

Two independent paths read a kept prefix - decode attention over the pages, and the pages
read back into the arena for the ordinary decode attention - so they check each other; a
model whose K and V are exact in 8 bits (constant V, zero K) has to give the unkept
request's record.  fp32 scores of two kernels agree within the parity tests' 1e-4."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SCORE_TOL = 1e-4


@pytest.fixture(scope='module', autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.fail('CUDA device required for -m gpu tests')


def make_engine(tiny, weights=None, dtype='fp32', **kw):
    from rapidtinyrec_b200.constraints import GpuSidConstraintTables
    from rapidtinyrec_b200.engine import BeamEngine
    c = tiny['cfg'].with_dtype(dtype)
    tables = GpuSidConstraintTables(tiny['constraints'], c.root, c.newline, c.eos)
    return BeamEngine(c, tiny['weights'] if weights is None else weights, tables, max_prefix=128, **kw)


@pytest.fixture(scope='module')
def engine(tiny):
    e = make_engine(tiny)
    yield e
    e.close()


def prompts(tiny, n=3):
    return [u.prompt_token_ids for u in tiny['users'][:n]]


def same(a, b, tol=SCORE_TOL):
    assert a['token_ids'] == b['token_ids'] and a['beam_indices'] == b['beam_indices']
    for key in ('sequence_logp', 'transition_logp'):
        assert np.abs(np.array(a[key]) - np.array(b[key])).max() <= tol, key


def pages_for(ids, page):
    return -(-len(ids) // page)


@pytest.mark.parametrize('page', [16, 64])
def test_both_ways_of_reading_a_kept_prefix_agree(tiny, engine, page):
    store = engine.prefix_store(64, page)
    free = list(range(63, -1, -1))
    kept, first, scores = [], [], []
    for ids in prompts(tiny):
        plain = engine.generate(ids)
        record, k = engine.generate_and_keep(ids, store, [free.pop() for _ in range(pages_for(ids, page))])
        assert record == plain  # keeping changes nothing
        kept.append(k)
        engine.prefill(ids)
        first.append(engine.step_scores(0))
    for ids, k, want in zip(prompts(tiny), kept, first):
        over_pages = engine.generate_kept(k)
        assert torch.equal(engine.step_scores(0), want)  # step 0 comes from the same hidden state
        back = engine.generate_kept(k, in_place=False)
        assert torch.equal(engine.step_scores(0), want)
        same(over_pages, back)
        scores.append(over_pages)
    for k, want in zip(reversed(kept), reversed(scores)):  # in any order, again and again
        assert engine.generate_kept(k) == want
    ids = prompts(tiny)[0]
    assert engine.generate(ids) == engine.generate(ids)
    engine.generate_kept(kept[1])
    plain = engine.generate(ids)  # the captured graph reads the arena as before
    same(plain, engine.generate_and_keep(ids, store, [free.pop() for _ in range(pages_for(ids, page))])[0], 0)


@pytest.mark.parametrize('heads', [4, 12])
def test_a_prefix_that_is_exact_in_8_bits_gives_the_same_record(tiny, heads):
    """K = 0 and V = a bias of e4m3 values per layer and head: nothing is rounded, so a page, layer
    or head taken for another shows."""
    import dataclasses
    from rapidtinyrec_b200 import workload
    cfg = dataclasses.replace(tiny['cfg'], heads=heads)
    weights = dict(workload.synth_weights(cfg, seed=3, backend='numpy'))
    g = torch.Generator().manual_seed(5)
    for name in list(weights):
        if '.k_proj.' in name or name.endswith('v_proj.weight'):
            weights[name] = torch.zeros_like(weights[name])
        if name.endswith('v_proj.bias'):
            weights[name] = torch.randint(-7, 8, weights[name].shape, generator=g).float() / 8
    e = make_engine({**tiny, 'cfg': cfg}, weights)
    store = e.prefix_store(20, 16)
    for n, ids in enumerate(prompts(tiny, 2)):
        count = pages_for(ids, 16)
        record, kept = e.generate_and_keep(ids, store, range(n * 10, n * 10 + count))
        same(e.generate_kept(kept), record)
        same(e.generate_kept(kept, in_place=False), record)
    e.close()


@pytest.mark.parametrize('attn', ['rows', 'tc', 'folded'])
def test_kept_prefixes_beside_every_decode_attention(tiny, monkeypatch, attn):
    """fp32 sessions of the other decode attentions: over the pages all give the same record; read back
    where the kernel reads the arena, refused where it reads copies of it."""
    from rapidtinyrec_b200._native import NativeError
    ids = prompts(tiny)[2]
    monkeypatch.setenv('RTR_ATTN', attn)
    e = make_engine(tiny, max_users=2)
    store = e.prefix_store(8)
    plain = e.generate(ids)
    record, kept = e.generate_and_keep(ids, store, range(pages_for(ids, 64)))
    same(record, plain)
    over_pages = e.generate_kept(kept)
    if e.report()['decode_attention'] == 1:
        with pytest.raises(NativeError, match='in place'):
            e.generate_kept(kept, in_place=False)
    else:
        same(e.generate_kept(kept, in_place=False), over_pages)
    two = e.generate_batch([ids, prompts(tiny)[0]])
    same(two[0], plain)
    same(e.generate_kept(kept), over_pages, 0)
    same(e.generate(ids), plain, 0)
    e.close()


@pytest.mark.parametrize('attn', [None, 'rows'])
def test_a_bf16_prefix_that_is_exact_in_8_bits_gives_the_same_record(tiny, monkeypatch, attn):
    """K = 0 and V = a bias of eighths: every weight is the same, an attention's output is V times 1 +-
    2^-10 at most (weights of 11 bits, fp32 sums) before it is rounded to the bf16 that V is.  So nothing
    differs between the kept and the unkept request, whatever kernel has them."""
    from rapidtinyrec_b200 import workload
    if attn:
        monkeypatch.setenv('RTR_ATTN', attn)
    weights = dict(workload.synth_weights(tiny['cfg'], seed=3, backend='numpy'))
    g = torch.Generator().manual_seed(6)
    for name in list(weights):
        if '.k_proj.' in name or name.endswith('v_proj.weight'):
            weights[name] = torch.zeros_like(weights[name])
        if name.endswith('v_proj.bias'):
            weights[name] = torch.randint(-7, 8, weights[name].shape, generator=g).float() / 8
    e = make_engine(tiny, weights, dtype='bf16')
    store = e.prefix_store(20, 16)
    for n, ids in enumerate(prompts(tiny, 2)):
        record, kept = e.generate_and_keep(ids, store, range(n * 10, n * 10 + pages_for(ids, 16)))
        same(e.generate_kept(kept), record, 0)
        if attn:
            same(e.generate_kept(kept, in_place=False), record, 0)
    e.close()


def test_bf16_prefixes(tiny, monkeypatch):
    """bf16 sessions: their default decode attention reads copies of the arena, so only in place;
    with the per-head kernel both ways, within the differences of the framework's own bf16
    attention kernels (every operation rounds to bf16: up to 0.017 on this model; bound 0.1)."""
    from rapidtinyrec_b200._native import NativeError
    ids = prompts(tiny)[0]
    count = pages_for(ids, 64)
    e = make_engine(tiny, dtype='bf16')
    store = e.prefix_store(8)
    record, kept = e.generate_and_keep(ids, store, range(count))
    a = e.generate_kept(kept)
    if e.report()['decode_attention'] == 1:
        with pytest.raises(NativeError, match='in place'):
            e.generate_kept(kept, in_place=False)
    assert e.generate_kept(kept) == a
    assert np.abs(np.array(a['sequence_logp']) - np.array(record['sequence_logp'])).max() < 1  # the right prefix
    e.close()
    monkeypatch.setenv('RTR_ATTN', 'rows')
    e = make_engine(tiny, dtype='bf16')
    store = e.prefix_store(8)
    _, kept = e.generate_and_keep(ids, store, range(count))
    a, b = e.generate_kept(kept), e.generate_kept(kept, in_place=False)
    assert np.abs(np.array(a['sequence_logp']) - np.array(b['sequence_logp'])).max() <= 0.1
    e.close()


def test_calls_out_of_order_and_what_does_not_fit(tiny, engine):
    from rapidtinyrec_b200._native import RTR_ERR_ARG, RTR_ERR_DEVICE, RTR_ERR_STATE, NativeError
    from rapidtinyrec_b200.kv_cache import KvCache8
    ids = prompts(tiny)[0]
    count = pages_for(ids, 64)
    store = engine.prefix_store(8)
    plain = engine.generate(ids)

    def refused(code, call):
        with pytest.raises(NativeError) as e:
            call()
        assert e.value.code == code, e.value

    refused(RTR_ERR_STATE, lambda: engine.keep_prefix(ids, store, range(count)))  # after a whole request
    engine.prefill(ids)
    refused(RTR_ERR_ARG, lambda: engine.keep_prefix(ids, store, range(count - 1)))
    refused(RTR_ERR_ARG, lambda: engine.keep_prefix(ids, KvCache8.allocate(8, 2, 64, 64), range(count)))
    for bad in ([0, 0], [0, 8], [-1, 0]):
        with pytest.raises(ValueError):
            engine.keep_prefix(ids, store, bad)
    kept = engine.keep_prefix(ids, store, range(count))
    engine.decode_step(1)
    refused(RTR_ERR_STATE, lambda: engine.keep_prefix(ids, store, range(count)))
    refused(RTR_ERR_ARG, lambda: engine.generate_kept(kept._replace(table=kept.table[:count - 1])))
    refused(RTR_ERR_ARG, lambda: engine.generate_kept(kept._replace(ids=kept.ids[:2])))
    refused(RTR_ERR_DEVICE, lambda: engine.generate_kept(kept._replace(table=kept.table + 8)))
    record = engine.generate_kept(kept)
    refused(RTR_ERR_STATE, lambda: engine.keep_prefix(ids, store, range(count)))
    assert engine.generate_kept(kept) == record
    assert engine.generate(ids) == plain
    store.check()


def test_prefixes_of_another_engine(tiny, engine):
    """Another engine of the model and type takes a kept prefix; one of another type has a hidden
    state of another size and refuses it."""
    ids = prompts(tiny)[1]
    store = engine.prefix_store(8)
    record, kept = engine.generate_and_keep(ids, store, range(pages_for(ids, 64)))
    again = engine.generate_kept(kept)
    e = make_engine(tiny)
    assert e.generate_kept(kept) == again
    e.close()
    e = make_engine(tiny, dtype='bf16')
    with pytest.raises(ValueError, match='another'):
        e.generate_kept(kept)
    e.close()
    with pytest.raises(ValueError, match='another'):
        engine.generate_kept(kept._replace(hidden=kept.hidden[:-1]))
    assert engine.generate_kept(kept) == again


def test_wider_tables_give_back_what_narrower_ones_took(tiny):
    """Tables of more pages than the prompt needs, each wider than the last: the session ends up with
    the room of the widest alone; and a narrow one's launches are counted as its own."""
    ids = prompts(tiny)[0]
    n = pages_for(ids, 16)
    bytes_, launches = [], []
    for widths in ([n, n + 1, 600, 900, 1300], [1300]):
        e = make_engine(tiny)
        store = e.prefix_store(1300, 16)
        records = []
        for w in widths:
            kept = e.generate_and_keep(ids, store, range(w))[1]
            records.append(e.generate_kept(kept))
        for r in records[1:]:
            same(r, records[0])
        bytes_.append(e.report()['device_bytes'])
        before = e.report()['kernel_launches']
        e.generate_kept(kept)
        launches.append(e.report()['kernel_launches'] - before)
        kept = e.generate_and_keep(ids, store, range(n))[1]
        before = e.report()['kernel_launches']
        same(e.generate_kept(kept), records[0])
        launches.append(e.report()['kernel_launches'] - before)
        e.close()
    assert bytes_[0] == bytes_[1]
    assert launches[0] == launches[2] and launches[1] == launches[3]
    assert launches[0] - launches[1] == 4 * tiny['cfg'].layers  # the wide ones' join kernel


def test_prefixes_of_another_model_of_the_same_shapes(tiny, engine):
    """Other weights, or another rope: refused.  The same weights given on the device: taken."""
    import dataclasses
    ids = prompts(tiny)[1]
    store = engine.prefix_store(8)
    _, kept = engine.generate_and_keep(ids, store, range(pages_for(ids, 64)))
    again = engine.generate_kept(kept)
    last = sorted(n for n in tiny['weights'] if n.endswith('k_proj.weight'))[-1]
    other = dict(tiny['weights'])
    other[last] = other[last] * 1.01
    cfg = dataclasses.replace(tiny['cfg'], rope_theta=tiny['cfg'].rope_theta / 10)
    for model, weights in ((tiny, other), ({**tiny, 'cfg': cfg}, None)):
        e = make_engine(model, weights)
        for in_place in (True, False):
            with pytest.raises(ValueError, match='another'):
                e.generate_kept(kept, in_place=in_place)
        e.close()
    e = make_engine(tiny, {n: w.cuda() for n, w in tiny['weights'].items()})
    assert e.generate_kept(kept) == again
    e.close()


def test_a_prefix_whose_pages_were_given_away_is_refused(tiny, engine):
    from rapidtinyrec_b200._native import NativeError
    a, b = prompts(tiny)[:2]
    store = engine.prefix_store(8, 16)
    n = max(pages_for(a, 16), pages_for(b, 16))
    assert n < 8
    _, first = engine.generate_and_keep(a, store, range(n))
    record = engine.generate_kept(first)
    # what refuses to be kept takes no pages
    with pytest.raises(NativeError):
        engine.keep_prefix(a, store, range(n))
    assert engine.generate_kept(first) == record
    engine.prefill(b)
    with pytest.raises(NativeError):
        engine.keep_prefix(b, store, [0])
    assert engine.generate_kept(first) == record
    for count in (n, 1):  # all of its pages, or one
        _, second = engine.generate_and_keep(b, store, list(range(count - 1, -1, -1)) + list(range(7, 7 - (n - count), -1)))
        for in_place in (True, False):
            with pytest.raises(ValueError, match='given to another'):
                engine.generate_kept(first, in_place=in_place)
        other = engine.generate_kept(second)
        _, first = engine.generate_and_keep(a, store, range(n))
        assert engine.generate_kept(first) == record != other
        with pytest.raises(ValueError, match='given to another'):
            engine.generate_kept(second)


def test_what_others_left_undone_on_the_store_is_raised_before_pages_are_taken(tiny, engine):
    from rapidtinyrec_b200._native import NativeError
    a, b = prompts(tiny)[:2]
    store = engine.prefix_store(8)
    pages = range(max(pages_for(a, 64), pages_for(b, 64)))
    _, first = engine.generate_and_keep(a, store, pages)
    record = engine.generate_kept(first)
    dev = store.device
    q = torch.zeros(1, store.kv_heads, store.head_dim, device=dev)
    store.attention(q, torch.full((1, 1), 8, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev))
    engine.prefill(b)
    with pytest.raises(NativeError, match='page'):
        engine.keep_prefix(b, store, pages)
    assert engine.generate_kept(first) == record
    engine.prefill(b)
    engine.generate_kept(engine.keep_prefix(b, store, pages))


def test_a_prompt_that_was_not_prefilled_is_not_kept(tiny, engine):
    ids = list(prompts(tiny)[0])
    store = engine.prefix_store(8)
    engine.prefill(ids)
    for wrong in (ids[:-1], ids + ids[-1:], ids[:-1] + [ids[-1] + 1]):
        with pytest.raises(ValueError, match='prefilled'):
            engine.keep_prefix(wrong, store, range(pages_for(wrong, 64)))
    given = np.array(ids, dtype=np.int32)
    kept = engine.keep_prefix(given, store, range(pages_for(ids, 64)))
    record = engine.generate_kept(kept)
    given[:] = 0  # the kept prompt is a copy
    assert engine.generate_kept(kept) == record


@pytest.mark.parametrize('fault', ['token', 'wait'])
def test_a_prefill_that_failed_is_not_kept(tiny, engine, fault):
    """A token outside the vocabulary, or a bounded wait that ran out: the store stays as it was, and
    the engine serves on."""
    from rapidtinyrec_b200 import _native
    ids = list(prompts(tiny)[0])
    store = engine.prefix_store(8)
    pages = range(pages_for(ids, 64))
    record, kept = engine.generate_and_keep(ids, store, pages)
    again = engine.generate_kept(kept)
    before = store.k.view(torch.uint8).clone(), store.k_scale.clone()
    wrong = list(ids)
    if fault == 'token':
        wrong[1] = tiny['cfg'].vocab
        engine.prefill(wrong)
    else:
        _native.wait_control(0, 4_000_000, withhold_activation_copies=True)
        try:
            engine.prefill(wrong)
            torch.cuda.synchronize()
        finally:
            _native.wait_control(0)
    with pytest.raises(_native.NativeError) as e:
        engine.keep_prefix(wrong, store, pages)
    assert e.value.code == _native.RTR_ERR_DEVICE
    assert torch.equal(store.k.view(torch.uint8), before[0]) and torch.equal(store.k_scale, before[1])
    assert engine.generate_kept(kept) == again
    assert engine.generate(ids) == record
    assert engine.generate_and_keep(ids, store, pages)[0] == record


def test_a_refused_kept_prefix_ends_the_former_request(tiny, engine):
    from rapidtinyrec_b200._native import RTR_ERR_ARG, RTR_ERR_STATE, NativeError
    from rapidtinyrec_b200.kv_cache import KvCache8
    ids = prompts(tiny)[2]
    store = engine.prefix_store(8)
    record, kept = engine.generate_and_keep(ids, store, range(pages_for(ids, 64)))
    odd = KvCache8(store.k, store.v, store.k_scale, store.v_scale)
    odd._c.page_stride += 8  # refused on the host, after the session began the request
    for in_place in (True, False):
        engine.prefill(ids)
        with pytest.raises(NativeError, match='16 bytes') as e:
            engine.generate_kept(kept._replace(store=odd), in_place=in_place)
        assert e.value.code == RTR_ERR_ARG
        with pytest.raises(NativeError) as e:
            engine.decode_step(1)
        assert e.value.code == RTR_ERR_STATE
    assert engine.generate(ids) == record
    store.check()
