"""The serving operators on the GPU against their formulas in 64 bits: appending to and reading a
paged cache, attention of a ragged batch over it, drawing tokens."""
import math

import pytest
import torch

from parrot_b200 import bridge
from tests.serving_support import (E4M3, Paged, attention, quantise, rope_tables, rotate_f32,
                                   sample_row, starts)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------- append
def _append_expected(cache, qkv, queries, q_heads, rope):
    """The pools after the call, and the queries, on the CPU."""
    sides = 1 if cache.value is None else 2
    x = qkv.float().view(qkv.shape[0], q_heads + sides * cache.kv_heads, cache.dim)
    pos = torch.cat([torch.arange(c - n, c) for n, c in zip(queries, cache.contexts)])
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(queries)]).long()
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + cache.kv_heads], x[:, q_heads + cache.kv_heads:]
    if rope is not None:
        cos, sin = rope[0][pos][:, None], rope[1][pos][:, None]
        q, k = rotate_f32(q, cos, sin), rotate_f32(k, cos, sin)
    page, row = cache.table[seq, pos // cache.page].long(), pos % cache.page
    pools = []
    for side, new in (("key", k), ("value", v)):
        pool, scale = getattr(cache, side), getattr(cache, side + "_scale")
        if pool is None:
            continue
        pool = pool.clone()
        if scale is None:
            pool[page, :, row] = new.to(torch.bfloat16)
        else:
            scale = scale.clone()
            numbers, byte = quantise(new)
            pool.view(torch.uint8)[page, :, row] = numbers.view(torch.uint8)
            scale[page, :, row] = byte
        pools.append((pool, scale))
    return q.to(torch.bfloat16), pools


def _same(pool, got):
    a, b = (t.view(torch.uint8) if t.dtype == E4M3 else t.view(torch.int16) if t.dtype == torch.bfloat16 else t
            for t in (pool, got.cpu()))
    return torch.equal(a, b)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,latent,queries,contexts", [
    (8, 2, 96, 64, False, [1, 1, 1], [1, 64, 65]),
    (8, 2, 96, 16, False, [33, 1, 100, 0, 7], [40, 17, 100, 5, 300]),
    (4, 2, 32, 32, False, [5, 0, 0, 3], [5, 9, 0, 64]),
    (12, 4, 64, 128, False, [129], [1000]),
    (0, 1, 128, 256, True, [2, 300], [2, 511]),
    (3, 1, 128, 16, False, [17], [17]),
])
def test_append_writes_the_rows_bit_for_bit(e4m3, q_heads, kv_heads, dim, page, latent, queries, contexts):
    cache = Paged(contexts, kv_heads=kv_heads, dim=dim, page=page, e4m3=e4m3, latent=latent, seed=dim)
    kv = cache.device()
    tokens, sides = sum(queries), 1 if latent else 2
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(tokens, (q_heads + sides * kv_heads) * dim, generator=g).to(torch.bfloat16)
    rope = None if latent else rope_tables(max(contexts), dim)
    q = bridge.b200_paged_append(kv, qkv.cuda(), cache.table.cuda(), starts(queries).cuda(), ints(contexts),
                                 q_heads, None if rope is None else tuple(t.cuda() for t in rope))
    want_q, pools = _append_expected(cache, qkv, queries, q_heads, rope)
    assert (q is None) == (q_heads == 0)
    if q is not None:
        assert _same(want_q, q)
    assert _same(pools[0][0], kv.key)
    if not latent:
        assert _same(pools[1][0], kv.value)
    if e4m3:
        assert _same(pools[0][1], kv.key_scale)
        assert latent or _same(pools[1][1], kv.value_scale)


def test_append_edge_numbers_in_8_bits():
    """Zeros, the scale's borders, subnormal rows, infinities and NaN."""
    rows = torch.zeros(12, 96)
    rows[1, 0] = 448.0
    rows[2, 0] = 450.0                # one step above: the next power of two
    rows[3] = 2.0 ** -120             # below the least scale's numbers
    rows[4, 3] = 3.0e38
    rows[5, 5] = math.inf
    rows[5, 6] = 1.0
    rows[6, 7] = math.nan
    rows[6, 8] = 2.0
    rows[7] = torch.linspace(-3, 3, 96)
    rows[8, 0], rows[8, 1] = 1.0, 2.0 ** -17  # far below the largest: an e4m3 subnormal or zero
    rows[9] = -0.0
    rows[10] = math.nan
    rows[11, 1] = -math.inf
    x = rows.to(torch.bfloat16)
    cache = Paged([12], kv_heads=1, dim=96, page=16, e4m3=True, latent=True)
    kv = cache.device()
    bridge.b200_paged_append(kv, x.cuda(), cache.table.cuda(), ints([0, 12]), ints([12]), 0)
    numbers, byte = quantise(x.float())
    page = int(cache.table[0, 0])
    got, got_byte = kv.key[page, 0, :12].cpu(), kv.key_scale[page, 0, :12].cpu()
    assert torch.equal(got_byte, byte)
    assert torch.equal(torch.isnan(got.float()), torch.isnan(numbers.float()))
    assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(numbers.float()))
    # reading back: exact bf16 values, NaN in the same places
    dense, none = bridge.b200_paged_gather(kv, cache.table.cuda(), ints([12]), 13)
    assert none is None
    want = numbers.double() * torch.exp2(byte.double() - 127)[:, None]
    got = dense[0, 0, :12].cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.equal(want.nan_to_num(), want.nan_to_num().to(torch.bfloat16).double())
    assert not dense[0, 0, 12].any()


def test_append_strided_rows_and_rows_behind_the_last_sequence():
    cache = Paged([3, 5], kv_heads=2, dim=96, page=16)
    kv = cache.device()
    before = kv.key.clone()
    wide = torch.randn(12, 2 * (8 + 4) * 96).to(torch.bfloat16)
    qkv = wide.cuda()[:, :12 * 96]
    rope = rope_tables(8, 96)
    q = bridge.b200_paged_append(kv, qkv, cache.table.cuda(), ints([0, 3, 8]), ints([3, 5]), 8,
                                 tuple(t.cuda() for t in rope))
    want_q, pools = _append_expected(cache, wide[:8, :12 * 96].contiguous(), [3, 5], 8, rope)
    assert _same(want_q, q[:8])
    assert _same(pools[0][0], kv.key) and _same(pools[1][0], kv.value)
    assert not torch.equal(before, kv.key)


def test_append_reports_and_skips_what_does_not_exist():
    cache = Paged([40, 4, 3], kv_heads=1, dim=32, page=16, latent=True)
    kv = cache.device()
    cache.table[0, 2] = 999                       # no such page: rows 32 .. 39
    before = kv.key.clone()
    x = torch.randn(12, 32).to(torch.bfloat16)
    status = ints([0, 0, 0, 0])
    # sequence 0 appends 8 rows at 32 .. 39, sequence 1 four, sequence 2 none
    bridge.b200_paged_append(kv, x.cuda(), cache.table.cuda(), ints([0, 8, 12, 12]), ints([40, 4, 3]), 0,
                             status=status)
    assert status.tolist()[0] == 2 and status.tolist()[2] == 999
    before[int(cache.table[1, 0]), 0, :4] = x[8:].cuda()
    assert torch.equal(before, kv.key)
    # a position past the table, and one before the start
    for length in (49, 2):
        status.zero_()
        bridge.b200_paged_append(kv, x[:4].cuda(), cache.table[1:2].cuda(), ints([0, 4]), ints([length]), 0,
                                 status=status)
        assert status.tolist()[0] == 2


# ----------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kv_heads,dim,page,latent,contexts,max_len", [
    (2, 96, 64, False, [1, 64, 65, 0, 200], 256), (1, 128, 16, True, [33, 16], 33),
    (4, 64, 32, False, [31], 100), (2, 32, 256, False, [300, 5], 150)])
def test_gather_is_exact_and_zero_behind_the_context(e4m3, kv_heads, dim, page, latent, contexts, max_len):
    cache = Paged(contexts, kv_heads=kv_heads, dim=dim, page=page, e4m3=e4m3, latent=latent, seed=3)
    kv = cache.device()
    k, v = bridge.b200_paged_gather(kv, cache.table.cuda(), ints(contexts), max_len)
    assert (v is None) == latent
    for side, got in (("key", k), ("value", v)):
        if got is None:
            continue
        for b, n in enumerate(contexts):
            n = min(n, max_len)
            want = torch.zeros(kv_heads, max_len, dim, dtype=torch.float64)
            if n:
                want[:, :n] = cache.rows(side, b, n)
            assert torch.equal(got[b].cpu().double(), want), (side, b)
    out = (torch.full_like(k, 7), None if v is None else torch.full_like(v, 7))
    k2, v2 = bridge.b200_paged_gather(kv, cache.table.cuda(), ints(contexts), max_len, out=out)
    assert k2.data_ptr() == out[0].data_ptr() and torch.equal(k, k2) and (v is None or torch.equal(v, v2))


# ------------------------------------------------------------------------------------- attention
def _attend(cache, queries, heads, window, sinks, seed=0, q=None, scale=None, kv=None):
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = torch.randn(sum(queries), heads, cache.dim, generator=g).to(torch.bfloat16)
    scale = cache.dim ** -0.5 if scale is None else scale
    out = bridge.b200_paged_attention(q.cuda(), cache.device() if kv is None else kv, cache.table.cuda(),
                                      starts(queries).cuda(), ints(cache.contexts), window=window,
                                      sinks=sinks, scale=scale)
    want, bound = attention(q, cache, queries, window, sinks, scale)
    off = ((out.cpu().double() - want).abs() / bound)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    assert float(off.nan_to_num().max() if off.numel() else 0.0) <= 1.0
    return out


SHAPES = [(8, 2, 96, False), (8, 1, 128, True), (4, 2, 32, False), (12, 4, 64, False),
          (4, 4, 128, False), (3, 1, 96, False), (40, 1, 64, False)]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,latent", SHAPES)
@pytest.mark.parametrize("queries,contexts,page,window,sinks", [
    ([1], [1], 16, 0, 0),
    ([1, 1, 1, 1], [1, 63, 64, 65], 64, 0, 0),
    ([1, 1, 1], [700, 129, 512], 32, 128, 4),
    ([1, 1], [300, 1000], 16, 1, 0),
    ([1, 1], [300, 1000], 16, 7, 100),
    ([2, 4, 3, 1], [2, 400, 64, 513], 64, 60, 1),
    ([40], [40], 64, 0, 0),
    ([129, 1, 0, 65], [129, 500, 30, 700], 32, 0, 0),
    ([300, 130], [300, 513], 128, 100, 5),
    ([257], [1024], 64, 200, 130),
    ([33, 31], [33, 290], 256, 16, 300),
    ([64], [64 + 128], 16, 1, 1),
])
def test_attention_matches_the_formula(e4m3, heads, kv_heads, dim, latent, queries, contexts, page, window, sinks):
    cache = Paged(contexts, kv_heads=kv_heads, dim=dim, page=page, e4m3=e4m3, latent=latent,
                  seed=len(queries) + page)
    _attend(cache, queries, heads, window, sinks, seed=page + window)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("queries,contexts", [([1, 1, 2], [4096, 2500, 2049]), ([700, 1], [2600, 3000])])
def test_attention_at_the_model_window(e4m3, queries, contexts):
    cache = Paged(contexts, kv_heads=2, dim=96, page=64, e4m3=e4m3, seed=5)
    _attend(cache, queries, 8, 2048, 4)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,latent", SHAPES)
@pytest.mark.parametrize("queries,contexts,page,window,sinks", [
    ([1], [5000], 64, 0, 0), ([2, 1, 0], [4097, 100, 9], 32, 0, 0), ([3], [9001], 128, 5000, 40)])
def test_attention_of_few_rows_over_long_contexts(e4m3, heads, kv_heads, dim, latent, queries, contexts, page,
                                                  window, sinks):
    cache = Paged(contexts, kv_heads=kv_heads, dim=dim, page=page, e4m3=e4m3, latent=latent, seed=dim)
    _attend(cache, queries, heads, window, sinks, seed=heads)


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_of_one_long_context_with_values_that_are_not_finite(e4m3):
    """A NaN reaches the rows that see it, in its column alone; behind the rows it reaches nobody."""
    cache = Paged([6000], kv_heads=1, dim=96, page=64, e4m3=e4m3, seed=3)
    for at, column in ((4500, 17), (5999, 40)):
        page = int(cache.table[0, at // 64])
        if e4m3:
            cache.value.view(torch.uint8)[page, 0, at % 64, column] = 0x7f
        else:
            cache.value[page, 0, at % 64, column] = math.nan
    out = _attend(cache, [2], 4, 0, 0)
    assert torch.isnan(out[..., 17]).all() and torch.isnan(out[1, :, 40]).all()
    assert int(torch.isnan(out).sum()) == 3 * 4


@pytest.mark.parametrize("queries", [[1, 1], [90, 1]])
def test_attention_large_scores_keep_the_running_maximum(queries):
    """Scores of some hundreds, rising and falling along the keys."""
    cache = Paged([600, 333], kv_heads=1, dim=96, page=32, seed=2)
    ramp = torch.linspace(0.1, 9.0, cache.key.shape[0])[:, None, None, None]
    cache.key = (cache.key.float() * ramp).to(torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(sum(queries), 4, 96, generator=g) * 4).to(torch.bfloat16)
    _attend(cache, queries, 4, 0, 0, q=q)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("queries,contexts,window,sinks", [
    ([1, 1], [200, 70], 50, 3), ([2, 3], [200, 70], 50, 3), ([100, 70], [200, 70], 50, 3),
    ([150], [150], 0, 0)])
def test_attention_ignores_whatever_masked_places_hold(e4m3, queries, contexts, window, sinks):
    """NaN and infinities behind the context, outside the window and in pages of nobody."""
    cache = Paged(contexts, kv_heads=2, dim=96, page=16, e4m3=e4m3, seed=9)
    kv = cache.device()
    clean = _attend(cache, queries, 8, window, sinks, kv=kv)
    table, poison = cache.table.clone(), (0x7f if e4m3 else math.nan)
    owned = torch.zeros(cache.pages, 16, dtype=torch.bool)
    for b, (n, c) in enumerate(zip(queries, contexts)):
        for j in range(c):
            first = c - n
            if window == 0 or j < sinks or first - j < window:
                owned[int(cache.table[b, j // 16]), j % 16] = True
        for p in range(-(-c // 16)):
            if not owned[int(cache.table[b, p])].any():
                table[b, p] = -5  # given away
    where = ~owned.cuda()[:, None, :, None].expand(kv.key.shape)
    for i, pool in enumerate((kv.key, kv.value)):
        if e4m3:
            pool.view(torch.uint8)[where] = poison
        else:
            pool[where] = poison if i else math.inf
    status = ints([0, 0, 0, 0])
    g = torch.Generator().manual_seed(0)
    q = torch.randn(sum(queries), 8, 96, generator=g).to(torch.bfloat16).cuda()
    out = bridge.b200_paged_attention(q, kv, table.cuda(), starts(queries).cuda(), ints(contexts),
                                      window=window, sinks=sinks, status=status)
    assert torch.equal(out, clean)
    assert status.tolist()[0] == 0


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("queries,contexts,window,at", [([4], [60], 0, 57), ([130], [140], 0, 100),
                                                        ([130], [400], 64, 290), ([3], [40], 8, 31)])
def test_a_bad_value_reaches_only_the_tokens_that_see_it(e4m3, bad, queries, contexts, window, at):
    """A key/value that some tokens of the chunk see and others do not."""
    cache = Paged(contexts, kv_heads=1, dim=96, page=16, e4m3=e4m3, seed=4)
    kv = cache.device()
    clean = _attend(cache, queries, 4, window, 0, kv=kv)
    page, row = int(cache.table[0, at // 16]), at % 16
    if e4m3:
        kv.value.view(torch.uint8)[page, 0, row, 5] = 0x7f
    else:
        kv.value[page, 0, row, 5] = bad
    g = torch.Generator().manual_seed(0)
    q = torch.randn(sum(queries), 4, 96, generator=g).to(torch.bfloat16).cuda()
    out = bridge.b200_paged_attention(q, kv, cache.table.cuda(), starts(queries).cuda(), ints(contexts),
                                      window=window)
    pos = torch.arange(contexts[0] - queries[0], contexts[0])
    sees = (pos >= at) & ((pos - at < window) if window else torch.tensor(True))
    assert sees.any() and not sees.all()
    same = out == clean
    assert same[~sees].all()
    assert not torch.isfinite(out[sees][:, :, 5]).any()
    keep = [d for d in range(96) if d != 5]
    assert same[:, :, keep].all()


def test_attention_strided_queries_rows_behind_and_empty_contexts():
    cache = Paged([50, 0, 20], kv_heads=2, dim=96, page=16, seed=1)
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(12, 12 * 96, generator=g).to(torch.bfloat16)
    q = wide.cuda()[:, :8 * 96].unflatten(1, (8, 96))
    # sequence 1 has two rows and no context: they see nothing; rows 10, 11 belong to no one
    out = bridge.b200_paged_attention(q, cache.device(), cache.table.cuda(), ints([0, 5, 7, 10]),
                                      ints([50, 0, 20]))
    want, bound = attention(wide[:, :8 * 96].reshape(12, 8, 96)[[0, 1, 2, 3, 4, 7, 8, 9]],
                            _with(cache, contexts=[50, 20], table=cache.table[[0, 2]]), [5, 3], 0, 0, 96 ** -0.5)
    got = out[[0, 1, 2, 3, 4, 7, 8, 9]].cpu().double()
    assert float(((got - want).abs() / bound).max()) <= 1
    assert not out[5:7].any()


def _with(cache, **kw):
    c = Paged.__new__(Paged)
    c.__dict__.update(cache.__dict__, **kw)
    return c


def test_a_missing_page_reads_as_zeros_and_is_reported():
    cache = Paged([100], kv_heads=1, dim=64, page=32, seed=6)
    kv = cache.device()
    for n in (1, 60):
        table = cache.table.clone()
        table[0, 1] = cache.pages
        status = ints([0, 0, 0, 0])
        g = torch.Generator().manual_seed(0)
        q = torch.randn(n, 2, 64, generator=g).to(torch.bfloat16)
        out = bridge.b200_paged_attention(q.cuda(), kv, table.cuda(), ints([0, n]), ints([100]), status=status)
        zeroed = _with(cache, key=cache.key.clone(), value=cache.value.clone())
        zeroed.key[int(cache.table[0, 1])] = 0
        zeroed.value[int(cache.table[0, 1])] = 0
        want, bound = attention(q, zeroed, [n], 0, 0, 64 ** -0.5)
        assert float(((out.cpu().double() - want).abs() / bound).max()) <= 1
        assert status.tolist()[0] == 2 and status.tolist()[2] == cache.pages


@pytest.mark.parametrize("queries", [[1, 1, 1], [1, 200, 3]])
def test_attention_repeats_bit_for_bit_in_graphs_on_two_streams(queries):
    cache = Paged([900, 400, 64], kv_heads=2, dim=96, page=64, seed=8)
    kv, table = cache.device(), cache.table.cuda()
    start, length = starts(queries).cuda(), ints(cache.contexts)
    qs = [torch.randn(sum(queries), 8, 96, device="cuda").to(torch.bfloat16) for _ in range(2)]

    def call(q):
        return bridge.b200_paged_attention(q, kv, table, start, length, window=300, sinks=4)
    eager = [call(q).clone() for q in qs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(q))
        graphs.append(graph)
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for want, got in zip(eager, outs):
        assert torch.equal(want, got)
    # a replay at new lengths: the lengths are read on the device
    length.copy_(ints([500, 400, 20]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], call(qs[0])) and not torch.equal(outs[0], eager[0])


@pytest.mark.parametrize("queries", [[1, 1, 1], [70, 1, 40]])
def test_a_captured_step_follows_the_lists_it_reads(queries):
    """Append, attention and read-back captured once and replayed after the page table, the
    lengths and the rows changed in place."""
    contexts = [200, 33, 90]
    cache = Paged(contexts, kv_heads=2, dim=96, page=16, e4m3=True, seed=4, spare=30)
    kv, width = cache.device(), 18
    free = [p for p in range(cache.pages) if p not in set(cache.table.flatten().tolist())]
    table = torch.full((3, width), -1, dtype=torch.int32)
    table[:, :cache.table.shape[1]] = cache.table
    more = table.clone()
    for b, n in enumerate(contexts):
        have, need = -(-n // 16), -(-(n + 50) // 16)
        for i in range(have, need):
            more[b, i] = free.pop()
    first = table.cuda()
    start, length = starts(queries).cuda(), ints(contexts)
    tables = tuple(t.cuda() for t in rope_tables(300, 96))
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn(sum(queries), 12 * 96, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    qkv = rows[0].clone()

    def step(kv, table, length, qkv):
        q = bridge.b200_paged_append(kv, qkv, table, start, length, 8, tables)
        y = bridge.b200_paged_attention(q, kv, table, start, length, window=64, sinks=3)
        return y, *bridge.b200_paged_gather(kv, table, length, 260)

    def fresh():
        return bridge.PagedKV(*(t.clone() for t in (kv.key, kv.value, kv.key_scale, kv.value_scale)))
    eager_kv = fresh()
    want = [step(eager_kv, first, length, rows[0]),
            step(eager_kv, more.cuda(), length + 50, rows[1])]
    step(fresh(), first, length, qkv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kv, first, length, qkv)
    graph.replay()
    got = [t.clone() for t in out]
    first.copy_(more)
    length.add_(50)
    qkv.copy_(rows[1])
    graph.replay()
    for a, b in zip(want[0] + want[1], got + list(out)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("most", [3, 40])
def test_more_sequences_than_lanes(e4m3, most):
    """Seventy sequences, some of them without new tokens, some without any."""
    g = torch.Generator().manual_seed(most)
    queries = torch.randint(0, most + 1, (70,), generator=g).tolist()
    contexts = [n + int(torch.randint(0, 150, (1,), generator=g)) * (i % 5 > 0) for i, n in enumerate(queries)]
    cache = Paged(contexts, kv_heads=2, dim=96, page=16, e4m3=e4m3, seed=1)
    _attend(cache, queries, 8, 40, 2)


def test_numbers_that_do_not_fit_the_call_are_refused():
    cache = Paged([50], kv_heads=1, dim=96, page=16)
    kv, q = cache.device(), torch.randn(1, 2, 96, device="cuda").to(torch.bfloat16)
    lists = cache.table.cuda(), ints([0, 1]), ints([50])
    whole = bridge.b200_paged_attention(q, kv, *lists)
    for window in (50, 10 ** 6, 2 ** 31 - 1):       # no position is that far
        assert torch.equal(whole, bridge.b200_paged_attention(q, kv, *lists, window=window, sinks=2 ** 31 - 1))
    for kw in (dict(window=2 ** 32 + 5), dict(window=-1), dict(window=4, sinks=2 ** 32), dict(sinks=-1),
               dict(window=2 ** 31)):
        with pytest.raises(ValueError, match="window and sinks"):
            bridge.b200_paged_attention(q, kv, *lists, **kw)
    logits, u = torch.randn(1, 64, device="cuda"), torch.full((1,), 0.5, device="cuda")
    for k in (-1, 2 ** 31, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="top_k"):
            bridge.b200_sample(logits, u, top_k=k)


def test_offsets_past_32_bits():
    """A pool whose last pages lie behind 2**31 numbers."""
    page, dim = 256, 128
    pages = (2 ** 31) // (page * dim) + 3
    pool = torch.empty((pages, 1, page, dim), device="cuda", dtype=torch.bfloat16)
    kv = bridge.PagedKV(pool)
    table = ints([[pages - 1, 0, pages - 2]])
    x = torch.randn(600, dim, device="cuda").to(torch.bfloat16)
    bridge.b200_paged_append(kv, x, table, ints([0, 600]), ints([600]), 0)
    dense, _ = bridge.b200_paged_gather(kv, table, ints([600]), 600)
    assert torch.equal(dense[0, 0], x)
    small = bridge.PagedKV(torch.stack([pool[pages - 1], pool[0], pool[pages - 2]]))
    for n in (1, 100):
        q = torch.randn(n, 8, dim, device="cuda").to(torch.bfloat16)
        far = bridge.b200_paged_attention(q, kv, table, ints([0, n]), ints([600]))
        near = bridge.b200_paged_attention(q, small, ints([[0, 1, 2]]), ints([0, n]), ints([600]))
        assert torch.equal(far, near)


# -------------------------------------------------------------------------------------- sampling
def _draw(logits, u, t, k, p, m):
    ids, logp = bridge.b200_sample(logits.cuda(), u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    assert ids.shape == (logits.shape[0], 1) and ids.dtype == torch.int64
    for r in range(logits.shape[0]):
        token, want = sample_row(logits[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert int(ids[r, 0]) == token, (r, int(ids[r, 0]), token, float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        # one rounding to fp32 of a 64-bit logarithm whose masses are off by 2**-45 each
        assert float(logp[r]) == want or abs(float(logp[r]) - want) <= 2.0 ** -23 * abs(want) + 1e-7
    return ids


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4097, 32768])
def test_sampling_draws_the_defined_token(dtype, vocab):
    rows = 48
    g = torch.Generator().manual_seed(vocab)
    logits = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    u = torch.rand(rows, generator=g)
    i = torch.arange(rows)
    t = torch.tensor([1.0, 0.7, 0.0, 2.5, 0.05])[i % 5]
    k = torch.tensor([0, 1, 5, 50, 40000, 3])[i % 6].int()
    p = torch.tensor([1.0, 0.9, 0.5, 0.01, 0.999, 0.0, 1.5])[i % 7]
    m = torch.tensor([0.0, 0.1, 0.0, 0.001])[i % 4]
    _draw(logits, u, t, k, p, m)


def test_sampling_ties_and_borders():
    """Equal logits: the lower index first, a set cut inside the tie, a draw on a border."""
    rows, vocab = 40, 64
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16)
    logits[1::2, 10:20] = 1.0
    logits[2::4, 5] = -0.0
    u = torch.linspace(0, 1 - 2 ** -24, rows)
    u[0], u[4], u[8] = 0.0, 0.5, 0.25           # 32 / 64 and 16 / 64 of equal masses: exact borders
    one = torch.ones(rows)
    k = torch.tensor([0, 15, 7, 64, 63])[torch.arange(rows) % 5].int()
    p = torch.tensor([1.0, 0.5, 0.25, 0.75])[torch.arange(rows) % 4]
    _draw(logits, u, one, k, p, 0 * one)
    _draw(logits, u, one, k, 0 * p + 1, one)     # min_p 1: the largest alone
    _draw(logits.float(), u, one * 0.3, k, p, 0 * one)


def test_sampling_masked_and_broken_logits():
    inf = math.inf
    rows = torch.full((6, 500), -inf)
    rows[1, 77] = -3.0
    rows[2, 3:9] = torch.tensor([1.0, math.nan, 2.0, math.nan, -inf, 2.0])
    rows[3] = math.nan
    rows[4, 10], rows[4, 20], rows[4, 30] = inf, inf, 5.0
    rows[5, 499], rows[5, 0] = torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).min
    for dtype in (torch.bfloat16, torch.float32):
        for t, k, p in ((1.0, 0, 1.0), (0.0, 0, 1.0), (0.5, 3, 0.9), (1e-30, 0, 0.5), (1e30, 0, 0.7)):
            full = torch.full((6,), t)
            ids = _draw(rows.to(dtype), torch.linspace(0, 0.99, 6), full, torch.full((6,), k).int(),
                        torch.full((6,), p), torch.zeros(6))
            assert ids[0, 0] == -1 and ids[1, 0] == 77 and ids[3, 0] == -1


def test_sampling_numbers_for_all_rows_strides_and_a_single_position():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(9, 1, 700, generator=g).to(torch.bfloat16)
    u = torch.rand(9, generator=g)
    view = wide.cuda()[:, :, 3:602]
    ids, logp = bridge.b200_sample(view, u.cuda(), temperature=0.8, top_k=20, top_p=0.9, min_p=0.02)
    for r in range(9):
        token, want = sample_row(wide[r, 0, 3:602], float(u[r]), float(torch.tensor(0.8)), 20,
                                 float(torch.tensor(0.9)), float(torch.tensor(0.02)))
        assert int(ids[r]) == token and abs(float(logp[r]) - want) <= 1e-6
    greedy, zero = bridge.b200_sample(view, u.cuda(), temperature=0.0)
    assert torch.equal(greedy[:, 0].cpu(), wide[:, 0, 3:602].float().argmax(-1)) and not zero.any()


def test_sampling_frequencies_follow_the_shares():
    """Over an even grid of random numbers each token comes up its share of times, within one."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(300, generator=g).to(torch.bfloat16)
    n = 4096
    u = (torch.arange(n).float() + 0.5) / n
    ids, _ = bridge.b200_sample(logits.cuda().expand(n, -1), u.cuda(), temperature=1.0)
    share = torch.softmax(logits.double(), 0) * n
    count = torch.bincount(ids[:, 0].cpu(), minlength=300).double()
    assert float((count - share).abs().max()) <= 1.0
