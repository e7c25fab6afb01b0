"""The serving operators at the edges of their ranges, against their formulas in 64 bits."""
import math

import pytest
import torch

from parrot_b200 import bridge
from tests.serving_support import E4M3, Paged, attention, quantise, sample_row, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _inference():
    with torch.inference_mode():
        yield


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _call(cache, queries, q, window=0, sinks=0, scale=None, table=None, status=None):
    return bridge.b200_paged_attention(q.cuda(), cache.device(), (cache.table if table is None else table).cuda(),
                                       starts(queries).cuda(), ints(cache.contexts), window=window, sinks=sinks,
                                       scale=scale, status=status).cpu()


def _assert_formula(out, cache, queries, q, window=0, sinks=0, scale=None):
    """Finite results within the formula's bound; NaN and each infinity where the formula has them."""
    want, bound = attention(q, cache, queries, window, sinks, cache.dim ** -0.5 if scale is None else scale)
    got = out.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    for inf in (math.inf, -math.inf):
        assert torch.equal(got == inf, want == inf)
    finite = torch.isfinite(want)
    assert float(((got - want).abs() / bound)[finite].max() if finite.any() else 0.0) <= 1.0


def _queries(n, heads, dim, seed):
    return torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


# ------------------------------------------------------------- value rows of very different size
def _numbers(shape, seed):
    """Magnitudes in [1/2, 1) of either sign: no 8-bit number of such a row is zero."""
    g = torch.Generator().manual_seed(seed)
    x = 0.5 + 0.5 * torch.rand(shape, generator=g)
    return torch.where(torch.rand(shape, generator=g) < 0.5, -x, x)


def _spread_cache(context, dim, kv_heads, order, rise, q, e4m3=True):
    """Keys whose scores rise by `rise` (natural logarithm) along the context, or fall, for the query
    direction `q` [dim]; values of 2**60 down to 2**-60, or up, or in any order."""
    cache = Paged([context], kv_heads=kv_heads, dim=dim, page=32, e4m3=e4m3, seed=1)
    along = torch.linspace(0, 1, context)
    if order == "scores fall, values grow":
        along = along.flip(0)
    score = along * rise
    exponent = (60 - 120 * along).round()
    if order == "any order":
        turn = torch.randperm(context, generator=torch.Generator().manual_seed(3))
        exponent = exponent[turn]
    unit = q.float() / float(q.double().norm()) ** 2 * dim ** 0.5   # scale dim**-0.5: q . k is the score
    key = (score[:, None] * unit).expand(kv_heads, -1, -1)
    value = _numbers((kv_heads, context, dim), 2) * torch.exp2(exponent)[:, None]
    for side, rows in (("key", key), ("value", value)):
        pool = torch.zeros(cache.pages, kv_heads, 32, dim)
        for j in range(context):
            pool[int(cache.table[0, j // 32]), :, j % 32] = rows[:, j]
        if e4m3:
            numbers, scale = quantise(pool)
            setattr(cache, side, numbers)
            setattr(cache, side + "_scale", scale)
        else:
            setattr(cache, side, pool.to(torch.bfloat16))
    return cache


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("queries", [[1], [2], [100]])
@pytest.mark.parametrize("context", [320, 1000, 5000])
@pytest.mark.parametrize("order,rise", [("scores rise, values shrink", 50.0), ("scores rise, values shrink", 85.0),
                                        ("scores rise, values shrink", 110.0), ("scores fall, values grow", 110.0),
                                        ("any order", 30.0)])
def test_values_of_very_different_size(order, rise, context, queries, e4m3):
    """What softmax has made negligible must not set the precision of what counts."""
    dim, kv_heads = 96, 2
    one = _queries(1, 1, dim, 5)[0, 0]
    cache = _spread_cache(context, dim, kv_heads, order, rise, one, e4m3)
    # each head the same direction, at its own strength
    strength = torch.tensor([1.0, 0.5, -1.0, 0.25])
    q = (one.float() * strength[:, None]).to(torch.bfloat16).expand(sum(queries), 4, dim).contiguous()
    out = _call(cache, queries, q)
    _assert_formula(out, cache, queries, q)


@pytest.mark.parametrize("queries", [[1], [2], [100]])
@pytest.mark.parametrize("first,later,rise", [(120, -100, 200.0), (-100, 120, -200.0), (-100, 120, 0.0),
                                              (120, -100, 60.0), (-102, -102, 10.0), (-102, -102, -10.0)])
def test_values_at_both_ends_of_the_range(first, later, rise, queries):
    """Half of the context at one scale, half at the other, with a step of the scores between them."""
    context, dim = 700, 96
    cache = Paged([context], kv_heads=1, dim=dim, page=32, e4m3=True, seed=1)
    one = _queries(1, 1, dim, 5)[0, 0]
    unit = one.float() / float(one.double().norm()) ** 2 * dim ** 0.5
    value = _numbers((context, dim), 2) * torch.exp2(torch.where(torch.arange(context) < 350, first, later).float())[:, None]
    for side, rows in (("key", torch.where(torch.arange(context) < 350, 0.0, rise)[:, None] * unit), ("value", value)):
        pool = torch.zeros(cache.pages, 1, 32, dim)
        for j in range(context):
            pool[int(cache.table[0, j // 32]), 0, j % 32] = rows[j]
        numbers, scale = quantise(pool)
        setattr(cache, side, numbers)
        setattr(cache, side + "_scale", scale)
    q = one.expand(sum(queries), 2, dim).contiguous()
    _assert_formula(_call(cache, queries, q), cache, queries, q)


@pytest.mark.parametrize("first,later", [(3, -36), (-36, 3)])
@pytest.mark.parametrize("context", [300, 4500])
def test_latent_rows_of_very_different_size(first, later, context):
    """A latent: large rows that the queries turn away from, beside small ones that they do not, and
    the reverse order."""
    cache = Paged([context], kv_heads=1, dim=128, page=64, e4m3=True, latent=True, seed=1)
    q = _queries(1, 1, 128, 6)
    g = torch.Generator().manual_seed(7)
    pool = torch.zeros(cache.pages, 1, 64, 128)
    for j in range(context):
        e = first if j < context // 2 else later
        row = _numbers((128,), j) * 2.0 ** e
        if e > 0:   # score about -60 for every head below
            row = -q[0, 0].float().sign() * row.abs()
        pool[int(cache.table[0, j // 64]), 0, j % 64] = row
    cache.key, cache.key_scale = quantise(pool)
    q = q.expand(1, 8, 128).contiguous()
    _assert_formula(_call(cache, [1], q), cache, [1], q)


@pytest.mark.parametrize("queries", [[1, 1], [90, 1], [4]])
def test_large_scores_keep_the_running_maximum_in_8_bits(queries):
    contexts = [600, 333][:len(queries)]
    cache = Paged(contexts, kv_heads=1, dim=96, page=32, seed=2, e4m3=True)
    x = torch.randn(cache.key.shape, generator=torch.Generator().manual_seed(3))
    ramp = torch.linspace(0.1, 9.0, cache.key.shape[0])[:, None, None, None]
    cache.key, cache.key_scale = quantise(x * ramp)
    q = (_queries(sum(queries), 4, 96, 1).float() * 4).to(torch.bfloat16)
    _assert_formula(_call(cache, queries, q), cache, queries, q)


# ------------------------------------------------------------------------ numbers that are not finite
SIGNS = [(math.inf,), (-math.inf,), (math.nan,), (math.inf, -math.inf), (math.inf, math.inf)]


@pytest.mark.parametrize("bad", SIGNS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 96), (8, 2, 128), (3, 1, 32)])
@pytest.mark.parametrize("queries,context,window,sinks,at", [
    ([1], 300, 0, 0, 100), ([4], 60, 0, 0, 57), ([4], 400, 0, 0, 30), ([3], 5000, 0, 0, 4000),
    ([130], 140, 0, 0, 100),        # on the diagonal
    ([130], 1000, 0, 0, 200),       # where every row sees it
    ([130], 400, 64, 0, 290),       # at the window's start
    ([300], 700, 100, 5, 3),        # among the first tokens
    ([500], 500, 0, 0, 0),
])
def test_an_infinite_value_is_what_the_formula_says(queries, context, window, sinks, at, heads, kv_heads, dim, bad):
    """Wherever it lies in a tile: an infinity for the rows that see it, NaN beside its opposite."""
    cache = Paged([context], kv_heads=kv_heads, dim=dim, page=16, seed=4)
    for i, x in enumerate(bad):
        cache.value[int(cache.table[0, (at + i) // 16]), 0, (at + i) % 16, 5] = x
    q = _queries(sum(queries), heads, dim, 0)
    out = _call(cache, queries, q, window, sinks)
    _assert_formula(out, cache, queries, q, window, sinks)


@pytest.mark.parametrize("column", [5, 100])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("queries,context,at", [
    ([1], 300, 100), ([4], 60, 57), ([3], 5000, 4000), ([130], 140, 100), ([130], 1000, 200), ([500], 500, 0)])
def test_an_infinite_latent_row_is_what_the_formula_says(queries, context, at, bad, column):
    """Its score is an infinity of either sign, as the query has it: a row that turns away from it
    loses its column alone (zero times infinity), one that turns to it, or a NaN, everything."""
    cache = Paged([context], kv_heads=1, dim=128, page=16, latent=True, seed=4)
    cache.key[int(cache.table[0, at // 16]), 0, at % 16, column] = bad
    q = _queries(sum(queries), 8, 128, 0)
    q[:, 2, column] = 0.0          # zero times infinity
    out = _call(cache, queries, q)
    _assert_formula(out, cache, queries, q)


def test_two_infinite_numbers_in_a_latent_row():
    cache = Paged([150], kv_heads=1, dim=128, page=16, latent=True, seed=4)
    row = cache.key[int(cache.table[0, 100 // 16]), 0, 100 % 16]
    row[5], row[70] = math.inf, -math.inf
    for queries in ([130], [3]):
        q = _queries(sum(queries), 8, 128, 0)
        q[:, 0, 5], q[:, 0, 70] = 1.0, 1.0
        q[:, 1, 5], q[:, 1, 70] = -1.0, 1.0
        q[:, 2, 5], q[:, 2, 70] = 1.0, -1.0
        q[:, 3, 9] = math.nan
        _assert_formula(_call(cache, queries, q), cache, queries, q)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("queries,context,at", [
    ([1], 300, 100), ([4], 60, 57), ([3], 5000, 4000), ([130], 140, 100), ([130], 1000, 200), ([500], 500, 0)])
def test_an_infinite_key_is_what_the_formula_says(queries, context, at, bad, e4m3):
    """A score of -infinity has no weight, one of +infinity or NaN leaves a row of NaN; a token whose
    only key has no weight has 0 / 0."""
    if e4m3 and not math.isnan(bad):
        pytest.skip("8-bit numbers have no infinity")
    cache = Paged([context], kv_heads=1, dim=96, page=16, e4m3=e4m3, seed=4)
    page = int(cache.table[0, at // 16])
    if e4m3:
        cache.key.view(torch.uint8)[page, 0, at % 16, 7] = 0x7f
    else:
        cache.key[page, 0, at % 16, 7] = bad
    q = _queries(sum(queries), 4, 96, 0)
    _assert_formula(_call(cache, queries, q), cache, queries, q)


# ------------------------------------------------------------------------------------- fp32 queries
def _assert_formula_f32(out, cache, queries, q, window=0, sinks=0, scale=None):
    """Within a bound that bf16 queries, weights or results would miss.

    Queries and weights are two bf16 numbers each, off by at most 2**-16 and 2**-17.  With
    S = scale sum |q| |k|, a score is off by 2**-16 S and by D + 3 fp32 roundings of its terms (2**-22 S
    each at most, however the products are summed), so a weight by twice that, relative; the sums over
    the keys by 2**-16 more.  Where S is small beside 1 a result is off by less than a step of 2**-14.
    """
    scale = cache.dim ** -0.5 if scale is None else scale
    want, bound = attention(q, cache, queries, window, sinks, scale)
    mass = bound / (2.0 ** -8 + 2.0 ** -12)                 # at least sum p |v| / sum p
    first = 0
    size = torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64)
    for b, n in enumerate(queries):
        k = cache.rows("key", b).abs().nan_to_num(0.0, 0.0)
        if n:
            size[first:first + n] = (q[first:first + n].double().abs().nan_to_num(0.0, 0.0)
                                     @ k[0].T).amax(-1, keepdim=True) * scale
        first += n
    tight = mass * (2 * (2.0 ** -16 + (cache.dim + 3) * 2.0 ** -22) * size + 2.0 ** -16 + 2.0 ** -17)
    assert out.dtype == torch.float32
    got = out.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    finite = torch.isfinite(want)
    assert bool(((got - want).abs() <= tight.expand_as(want))[finite].all())


@pytest.mark.parametrize("heads,dim", [(8, 128), (3, 96), (40, 64), (4, 32)])
@pytest.mark.parametrize("queries,contexts,page,window,sinks", [
    ([1], [1], 16, 0, 0), ([1, 1, 1, 1], [1, 63, 64, 65], 64, 0, 0), ([1, 1], [300, 1000], 16, 7, 100),
    ([2, 4, 3, 1], [2, 400, 64, 513], 64, 60, 1), ([1], [5000], 64, 0, 0), ([40], [40], 64, 0, 0),
    ([129, 1, 0, 65], [129, 500, 30, 700], 32, 0, 0), ([300, 130], [300, 513], 128, 100, 5),
    ([257], [1024], 64, 200, 130), ([64] * 40, [200] * 40, 32, 0, 0)])
def test_fp32_queries_over_a_latent_cache(queries, contexts, page, window, sinks, heads, dim):
    cache = Paged(contexts, kv_heads=1, dim=dim, page=page, latent=True, seed=len(queries) + page)
    q = torch.randn(sum(queries), heads, dim, generator=torch.Generator().manual_seed(page + window))
    out = _call(cache, queries, q, window, sinks)
    _assert_formula_f32(out, cache, queries, q, window, sinks)


@pytest.mark.parametrize("queries", [[1], [200]])
def test_fp32_queries_strided_and_rows_of_nobody(queries):
    n = sum(queries)
    cache = Paged([n + 30], kv_heads=1, dim=96, page=16, latent=True, seed=2)
    wide = torch.randn(n + 3, 5, 104, generator=torch.Generator().manual_seed(3))
    for view in (wide[:, 1:4, 4:100], wide.flatten(1)[:, 4:292].unflatten(1, (3, 96)),
                 wide.flatten(1)[:, 1:289].unflatten(1, (3, 96))):
        dev = wide.cuda()
        q = torch.as_strided(dev, view.shape, view.stride(), view.storage_offset())
        out = bridge.b200_paged_attention(q, cache.device(), cache.table.cuda(), starts(queries).cuda(),
                                          ints(cache.contexts))
        _assert_formula_f32(out[:n].cpu(), cache, queries, view[:n].contiguous())


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("queries,context,at", [([1], 300, 100), ([4], 60, 57), ([130], 140, 100), ([130], 1000, 200)])
def test_fp32_queries_and_an_infinite_latent_row(queries, context, at, bad):
    """Both parts of a query have its sign: their products with an infinity are the same one."""
    cache = Paged([context], kv_heads=1, dim=128, page=16, latent=True, seed=4)
    cache.key[int(cache.table[0, at // 16]), 0, at % 16, 5] = bad
    q = torch.randn(sum(queries), 8, 128, generator=torch.Generator().manual_seed(0))
    q[:, 1] = q[:, 1].to(torch.bfloat16).float()     # nothing left for the low part
    q[:, 2, 5] = 0.0
    _assert_formula_f32(_call(cache, queries, q), cache, queries, q)


@pytest.mark.parametrize("queries", [[1, 1, 1], [1, 200, 3]])
def test_fp32_queries_in_a_graph_follow_the_lists(queries):
    contexts = [900, 400, 64]
    cache = Paged(contexts, kv_heads=1, dim=128, page=64, latent=True, seed=8)
    kv, table, start, length = cache.device(), cache.table.cuda(), starts(queries).cuda(), ints(contexts)
    q = torch.randn(sum(queries), 8, 128, device="cuda")
    eager = bridge.b200_paged_attention(q, kv, table, start, length)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bridge.b200_paged_attention(q, kv, table, start, length)
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, eager)
    length.copy_(ints([500, 400, 20]))
    graph.replay()
    assert torch.equal(out, bridge.b200_paged_attention(q, kv, table, start, length)) and not torch.equal(out, eager)


def test_fp32_queries_need_a_bf16_latent_cache():
    q = torch.zeros(1, 2, 96, device="cuda")
    for kw in (dict(latent=False), dict(latent=True, e4m3=True)):
        cache = Paged([4], kv_heads=1, dim=96, page=16, **kw)
        with pytest.raises(RuntimeError, match="bf16 latent"):
            bridge.b200_paged_attention(q, cache.device(), cache.table.cuda(), ints([0, 1]), ints([4]))


# ------------------------------------------------------------------------------------------- scales
def test_every_scale_reads_as_the_power_of_two_it_stands_for():
    """Read back, all 256 numbers at the bytes 1 .. 254: number * 2**(byte - 127), rounded once to bf16 where that
    leaves its normal numbers (the bytes that the append writes, 17 .. 246, never do)."""
    page = 128
    cache = Paged([4 * page], kv_heads=1, dim=128, page=page, e4m3=True, latent=True)
    at = torch.arange(508)
    numbers = torch.arange(256, dtype=torch.uint8).view(2, 128)[at % 2]
    byte = (1 + at // 2).to(torch.uint8)
    for j in range(508):
        p = int(cache.table[0, j // page])
        cache.key.view(torch.uint8)[p, 0, j % page] = numbers[j]
        cache.key_scale[p, 0, j % page] = byte[j]
    got, _ = bridge.b200_paged_gather(cache.device(), cache.table.cuda(), ints([508]), 508)
    got = got[0, 0].cpu()
    exact = numbers.view(E4M3).double() * torch.exp2(byte.double() - 127)[:, None]
    want = exact.to(torch.bfloat16)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan].view(torch.int16), want[~nan].view(torch.int16))
    written = (byte >= 17) & (byte <= 246)
    assert torch.equal(want[written].double().nan_to_num(), exact[written].nan_to_num())


# --------------------------------------------------------------------------- pages that do not exist
@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("n", [1, 3, 60, 400])
def test_a_missing_page_of_an_8_bit_cache_reads_as_zeros_and_is_reported(n, latent):
    cache = Paged([600], kv_heads=1, dim=128 if latent else 64, page=32, seed=6, e4m3=True, latent=latent)
    for wrong in (cache.pages, -1):
        table = cache.table.clone()
        table[0, 4] = wrong
        status = ints([0, 0, 0, 0])
        q = _queries(n, 2, cache.dim, 0)
        out = _call(cache, [n], q, table=table, status=status)
        zeroed = Paged.__new__(Paged)
        zeroed.__dict__.update(cache.__dict__, key=cache.key.clone())
        zeroed.key.view(torch.uint8)[int(cache.table[0, 4])] = 0
        if not latent:
            zeroed.value = cache.value.clone()
            zeroed.value.view(torch.uint8)[int(cache.table[0, 4])] = 0
        _assert_formula(out, zeroed, [n], q)
        assert status.tolist()[0] == 2 and status.tolist()[2] == wrong


# ------------------------------------------------------------------------------------------ sampling
def _assert_draws(logits, u, t, k, p, m, rows=None):
    ids, logp = bridge.b200_sample(logits.cuda(), u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    for r in range(logits.shape[0]) if rows is None else rows:
        token, want = sample_row(logits[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert int(ids[r, 0]) == token, (r, int(ids[r, 0]), token)
        assert abs(float(logp[r]) - want) <= 2.0 ** -23 * abs(want) + 1e-7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("where", ["at the top", "below it", "everywhere", "near one another"])
def test_sampling_among_thousands_of_equal_logits(where, dtype):
    """More tokens in one step of the histogram than the list of a step holds."""
    rows, vocab = 8, 9001
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(rows, vocab, generator=g)
    at = torch.randperm(vocab, generator=g)[:6000]
    if where == "at the top":
        logits[:, at] = 5.0
    elif where == "below it":
        logits[:, at] = 2.0
    elif where == "everywhere":
        logits[:] = -1.5
    else:   # a wide range, so that a step of it holds thousands of different logits
        logits = logits * 1e-3
        logits[:, 17] = -300.0
    i = torch.arange(rows)
    u = torch.rand(rows, generator=g)
    one = torch.ones(rows)
    for k, p in ((3000, 1.0), (0, 0.4), (5000, 0.5), (1, 1.0), (0, 0.9)):
        _assert_draws(logits.to(dtype), u, one, (0 * i + k).int(), 0 * one + p, 0 * one)


@pytest.mark.parametrize("dtype,vocab,rows", [(torch.bfloat16, 131072, 200), (torch.float32, 131072, 200),
                                              (torch.float32, 500001, 2), (torch.bfloat16, 524288, 3)])
def test_sampling_rows_longer_than_shared_memory_holds(dtype, vocab, rows):
    g = torch.Generator().manual_seed(vocab)
    logits = (2 * torch.randn(rows, vocab, generator=g)).to(dtype)
    u = torch.rand(rows, generator=g)
    i = torch.arange(rows)
    t = torch.tensor([1.0, 0.7, 0.0])[i % 3]
    k = torch.tensor([0, 40, 100000, 7])[i % 4].int()
    p = torch.tensor([0.9, 1.0, 0.3])[(i // 2) % 3]
    m = torch.tensor([0.0, 0.01])[(i // 3) % 2]
    _assert_draws(logits, u, t, k, p, m, rows=list(range(0, rows, max(1, rows // 12))))


@pytest.mark.parametrize("below", [28.0, 30.0, 31.0, 32.0])
def test_sampling_a_long_flat_tail_near_the_last_bit(below):
    """2**18 equal logits some 2**-43 below the largest: a mass is off by at most 2**-45 of the
    largest, so a border by at most vocab * 2**-45."""
    vocab = 1 << 18
    logits = torch.full((vocab,), -below)
    top = vocab // 3
    logits[top] = 0.0
    u = torch.cat([torch.tensor([0.0, 2.0 ** -44, 1 - 2.0 ** -24, 0.5]), torch.exp2(-torch.linspace(24, 32, 60))])
    ids, logp = bridge.b200_sample(logits.cuda().expand(len(u), -1).contiguous(), u.cuda())
    w = torch.exp(logits.double())
    upto, total = torch.cumsum(w, 0), float(w.sum())
    off = vocab * 2.0 ** -45
    for r in range(len(u)):
        token, target = int(ids[r]), float(u[r].double()) * total
        assert float(upto[token] - w[token]) - off <= target <= float(upto[token]) + off
        want = math.log(float(w[token]) / total)
        assert abs(float(logp[r]) - want) <= off + 2.0 ** -23 * abs(want) + 1e-7
