"""The serving operators at the edges of their ranges, against their formulas in 64 bits."""
import math

import pytest
import torch

from parrot_b200 import bridge
from tests.serving_support import Paged, attention, quantise, starts

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
                                              (120, -100, 60.0)])
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
