"""Serving through the model, at the edges: what a step reports, and which sequences it runs."""
import pytest
import torch

from parrot_b200 import bridge
from tests.test_model_gpu import TINY, _pair

pytestmark = pytest.mark.gpu


def test_a_step_reports_what_is_out_of_range_in_the_state():
    prod, _ = _pair(TINY, seed=31)
    ids = torch.randint(0, 32768, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    state = prod.paged_state(sequences=2, pages=8, page_size=16)
    prod.extend(ids[:20], [20], state)
    assert state.read_status() == [0, 0, 0, 0]
    good = state._table.clone()
    state._table[0, 0] = 77                       # a page that the pools do not have
    prod.extend(ids[20:21], [1], state)           # read by the kernel for few queries
    assert state.read_status(clear=True)[:3] == [2, 52, 77]
    prod.extend(ids[21:], [19], state)            # and by the one for many
    assert state.read_status(clear=True)[:3] == [2, 52, 77]
    state.dense(0, [0])
    assert state.read_status(clear=True)[:3] == [2, 52, 77]
    state._table = good
    state.release(0)
    state.batch([0], [20])
    state._table[0, 1] = -9                       # written by the append
    prod.extend(ids[:20], [20], state)
    assert state.read_status()[:3] == [2, 52, -9]   # the first entry stays
    assert state.read_status(clear=True)[:3] == [2, 52, -9]
    assert state.read_status() == [0, 0, 0, 0]


def test_the_status_word_of_a_batch_is_the_states():
    prod, _ = _pair(TINY, seed=31)
    state = prod.paged_state(sequences=1, pages=2, page_size=16, kv_dtype=torch.float8_e4m3fn)
    assert state.batch([0], [3]).status.data_ptr() == state.status.data_ptr()
    assert state.status.device.type == "cuda" and bridge.PAGE_SIZES


def test_sequences_without_new_tokens_do_not_change_a_step():
    """Listed beside one long piece they chose the kernel for few tokens a sequence."""
    prod, _ = _pair(TINY, seed=32)
    ids = torch.randint(0, 32768, (200,), generator=torch.Generator().manual_seed(2)).cuda()
    seen = []
    attention = bridge.b200_paged_attention

    def watch(q, kv, page_table, *args, **kw):
        seen.append(page_table.shape[0])
        return attention(q, kv, page_table, *args, **kw)
    states = [prod.paged_state(sequences=120, pages=16, page_size=16) for _ in range(2)]
    alone = prod.extend(ids, [200], states[0], sequences=[5])
    bridge.b200_paged_attention = watch
    try:
        beside = prod.extend(ids, [200 * (b == 5) for b in range(120)], states[1])
    finally:
        bridge.b200_paged_attention = attention
    assert set(seen) == {1} and torch.equal(alone, beside)
    assert states[1].lengths == [200 * (b == 5) for b in range(120)]
    with pytest.raises(ValueError):
        prod.extend(ids[:0], [0, 0], states[1], sequences=[0, 1])
    with pytest.raises(ValueError):
        prod.extend(ids[:1], [1, 0], states[1], sequences=[0, 0])


@pytest.mark.parametrize("pieces", [(1,), (3, 5), (9, 1), (200, 1, 40)])
def test_the_latent_layer_keeps_the_precision_of_the_dense_decode_step(pieces):
    """Over a bf16 cache the absorbed query, the weights and the context are not rounded to bf16.

    Against the formula in 64 bits from the same bf16 inputs, weights and latents: the result's one
    rounding (half a step, 2**-8 relative), and 2**-12 of its terms for the sums in fp32 and the two-part
    products (2**-16 each, times scores of up to 8).  A bf16 query or context would add 2**-8 of a
    context's numbers, which the second assertion holds to a quarter of that over the whole result.
    """
    from parrot_b200 import ModelConfig
    from parrot_b200.model import GlobalMLA, MLALatentCache
    cfg = ModelConfig()
    torch.manual_seed(5)
    layer = GlobalMLA(cfg).to("cuda", torch.bfloat16).eval()
    contexts = [n + 60 for n in pieces]
    with torch.inference_mode():
        for p in layer.parameters():
            p.normal_(0, 0.036)
        aq, ao = (w.double() for w in layer._absorbed())
        state = pm_state(cfg, contexts)
        kv = state.layers[0]
        prefix = [torch.randn(1, 60, cfg.dim, device="cuda").bfloat16() for _ in pieces]
        for b, x in enumerate(prefix):
            layer.extend(x, kv, state.batch([b], [60]), 0)
            state.advance([b], [60])
        x = torch.randn(1, sum(pieces), cfg.dim, device="cuda").bfloat16()
        got = layer.extend(x, kv, state.batch(range(len(pieces)), pieces), 0)[0]
        state.advance(range(len(pieces)), pieces)
        lat, _ = state.dense(0, range(len(pieces)))
        first, err, size = 0, 0.0, 0.0
        for b, n in enumerate(pieces):
            k = lat[b, 0, :contexts[b]].double()
            q = (x[0, first:first + n].double() @ aq.T).view(n, cfg.n_heads, -1)
            z = torch.einsum("thd,sd->hts", q, k) * cfg.head_dim ** -0.5
            assert float(z.abs().max()) < 8
            pos = torch.arange(contexts[b] - n, contexts[b], device="cuda")[:, None]
            z = z.masked_fill(torch.arange(contexts[b], device="cuda")[None] > pos, -float("inf"))
            ctx = torch.einsum("hts,sd->thd", torch.softmax(z, -1), k).reshape(n, -1)
            want = ctx @ ao.T
            terms = ctx.abs() @ ao.abs().T
            off = (got[first:first + n].double() - want).abs()
            assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * terms).all())
            rounded = (want.bfloat16().double() - want)
            err += float((got[first:first + n].double() - want).pow(2).sum())
            size += float(rounded.pow(2).sum())
            # and the dense cache's step gives the last token the same
            cache = MLALatentCache(lat[b:b + 1, 0, :contexts[b]].clone())
            at = torch.full((1,), contexts[b] - 1, device="cuda", dtype=torch.int32)
            dense = layer.decode(x[:, first + n - 1:first + n], cache, contexts[b] - 1, position_device=at)[0, 0]
            assert bool(((dense - got[first + n - 1]).double().abs()
                         <= 2.0 ** -7 * want[-1].abs() + 2.0 ** -11 * terms[-1]).all())
            first += n
        # root mean square: the result's rounding alone, and a quarter of one more at most
        assert err ** 0.5 <= 1.04 * size ** 0.5


@pytest.mark.parametrize("n", [1, 8, 30])
def test_a_latent_layer_of_more_heads_than_a_small_projection_takes(n):
    """16 heads of a latent of 128: 2048 numbers a row, more than b200_linear_small holds."""
    from parrot_b200 import ModelConfig
    from parrot_b200.model import GlobalMLA
    cfg = ModelConfig(n_heads=16, head_dim=32)
    torch.manual_seed(6)
    layer = GlobalMLA(cfg).to("cuda", torch.bfloat16).eval()
    with torch.inference_mode():
        for p in layer.parameters():
            p.normal_(0, 0.036)
        state = pm_state(cfg, [n])
        x = torch.randn(1, n, cfg.dim, device="cuda").bfloat16()
        got = layer.extend(x, state.layers[0], state.batch([0], [n]), 0)[0]
        state.advance([0], [n])
        k = state.dense(0, [0])[0][0, 0].double()
        aq, ao = (w.double() for w in layer._absorbed())
        z = torch.einsum("thd,sd->hts", (x[0].double() @ aq.T).view(n, 16, -1), k) * 32 ** -0.5
        z = z.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -float("inf"))
        ctx = torch.einsum("hts,sd->thd", torch.softmax(z, -1), k).reshape(n, -1)
        want, terms = ctx @ ao.T, ctx.abs() @ ao.abs().T
    # the bound of the test above, its 2**-12 for scores of up to 8 taken by size
    size = 1 + float(z[z > -1e30].abs().max()) / 8
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * size * terms).all())


def pm_state(cfg, contexts):
    from parrot_b200 import PagedState
    return PagedState(cfg, len(contexts), sum(-(-n // 16) for n in contexts), 16, torch.bfloat16, 0, "cuda", [False])
