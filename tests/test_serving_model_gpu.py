"""The serving operators run together, as ``Parrot.extend`` and ``Parrot.sample`` use them: a ragged batch
over a paged cache against the whole-sequence oracle."""
import pytest
import torch

from parrot_b200 import bridge
from tests.gpu_helpers import cosine
from tests.serving_support import sample_row
from tests.test_model_gpu import TINY, _assert_within_reference, _pair, _reference_bf16

pytestmark = pytest.mark.gpu


def _last_logits(orc, ref, sequences):
    """Logits after each whole sequence: fp32 oracle, and its bf16 execution on the GPU."""
    with torch.inference_mode():
        exp = torch.stack([orc(s[None]).logits[0, -1] for s in sequences])
        r = torch.stack([ref(s[None].cuda()).logits[0, -1] for s in sequences])
    return exp, r


def _router_logits(model):
    return [b.moe.last_trace.logits[-1].float().cpu() for b in model.blocks]


def _open_choices(orc, ref, ids):
    """The oracle's last logits for each router decision at the last token that rounding leaves open.

    The k-th and the next router logit differ by ``margin``.  The reference's bf16 execution is off by
    ``e`` at this token and layer; ours may be off by 1.5 e (the factor of the logits' bound below), so
    the difference of two logits by 3 e: with margin <= 3 e either expert is right, and the outputs of
    the two choices are not close.  The other choice is the oracle's with the runner-up's logit raised
    by just over ``margin``.
    """
    with torch.inference_mode():
        out = [orc(ids[None]).logits[0, -1]]
        own = _router_logits(orc)
        ref(ids[None].cuda())
        near = []
        for layer, (a, b) in enumerate(zip(own, _router_logits(ref))):
            k = orc.blocks[layer].moe.cfg.top_k
            value, index = a.topk(k + 1)
            margin = float(value[k - 1] - value[k])
            if margin <= 3 * float((a - b).abs().max()):
                near.append((layer, int(index[k]), margin))
        for turned in range(1, 1 << len(near)):
            for i, (layer, expert, margin) in enumerate(near):
                if turned >> i & 1:
                    bias = torch.zeros(len(ids), len(own[layer]))
                    bias[-1, expert] = margin * 1.001 + 1e-6
                    orc.blocks[layer].moe.router_bias = bias
            out.append(orc(ids[None]).logits[0, -1])
            for block in orc.blocks:
                block.moe.router_bias = None
    return out


def _assert_rows(logits, orc, ref, sequences, floor):
    """``_assert_within_reference``, each row against the nearest of its open choices."""
    exp, r = _last_logits(orc, ref, sequences)
    assert logits.shape == exp.shape
    nearest = torch.stack([min(_open_choices(orc, ref, s), key=lambda x: float((x - row).norm()))
                           for s, row in zip(sequences, logits.float().cpu())])
    # the reference's own distance from its choice stays what it is
    _assert_within_reference(logits, nearest, r.float().cpu() - exp + nearest, floor)


@pytest.mark.parametrize("residual", ["attnres", "standard"])
@pytest.mark.parametrize("page_size", [16, 64])
def test_extend_in_pieces_matches_the_whole_sequences(residual, page_size):
    prod, orc = _pair(TINY, seed=11, residual=residual)
    ref = _reference_bf16(orc)
    g = torch.Generator().manual_seed(12)
    ids = [torch.randint(0, 32768, (n,), generator=g) for n in (300, 170, 33)]
    state = prod.paged_state(sequences=5, pages=64, page_size=page_size)
    done = [0, 0, 0]
    owner = [4, 0, 2]                                     # any slots, in any order
    steps = [(150, 1, 7), (1, 99, 1), (100, 1, 0), (1, 0, 24), (47, 68, 1), (1, 1, 0)]
    for step in steps:
        new = torch.cat([s[d:d + n] for s, d, n in zip(ids, done, step)])
        logits = prod.extend(new.cuda(), step, state, sequences=owner)
        done = [d + n for d, n in zip(done, step)]
        shown = [s[:d] for s, d, n in zip(ids, done, step) if n]
        _assert_rows(logits, orc, ref, shown, 0.998)
    assert [state.lengths[o] for o in owner] == [300, 170, 33]
    # a released slot starts anew, on pages that others have used
    state.release(4)
    logits = prod.extend(ids[2].cuda(), [33], state, sequences=[4])
    _assert_rows(logits, orc, ref, [ids[2]], 0.998)


def test_extend_on_an_8_bit_cache():
    """The first layer sees the same inputs on either cache: its rows are the bf16 ones to half a step
    of e4m3 (2**-4 relative, 2**-10 of the row's scale below its range; 2**-8 more for the bf16 side's
    own rounding), and a row's scale is at most amax / 224."""
    prod, orc = _pair(TINY, seed=13)
    ids = torch.randint(0, 32768, (260,), generator=torch.Generator().manual_seed(14))
    state = prod.paged_state(sequences=1, pages=20, page_size=16, kv_dtype=torch.float8_e4m3fn)
    exact = prod.paged_state(sequences=1, pages=20, page_size=16)
    for lo, hi in ((0, 200), (200, 259), (259, 260)):
        logits = prod.extend(ids[lo:hi].cuda(), [hi - lo], state)
        plain = prod.extend(ids[lo:hi].cuda(), [hi - lo], exact)
        assert torch.isfinite(logits).all()
    _assert_rows(plain, orc, _reference_bf16(orc), [ids], 0.99)
    with torch.inference_mode():
        for got, want in zip(state.dense(0, [0]), exact.dense(0, [0])):
            got, want = got.double(), want.double()
            step = want.abs().amax(-1, keepdim=True) * (1 + 2.0 ** -8) / 224 * 2.0 ** -10
            assert bool(((got - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + step).all())


def test_sinks_keep_the_first_tokens_in_sight():
    """Behind a window of 128, with and without the first tokens: both run, and differ only once
    the first tokens have left the window."""
    prod, _ = _pair(TINY, seed=15)
    ids = torch.randint(0, 32768, (200,), generator=torch.Generator().manual_seed(16)).cuda()
    states = [prod.paged_state(sequences=1, pages=16, page_size=16, sink_tokens=k) for k in (0, 4)]
    a, b = (prod.extend(ids[:128], [128], s) for s in states)
    assert torch.equal(a, b)
    a, b = (prod.extend(ids[128:], [72], s) for s in states)
    assert not torch.equal(a, b) and cosine(a, b) > 0.9


def test_the_dense_cache_of_a_paged_prompt_decodes_on():
    """A prompt written to pages, read back as a dense cache, and continued by decode_step."""
    from parrot_b200.model import GenerationState, LocalKVCache, MLALatentCache
    prod, orc = _pair(TINY, seed=17)
    ref = _reference_bf16(orc)
    ids = torch.randint(0, 32768, (2, 90), generator=torch.Generator().manual_seed(18))
    state = prod.paged_state(sequences=2, pages=16, page_size=16)
    prod.extend(ids[:, :80].reshape(-1).cuda(), [80, 80], state)
    with torch.inference_mode():
        layers = []
        for i in range(TINY["n_layers"]):
            k, v = state.dense(i, [0, 1], max_len=TINY["max_seq_len"])
            layers.append(MLALatentCache(k[:, 0].contiguous()) if v is None else LocalKVCache(k, v))
        dense = GenerationState(layers, 80, 2, torch.full((1,), 80, device="cuda", dtype=torch.int32))
    for t in range(80, 90):
        logits, dense = prod.decode_step(ids[:, t:t + 1].cuda(), dense)
    _assert_rows(logits[:, 0], orc, ref, list(ids), 0.998)


def test_a_sampled_batch_runs_on_and_is_what_its_random_numbers_say():
    prod, _ = _pair(TINY, seed=19)
    g = torch.Generator().manual_seed(20)
    prompts = [torch.randint(0, 32768, (n,), generator=g) for n in (40, 3, 129)]

    def generate():
        state = prod.paged_state(sequences=3, pages=64, page_size=16, kv_dtype=torch.float8_e4m3fn, sink_tokens=2)
        u = torch.rand(6, 3, generator=torch.Generator().manual_seed(21))
        logits = prod.extend(torch.cat(prompts).cuda(), [40, 3, 129], state)
        out = []
        for i in range(6):
            ids, logp = prod.sample(logits, u[i].cuda(), temperature=0.7, top_k=50, top_p=0.9, min_p=0.001)
            for r in range(3):
                token, want = sample_row(logits[r].cpu(), float(u[i, r]), float(torch.tensor(0.7)), 50,
                                         float(torch.tensor(0.9)), float(torch.tensor(0.001)))
                assert int(ids[r]) == token and abs(float(logp[r]) - want) < 1e-5
            out.append(ids)
            logits = prod.extend(ids[:, 0], [1, 1, 1], state)
        return torch.cat(out, 1)
    assert torch.equal(generate(), generate())


def test_decode_sample_on_the_dense_cache():
    prod, _ = _pair(TINY, seed=22)
    ids = torch.randint(0, 32768, (2, 20), generator=torch.Generator().manual_seed(23))
    logits, state = prod.prefill(ids.cuda())
    u = torch.tensor([0.3, 0.8]).cuda()
    nxt, logp = prod.sample(logits, u)
    drawn, logp, state = prod.decode_sample(nxt, state, u, temperature=0.0)
    assert state.position == 21 and drawn.shape == (2, 1) and not logp.any()
    state2 = prod.prefill(ids.cuda())[1]
    greedy, _ = prod.decode_next(nxt, state2)
    assert torch.equal(drawn, greedy)


def test_extend_refuses_bad_arguments():
    prod, _ = _pair(TINY, seed=24)
    state = prod.paged_state(sequences=2, pages=4, page_size=16)
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    for args in ((ids, [4]), (ids, [5, 1]), (ids[None], [5]), (ids, [5], state, [2])):
        with pytest.raises(ValueError):
            prod.extend(args[0], args[1], state, *(args[3:]))
    with pytest.raises(RuntimeError, match="free pages"):
        prod.extend(torch.zeros(80, dtype=torch.int64, device="cuda"), [80], state)
    with pytest.raises(RuntimeError, match="eval"):
        prod.train().extend(ids, [5], state)
    assert state.lengths == [0, 0] and state.free_pages == 4
    with pytest.raises(RuntimeError, match="inference-only"):
        bridge.b200_sample(torch.zeros(1, 8, device="cuda"), torch.zeros(1, device="cuda"))
