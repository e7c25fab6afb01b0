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
