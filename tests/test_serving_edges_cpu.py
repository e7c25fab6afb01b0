"""Refusals of the serving calls and the paged state at the edges of their ranges."""
import ctypes

import pytest
import torch

from tests.test_serving_cpu import E, _batch, _kv, _state, lib  # noqa: F401 (lib is a fixture)

UNSUPPORTED = -3


@pytest.mark.parametrize("sequence", [-1, -3, 3, 100])
def test_a_sequence_that_does_not_exist_is_refused_everywhere(sequence):
    s = _state(pages=20)
    s.batch([0, 1, 2], [17, 5, 33])
    s.advance([0, 1, 2], [17, 5, 33])
    pages, lengths, table = [s.pages_of(b) for b in range(3)], list(s.lengths), s._table.clone()
    for call in (lambda: s.release(sequence), lambda: s.pages_of(sequence), lambda: s.dense(0, [0, sequence]),
                 lambda: s.reserve([sequence], [1]), lambda: s.advance([sequence], [1]),
                 lambda: s.batch([sequence], [1])):
        with pytest.raises(ValueError, match="sequences must be in"):
            call()
    assert [s.pages_of(b) for b in range(3)] == pages and s.lengths == lengths and torch.equal(s._table, table)
    assert s.free_pages == 20 - 6


def test_reservations_and_lengths_that_do_not_fit_are_refused():
    s = _state(pages=20)
    for seqs, counts in (([0, 0], [10, 10]), ([0], [-1]), ([0, 1], [3]), ([], [])):
        for call in (s.reserve, s.advance):
            with pytest.raises(ValueError):
                call(seqs, counts)
    with pytest.raises(ValueError, match="at least one sequence"):
        s.dense(0, [])
    s.reserve([0], [16])
    with pytest.raises(ValueError, match="no pages"):
        s.advance([1, 0], [0, 17])
    assert s.lengths == [0, 0, 0] and s.free_pages == 19
    s.advance([0], [16])
    assert s.lengths == [16, 0, 0]


def test_the_sequences_of_a_step_that_have_tokens():
    s = _state()
    assert s.with_tokens([2, 0, 1], [0, 3, 1]) == ([0, 1], [3, 1]) and s.with_tokens([1], [0]) == ([], [])
    for seqs, counts in (([0, 0], [1, 0]), ([3], [0]), ([0], [-1]), ([0, 1], [1])):
        with pytest.raises(ValueError):
            s.with_tokens(seqs, counts)


def test_attention_in_fp32_refuses_what_it_cannot_take(lib):  # noqa: F811
    def attend(kv=_kv(value=None), q=256, stride=768, out=256, heads=8, scale=0.1, **batch):
        return lib.parrot_paged_attention_f32(ctypes.byref(kv), ctypes.byref(_batch(**batch)), q, stride, out, heads,
                                              0, 0, scale, None, None)
    for kw in (dict(kv=_kv()), dict(kv=_kv(value=None, e4m3=1, key_scale=256))):
        assert attend(**kw) == UNSUPPORTED, kw
    for kw in (dict(q=None), dict(q=8), dict(stride=766), dict(stride=767), dict(out=None), dict(out=4), dict(heads=7),
               dict(scale=0.0), dict(kv=_kv(value=None, page_size=48)), dict(tokens=-1)):
        assert attend(**kw) == E, kw
    assert attend(tokens=0) == 0
