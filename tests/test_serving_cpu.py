"""Refusals of the serving operators, and their definitions where no GPU is needed."""
import ctypes

import pytest
import torch

from parrot_b200 import _lib, bridge
from parrot_b200 import build as pbuild
from tests.serving_support import E4M3, dequantise, quantise, sample_row

E = _lib.PARROT_EINVAL


@pytest.fixture(scope="module")
def lib():
    pbuild.build()
    return _lib.load()


def _kv(**kw):
    d = dict(key=256, value=256, key_scale=None, value_scale=None, pages=4, n_kv_heads=2, page_size=64,
             head_dim=96, e4m3=0)
    d.update(kw)
    return _lib.PagedKVStruct(*d.values())


def _batch(**kw):
    d = dict(page_table=256, query_start=256, context_len=256, batch=2, table_width=4, tokens=8)
    d.update(kw)
    return _lib.PagedBatchStruct(*d.values())


def _calls(lib, kv, batch):
    """Each entry point on these structs with otherwise good arguments (never reaching a launch)."""
    kv, batch = ctypes.byref(kv), ctypes.byref(batch)
    return [lib.parrot_paged_append_bf16(kv, batch, 256, 12 * 96, 8, 256, None, None, 0, None, None),
            lib.parrot_paged_gather_bf16(kv, batch, 256, 256, 16, None, None),
            lib.parrot_paged_attention_bf16(kv, batch, 256, 8 * 96, 256, 8, 0, 0, 0.1, None, None)]


@pytest.mark.parametrize("kw", [dict(page_size=48), dict(page_size=8), dict(page_size=512), dict(head_dim=80),
                                dict(head_dim=256), dict(pages=-1), dict(n_kv_heads=0), dict(key=None),
                                dict(key=264), dict(value=8), dict(e4m3=1), dict(e4m3=2),
                                dict(e4m3=1, key_scale=256), dict(key_scale=256),
                                dict(value=None, e4m3=1, key_scale=256, value_scale=256),
                                dict(pages=1 << 25, page_size=256)])
def test_paged_calls_refuse_bad_pools(lib, kw):
    assert all(rc < 0 for rc in _calls(lib, _kv(**kw), _batch()))
    assert lib.parrot_b200_last_error()


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(batch=65536), dict(table_width=-1), dict(tokens=-1),
                                dict(page_table=None), dict(context_len=None), dict(table_width=1 << 30)])
def test_paged_calls_refuse_bad_batches(lib, kw):
    assert all(rc == E for rc in _calls(lib, _kv(), _batch(**kw)))


def test_pools_without_pages_are_refused(lib):
    """They could name nothing to the copy engine."""
    assert all(rc == E for rc in _calls(lib, _kv(pages=0), _batch()))
    for shape in ((0, 2, 64, 96), (3, 0, 64, 96)):
        with pytest.raises(ValueError, match="at least one page"):
            bridge.PagedKV(torch.zeros(shape, dtype=torch.bfloat16))


def test_paged_calls_refuse_bad_arguments(lib):
    kv, batch = ctypes.byref(_kv()), ctypes.byref(_batch())
    latent = ctypes.byref(_kv(value=None))
    no_start = ctypes.byref(_batch(query_start=None))

    def append(k=kv, b=batch, qkv=256, stride=1152, heads=8, q=256, cos=None, sin=None, n=0):
        return lib.parrot_paged_append_bf16(k, b, qkv, stride, heads, q, cos, sin, n, None, None)
    for kw in (dict(b=no_start), dict(qkv=None), dict(qkv=8), dict(stride=1151), dict(stride=1144), dict(heads=-1),
               dict(q=None), dict(q=8), dict(cos=256), dict(sin=256), dict(cos=256, sin=256, n=0),
               dict(cos=8, sin=256, n=5), dict(heads=0, stride=384)):
        assert append(**kw) == E, kw

    def gather(k=kv, key=256, value=256, n=16):
        return lib.parrot_paged_gather_bf16(k, batch, key, value, n, None, None)
    for kw in (dict(key=None), dict(key=8), dict(value=None), dict(n=-1), dict(k=latent)):
        assert gather(**kw) == E, kw

    def attend(b=batch, q=256, stride=768, out=256, heads=8, window=0, sinks=0, scale=0.1):
        return lib.parrot_paged_attention_bf16(kv, b, q, stride, out, heads, window, sinks, scale, None, None)
    for kw in (dict(b=no_start), dict(q=None), dict(q=2), dict(stride=760), dict(stride=772), dict(out=None),
               dict(out=8), dict(heads=7), dict(heads=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attend(**kw) == E, kw
    # nothing to do: no launch
    none = ctypes.byref(_batch(tokens=0))
    assert append(b=none) == 0 and attend(b=none) == 0 and gather(n=0) == 0


def test_sample_refuses_bad_arguments(lib):
    def sample(ids=256, logits=256, f32=0, stride=100, rows=4, vocab=100, u=256, t=1.0, k=0, p=1.0, m=0.0):
        return lib.parrot_sample_rows(ids, None, logits, f32, stride, rows, vocab, u, None, t, None, k, None, p,
                                      None, m, None)
    for kw in (dict(ids=None), dict(logits=None), dict(logits=257), dict(logits=258, f32=1), dict(stride=99),
               dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 19) + 1, stride=1 << 20), dict(u=None), dict(t=-1.0),
               dict(t=float("nan")), dict(k=-1), dict(p=-0.5), dict(m=-0.1), dict(m=1.5), dict(p=float("nan"))):
        assert sample(**kw) == E, kw
    assert sample(rows=0) == 0


def test_paged_kv_refuses_bad_pools():
    def pool(dtype=torch.bfloat16, shape=(3, 2, 64, 96)):
        return torch.zeros(shape, dtype=torch.uint8).to(dtype) if dtype == E4M3 else torch.zeros(shape, dtype=dtype)
    scale = torch.zeros(3, 2, 64, dtype=torch.uint8)
    for args in ((pool(torch.float16),), (pool(shape=(3, 2, 48, 96)),), (pool(shape=(3, 2, 64, 80)),),
                 (pool()[0],), (pool(), pool(shape=(3, 2, 64, 32))), (pool(), pool(E4M3)), (pool(E4M3),),
                 (pool(E4M3), pool(E4M3), scale), (pool(), pool(), scale, scale),
                 (pool(E4M3), None, scale, scale), (pool(E4M3), None, scale[:2]),
                 (pool(E4M3), None, scale.int()), (pool().transpose(0, 1),)):
        with pytest.raises(ValueError):
            bridge.PagedKV(*args)
    kv = bridge.PagedKV(pool(E4M3), None, scale)
    assert (kv.struct.pages, kv.struct.n_kv_heads, kv.struct.page_size, kv.struct.head_dim, kv.struct.e4m3) == \
        (3, 2, 64, 96, 1)
    made = bridge.PagedKV.allocate(5, 2, 32, 64, "cpu", E4M3)
    assert made.value.shape == (5, 2, 32, 64) and made.value_scale.dtype == torch.uint8
    assert bridge.PagedKV.allocate(5, 1, 16, 128, "cpu", latent=True).value is None


def test_serving_calls_refuse_cpu_tensors():
    kv = bridge.PagedKV.allocate(2, 2, 16, 32, "cpu")
    i = torch.zeros(1, dtype=torch.int32)
    start = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 256, dtype=torch.bfloat16)
    with torch.inference_mode():
        with pytest.raises(RuntimeError, match="CUDA"):
            bridge.b200_paged_append(kv, x, i[None], start, i, 4)
        with pytest.raises(RuntimeError, match="CUDA"):
            bridge.b200_paged_gather(kv, i[None], i, 4)
        with pytest.raises(RuntimeError, match="CUDA"):
            bridge.b200_paged_attention(x.view(1, 8, 32), kv, i[None], start, i)
        with pytest.raises(RuntimeError, match="CUDA"):
            bridge.b200_sample(x, torch.zeros(1))


def test_an_8_bit_row_is_within_half_a_step_of_what_was_written():
    """e4m3 keeps 4 bits: half a step is 2**-4 of a number in range, and 2**-10 of the row's scale
    (448 of it is the most) below."""
    x = torch.randn(500, 96) * torch.exp2(torch.randint(-30, 30, (500, 1)).float())
    numbers, byte = quantise(x)
    got, e = dequantise(numbers, byte), byte.double() - 127
    bound = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * torch.exp2(e)[:, None])
    assert bool(((got - x.double()).abs() <= bound).all())
    assert torch.equal(got, got.to(torch.bfloat16).double())
    amax = x.abs().amax(1).double()
    assert bool((amax <= 448 * torch.exp2(e)).all()) and bool((amax > 224 * torch.exp2(e)).all())


def test_the_sampling_definition_on_a_row_by_hand():
    x = torch.tensor([0.0, 2.0, 1.0, 2.0, -1.0])
    w = torch.exp(x - 2)
    assert sample_row(x, 0.0, 1.0, 0, 1.0, 0.0)[0] == 0
    assert sample_row(x, 0.999, 1.0, 0, 1.0, 0.0)[0] == 4
    assert sample_row(x, 0.5, 1.0, 1, 1.0, 0.0)[0] == 1          # equals: the lower index
    assert sample_row(x, 0.5, 1.0, 2, 1.0, 0.0)[0] == 3          # {1, 3}: the border belongs to the next
    assert sample_row(x, 0.9, 1.0, 0, float(1 / w.sum()) - 1e-6, 0.0)[0] == 1
    assert sample_row(x, 0.9, 1.0, 0, float(1 / w.sum()) + 1e-6, 0.0)[0] == 3
    assert sample_row(x, 0.999, 1.0, 0, 1.0, 0.5)[0] == 3


# ---------------------------------------------------------------------------- the paged state
def _state(**kw):
    from parrot_b200 import ModelConfig, PagedState
    cfg = ModelConfig(dim=128, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=32, kv_latent_dim=32, n_experts=8,
                      expert_dim=128, shared_expert_dim=64, window_size=64, max_seq_len=100, global_every=2)
    d = dict(sequences=3, pages=8, page_size=16, kv_dtype=torch.bfloat16, sink_tokens=0)
    d.update(kw)
    return PagedState(cfg, d["sequences"], d["pages"], d["page_size"], d["kv_dtype"], d["sink_tokens"], "cpu",
                      [True, False])


def test_paged_state_hands_out_pages_and_takes_them_back():
    s = _state(kv_dtype=E4M3)
    assert [kv.key.shape for kv in s.layers] == [(8, 2, 16, 32), (8, 1, 16, 32)]
    assert s.layers[0].value is not None and s.layers[1].value is None and s.layers[1].value_scale is None
    b = s.batch([2, 0], [17, 16])
    assert b.tokens == 33 and b.query_start.tolist() == [0, 17, 33] and b.context_len.tolist() == [17, 16]
    assert b.page_table.tolist() == [s.pages_of(2), s.pages_of(0) + [-1]]
    s.advance([2, 0], [17, 16])
    assert s.lengths == [16, 0, 17] and s.free_pages == 5
    b = s.batch([0, 2], [1, 0])
    assert b.page_table.shape == (2, 2) and b.context_len.tolist() == [17, 17]
    s.advance([0, 2], [1, 0])
    owned = s.pages_of(0) + s.pages_of(2)
    assert len(set(owned)) == 4 and s.free_pages == 4
    with pytest.raises(RuntimeError, match="free pages"):
        s.batch([1], [65])
    assert s.free_pages == 4 and s.pages_of(1) == []        # all or none
    s.release(2)
    assert s.free_pages == 6 and s.lengths == [17, 0, 0]
    s.batch([1], [65])
    assert s.free_pages == 1


@pytest.mark.parametrize("seqs,counts", [([0], [101]), ([0, 0], [1, 1]), ([3], [1]), ([-1], [1]), ([0], [0]),
                                         ([0], [-1]), ([0, 1], [1]), ([], [])])
def test_paged_state_refuses_bad_steps(seqs, counts):
    s = _state(pages=20)
    with pytest.raises(ValueError):
        s.batch(seqs, counts)
    assert s.free_pages == 20


@pytest.mark.parametrize("kw", [dict(sequences=0), dict(pages=0), dict(page_size=24), dict(kv_dtype=torch.float16),
                                dict(sink_tokens=-1)])
def test_paged_state_refuses_bad_sizes(kw):
    with pytest.raises(ValueError):
        _state(**kw)


def test_padded_rows_are_few_and_near():
    from parrot_b200.paged import padded_rows
    sizes = [padded_rows(n) for n in range(1, 4097)]
    assert all(n <= p <= n * 1.25 for n, p in enumerate(sizes, 1)) and sizes == sorted(sizes)
    assert len(set(sizes)) <= 16 + 4 * 8 + 1 and padded_rows(4096) == 4096
