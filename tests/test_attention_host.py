"""Refusals of the attention and append entry points (no GPU needed): every
bad argument returns 0 with a message before any device work."""
import ctypes

import pytest


def _cache(qmv, **kw):
    a = dict(keys=4096, values=8192, ggml_type=1, kv_heads=2, head_dim=64, page_size=16, page_count=4)
    a.update(kw)
    return qmv.PagedCache(**a)


def _batch(qmv, **kw):
    a = dict(query_start=256, length=512, page_table=1024, sequences=1, tokens=1, max_pages=4, max_query=1)
    a.update(kw)
    return qmv.PagedBatch(**a)


def _paged(qmv, cache=None, batch=None, **kw):
    a = dict(ggml_type=1, heads=14, q=4096, q_ld=896, out=65536, out_ld=896)
    a.update(kw)
    qmv.paged_attention(cache or _cache(qmv), batch or _batch(qmv), **a)


def _append(qmv, cache=None, batch=None, **kw):
    a = dict(ggml_type=1, heads=14, q=4096, q_ld=896, k=4096, k_ld=128, v=4096, v_ld=128, rope_base=1e4, q_out=65536, q_out_ld=896)
    a.update(kw)
    qmv.paged_append(cache or _cache(qmv), batch or _batch(qmv), **a)


def _packed(qmv, **kw):
    a = dict(ggml_type=1, heads=14, kv_heads=2, head_dim=64, start=256, sequences=1, tokens=1, q=4096, q_ld=896, k=4096, k_ld=128,
             v=4096, v_ld=128, out=65536, out_ld=896)
    a.update(kw)
    qmv.packed_attention(**a)


CACHE = [
    (dict(ggml_type=30), "does not go with"), (dict(ggml_type=0), "does not go with"), (dict(page_size=8), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=512), "page_size"), (dict(page_count=0), "page_count"),
    (dict(keys=None), "null"), (dict(values=None), "null"), (dict(keys=4104), "aligned"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=4), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"), (dict(position_stride=68), "strides"),
    (dict(page_stride=0), "strides"), (dict(head_stride=-64), "strides"),
]
BATCH = [
    (dict(query_start=None), "null"), (dict(length=None), "null"), (dict(page_table=None), "null"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 30), "max_pages"), (dict(max_query=0), "max_query"), (dict(sequences=-1), "negative"), (dict(tokens=-1), "negative"),
]


@pytest.mark.parametrize("kw,message", CACHE)
@pytest.mark.parametrize("call", [_paged, _append])
def test_cache_refusals(qmv, call, kw, message):
    with pytest.raises(qmv.QmvError, match=message):
        call(qmv, cache=_cache(qmv, **kw))


@pytest.mark.parametrize("kw,message", BATCH)
@pytest.mark.parametrize("call", [_paged, _append])
def test_batch_refusals(qmv, call, kw, message):
    with pytest.raises(qmv.QmvError, match=message):
        call(qmv, batch=_batch(qmv, **kw))


@pytest.mark.parametrize("kw,message", [
    (dict(ggml_type=8), "unsupported type"), (dict(ggml_type=30), "does not go with"), (dict(heads=15), "multiple"), (dict(heads=0), "multiple"),
    (dict(heads=130), "query heads per"), (dict(q=None), "q is null"), (dict(out=None), "out is null"), (dict(q_ld=888), "q_ld"),
    (dict(q_ld=900), "16-byte"), (dict(out=65538), "16-byte"), (dict(out_ld=-896), "out_ld"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
])
def test_paged_refusals(qmv, kw, message):
    with pytest.raises(qmv.QmvError, match=message):
        _paged(qmv, **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(k_ld=64), "k_ld"), (dict(v=4100), "v must start"),
    (dict(q=None), "q is null"), (dict(q_out_ld=64), "q_out_ld"), (dict(rope_base=-1.0), "rope_base"), (dict(rope_base=0.5), "rope_base"),
    (dict(rope_base=float("inf")), "rope_base"), (dict(q_out=4096, q_out_ld=904), "same ld"), (dict(k_out=4096, k_out_ld=136), "same ld"),
])
def test_append_refusals(qmv, kw, message):
    with pytest.raises(qmv.QmvError, match=message):
        _append(qmv, **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(ggml_type=12), "unsupported type"), (dict(head_dim=80), "head_dim"), (dict(kv_heads=3), "multiple"), (dict(start=None), "start is null"),
    (dict(sequences=-1), "negative"), (dict(tokens=-1), "negative"), (dict(k=None), "k is null"), (dict(v_ld=100), "v_ld"),
    (dict(k_ld=132), "16-byte"), (dict(scale=-0.5), "scale"),
])
def test_packed_refusals(qmv, kw, message):
    with pytest.raises(qmv.QmvError, match=message):
        _packed(qmv, **kw)


def test_null_structs_are_refused(qmv):
    lib = qmv.lib()
    assert lib.qmv_paged_attention(None, None, 1, 14, 4096, 896, 65536, 896, 0.0, None) == 0
    assert "cache is null" in qmv.last_error()
    c = _cache(qmv)
    assert lib.qmv_paged_attention(c._ref, None, 1, 14, 4096, 896, 65536, 896, 0.0, None) == 0
    assert "batch is null" in qmv.last_error()
    assert lib.qmv_paged_append(None, None, 1, 14, None, 0, None, 0, None, 0, ctypes.c_float(0.0), None, 0, None, 0, None) == 0


def test_nothing_to_do_is_no_work(qmv):
    """No sequences or no tokens: success, and no device is touched."""
    _paged(qmv, batch=_batch(qmv, sequences=0))
    _paged(qmv, batch=_batch(qmv, tokens=0))
    _append(qmv, batch=_batch(qmv, sequences=0))
    _packed(qmv, sequences=0)
    _packed(qmv, tokens=0)


@pytest.mark.parametrize("page_size", [16, 256])
@pytest.mark.parametrize("call", [_paged, _append])
def test_positions_that_pass_32_bits_once_rounded_are_refused(qmv, call, page_size):
    """A length of 2^31 - 16 keys is a length in 32 bits, but its blocks of 128
    keys are not."""
    for pages in (2 ** 30 // page_size + 1, (2 ** 31 - 16) // page_size):
        with pytest.raises(qmv.QmvError, match="2\\^30 positions"):
            call(qmv, cache=_cache(qmv, page_size=page_size), batch=_batch(qmv, max_pages=pages))
