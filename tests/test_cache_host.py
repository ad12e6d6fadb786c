"""The cache and the shared-prefix attention without a GPU: what their entry points refuse, and what the Python classes check."""
import ctypes

import pytest
import torch

from pi05_megakernel_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def cache(**change):
    """A well-formed cache; no pointer is ever followed on the host."""
    fields = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, status=0x50000, format=_lib.CACHE_INT8, pages=8, layers=2, page_tokens=64,
                  kv_heads=2, head_dim=128)
    return _lib.Cache(**{**fields, **change})


def rows(**change):
    fields = dict(k=0x60000, v=0x70000, batch_stride=4096, layer_stride=2048, token_stride=256, head_stride=128, table=0x80000, starts=None,
                  counts=None, batch=2, layers=2, tokens=8, layer=0, table_stride=4, table_pages=4)
    return ctypes.byref(_lib.CacheRows(**{**fields, **change}))


def call(**change):
    fields = dict(q=0x60000, out=0x70000, lse=None, q_batch_stride=1024, q_token_stride=1024, q_head_stride=128, out_batch_stride=1024,
                  out_token_stride=1024, out_head_stride=128, prefix_table=0x80000, prefix_valid=None, table=0x90000, lengths=0xa0000, batch=2, tokens=1,
                  q_heads=8, layer=0, prefix_tokens=100, table_stride=4, table_pages=4, causal=1, scale=1.0)
    return ctypes.byref(_lib.SharedCall(**{**fields, **change}))


BAD_CACHES = [dict(k=None), dict(v=None), dict(status=None), dict(k=0x10008), dict(v_scale=0x40004), dict(k_scale=None), dict(format=3), dict(format=-1),
              dict(pages=0), dict(layers=0), dict(page_tokens=8), dict(page_tokens=40), dict(page_tokens=0), dict(kv_heads=0), dict(head_dim=96),
              dict(head_dim=512), dict(pages=1 << 30, page_tokens=1 << 12), dict(status=0x50004)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=[str(c) for c in BAD_CACHES])
def test_bad_caches_are_refused(lib, change):
    c, n, code, where = cache(**change), ctypes.c_size_t(), ctypes.c_int(), ctypes.c_int()
    assert lib.pi05_cache_write(0, c, rows(), None) == _lib.ERR_ARGUMENT
    assert lib.pi05_cache_read(0, c, rows(), None) == _lib.ERR_ARGUMENT
    assert lib.pi05_cache_status(0, c, None, code, where) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_workspace(148, c, 8, 2, 1, n) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(0, c, call(), 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT


BAD_ROWS = [dict(k=None), dict(v=None), dict(table=None), dict(k=0x60008), dict(batch=-1), dict(tokens=-1), dict(layers=-1), dict(layers=3), dict(layer=1),
            dict(layer=-1), dict(token_stride=260), dict(head_stride=4), dict(batch_stride=2), dict(table=0x80002), dict(table_pages=-1),
            dict(table_stride=-1), dict(counts=0x1), dict(starts=0x2), dict(batch=1 << 16), dict(tokens=1 << 30)]


@pytest.mark.parametrize("change", BAD_ROWS, ids=[str(c) for c in BAD_ROWS])
def test_bad_rows_are_refused(lib, change):
    assert lib.pi05_cache_write(0, cache(), rows(**change), None) == _lib.ERR_ARGUMENT
    assert lib.pi05_cache_read(0, cache(), rows(**change), None) == _lib.ERR_ARGUMENT
    assert lib.pi05_cache_write(-1, cache(), rows(), None) == _lib.ERR_ARGUMENT
    assert lib.pi05_cache_write(0, cache(), None, None) == _lib.ERR_ARGUMENT


BAD_CALLS = [dict(q=None), dict(out=None), dict(q=0x60008), dict(out=0x70002), dict(q_heads=0), dict(q_heads=7), dict(layer=2), dict(layer=-1),
             dict(prefix_tokens=-1), dict(prefix_table=None), dict(lengths=None), dict(table_pages=-1), dict(batch=-1), dict(tokens=-1), dict(q_head_stride=4),
             dict(out_token_stride=1), dict(lse=0x3), dict(table=0x90001), dict(prefix_table=0x80002), dict(scale=0.0),
             dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("change", BAD_CALLS, ids=[str(c) for c in BAD_CALLS])
def test_bad_calls_are_refused(lib, change):
    assert lib.pi05_shared_attention(0, cache(), call(**change), 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(0, cache(), None, 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(-1, cache(), call(), 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT


def test_bad_steps_are_refused(lib):
    """Without a handle, and before anything is followed."""
    assert lib.pi05_prefill_step(None, cache(), call(), 0x1000, 0x1000, 0x1000, 0x1000, 1, 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT


def test_workspace(lib):
    """It grows with batch and tokens, holds any smaller call's, and a call refuses one that is too small, not aligned or missing."""
    n, last = ctypes.c_size_t(), 0
    for batch, tokens in ((1, 1), (2, 1), (2, 3), (16, 3), (16, 50), (1024, 50)):
        assert lib.pi05_shared_workspace(148, cache(), 8, batch, tokens, n) == _lib.OK and n.value > last
        last = n.value
    assert lib.pi05_shared_workspace(148, cache(), 8, 1025, 1, n) == _lib.ERR_UNSUPPORTED
    assert lib.pi05_shared_workspace(148, cache(), 8, 1024, 1 << 20, n) == _lib.ERR_UNSUPPORTED
    assert lib.pi05_shared_workspace(148, cache(), 8, 0, 1, n) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_workspace(148, cache(), 9, 1, 1, n) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(0, cache(), call(), None, 1 << 30, None) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(0, cache(), call(), 0x100010, 1 << 30, None) == _lib.ERR_ARGUMENT
    assert lib.pi05_shared_attention(0, cache(), call(batch=1025), 0x100000, 1 << 30, None) == _lib.ERR_UNSUPPORTED


def test_nothing_to_do_is_done(lib):
    """No sequences, tokens or layers: nothing is launched, with or without a GPU."""
    for change in (dict(batch=0), dict(tokens=0), dict(layers=0)):
        assert lib.pi05_cache_write(0, cache(), rows(**change), None) == _lib.OK
        assert lib.pi05_cache_read(0, cache(), rows(**change), None) == _lib.OK
    for change in (dict(batch=0), dict(tokens=0)):
        assert lib.pi05_shared_attention(0, cache(), call(**change), 0x100000, 1 << 30, None) == _lib.OK


def test_without_a_gpu(lib):
    if torch.cuda.is_available():
        pytest.skip("there is a GPU")
    assert lib.pi05_cache_write(0, cache(), rows(), None) == _lib.ERR_NO_DEVICE
    assert lib.pi05_shared_attention(0, cache(), call(), 0x100000, 1 << 30, None) == _lib.ERR_NO_DEVICE
    from pi05_megakernel_b200.cache import KvCache
    with pytest.raises(RuntimeError, match="no CPU path"):
        KvCache(4, 1, 64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        KvCache.wrap(torch.zeros(4, 1, 64, 1, 256), torch.zeros(4, 1, 64, 1, 256))


@pytest.mark.parametrize("change", [dict(format="fp8"), dict(page_tokens=24), dict(page_tokens=0), dict(head_dim=80), dict(pages=0), dict(kv_heads=0)])
def test_python_refuses_a_bad_cache(change):
    from pi05_megakernel_b200.cache import KvCache
    with pytest.raises(ValueError):
        KvCache(**{**dict(pages=4, layers=1, page_tokens=64, kv_heads=1, head_dim=256, format="int8"), **change})


def test_packed_arguments_are_the_structures():
    """The Python classes pack the structures of the header by themselves: same sizes and places."""
    from pi05_megakernel_b200 import cache as C
    from pi05_megakernel_b200 import shared as S
    for packed, fields in ((C.ROWS, _lib.CacheRows), (S.CALL, _lib.SharedCall)):
        assert packed.size == ctypes.sizeof(fields)
        values = [i + 1 for i in range(len(fields._fields_))]
        raw = packed.pack(*values)
        got = fields.from_buffer_copy(raw)
        assert [getattr(got, name) for name, _ in fields._fields_] == values


def test_error_string_of_a_page_table(lib):
    assert b"page" in lib.pi05_error_string(_lib.ERR_PAGE_TABLE)


def test_places_of_keys_stay_in_32_bits(lib):
    """A prefix or a table of more than 2^30 tokens, whose whole tiles would pass the end of an int, is refused before a device is asked for."""
    for change in (dict(prefix_tokens=(1 << 30) + 1), dict(prefix_tokens=(1 << 31) - 1), dict(table_pages=(1 << 24) + 1), dict(table_pages=(1 << 31) - 1)):
        assert lib.pi05_shared_attention(0, cache(), call(**change), 0x100000, 1 << 40, None) == _lib.ERR_UNSUPPORTED
