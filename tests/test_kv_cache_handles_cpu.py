"""CPU: what a QuantizedKVCache and a KVBatch hand to the kernels follows their tensors: copies, pickles, replaced tensors.
The calls are caught before they reach the library."""
import copy
import ctypes
import io
import pickle

import pytest
import torch


@pytest.fixture
def caught(monkeypatch):
    """Caches may lie on the CPU, and a call only leaves its arguments here."""
    from gemlite_b200 import _lib, kv_cache
    calls = []
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(kv_cache.QuantizedKVCache, "_call", lambda self, fn, a: calls.append(type(a).from_buffer_copy(bytes(a))))
    return calls


def _cache(fmt="fp8", pages=4):
    from gemlite_b200 import QuantizedKVCache
    return QuantizedKVCache(pages, 16, 2, 64, fmt, device="cpu")


def _batch(B=2, P=2):
    from gemlite_b200 import KVBatch
    return KVBatch(torch.zeros((B, P), dtype=torch.int32), torch.zeros(B, dtype=torch.int32))


def _write(cache, batch, n=2):
    k = torch.zeros((n, 2, 64), dtype=torch.bfloat16)
    cache.write(None, k, k, batch)


def _addresses(a):
    return [a.k_codes, a.v_codes, a.k_scales, a.v_scales, a.k_zeros, a.v_zeros]


def _of(cache):
    return [None if t is None else t.data_ptr() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, cache.k_zeros, cache.v_zeros)]


def _saved(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("fmt", ["fp8", "int4"])
@pytest.mark.parametrize("make", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x)), _saved])
def test_copies_go_by_their_own_buffers(lib, caught, fmt, make):
    cache = _cache(fmt)
    other = make(cache)
    _write(cache, _batch()), _write(other, _batch())
    assert _addresses(caught[0]) == _of(cache) and _addresses(caught[1]) == _of(other)
    for mine, its in zip(_of(cache), _of(other)):
        assert mine != its or mine is None
    shared = copy.copy(cache)
    assert _of(shared) == _of(cache) and shared.kv_format == fmt
    assert (other.num_pages, other.page_size, other.n_kv_heads, other.head_dim) == (4, 16, 2, 64)


def test_replaced_buffers_are_checked_and_used(lib, caught):
    cache = _cache()
    cache.k_scales = torch.ones_like(cache.k_scales)
    _write(cache, _batch())
    assert _addresses(caught[-1]) == _of(cache)
    bigger = _cache(pages=9)
    for name in ("k_codes", "v_codes", "k_scales"):
        setattr(cache, name, getattr(bigger, name))
    for call in (lambda: _write(cache, _batch()), lambda: cache.read(_batch().page_table, _batch().ctx_lens),
                 lambda: cache.attend(torch.zeros((2, 2, 64), dtype=torch.bfloat16), _batch())):
        with pytest.raises(ValueError, match="v_scales"):       # 4 pages of scales for 9 pages of codes
            call()
    cache.v_scales = bigger.v_scales
    _write(cache, _batch())
    assert caught[-1].num_pages == 9 and _addresses(caught[-1]) == _of(bigger)
    # memory taken away and given back (the library refuses a null address)
    cache.k_codes.untyped_storage().resize_(0)
    _write(cache, _batch())
    assert caught[-1].k_codes is None
    a = caught[-1]
    assert lib.gl_kv_write(ctypes.byref(a), None) != 0 and b"null" in lib.gl_last_error()


def test_replaced_batch_tensors_are_checked_and_used(lib, caught):
    cache, batch = _cache(), _batch(2, 2)
    batch.page_table = torch.zeros((2, 7), dtype=torch.int32)
    _write(cache, batch)
    assert (caught[-1].max_pages, caught[-1].page_table_stride, caught[-1].page_table) == (7, 7, batch.page_table.data_ptr())
    batch.ctx_lens = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="ctx_lens"):
        _write(cache, batch)
    batch.page_table = torch.zeros((1, 3), dtype=torch.int32)
    _write(cache, batch)
    assert (caught[-1].batch, caught[-1].max_pages) == (1, 3)
    batch.page_table = torch.zeros((1, 3), dtype=torch.int64)
    with pytest.raises(ValueError, match="page_table"):
        _write(cache, batch)
    batch.page_table = torch.zeros((1, 3), dtype=torch.int32)
    batch.q_offsets = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="q_offsets"):
        _write(cache, batch)
    batch.q_offsets, batch.max_new = torch.zeros(2, dtype=torch.int32), 7
    _write(cache, batch)
    assert (caught[-1].q_offsets, caught[-1].max_new) == (batch.q_offsets.data_ptr(), 7)


def test_copies_of_a_batch(lib, caught):
    from gemlite_b200 import KVBatch
    batch = KVBatch(torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32), max_len=20, max_new=1)
    for other in (copy.deepcopy(batch), _saved(batch)):
        _write(_cache(), other)
        a = caught[-1]
        assert (a.page_table, a.lens, a.q_offsets) == (other.page_table.data_ptr(), other.ctx_lens.data_ptr(), other.q_offsets.data_ptr())
        assert other.page_table.data_ptr() != batch.page_table.data_ptr() and (a.max_len, a.max_new) == (20, 1)


def test_a_copy_that_left_the_gpu_is_refused(lib):
    """Loaded onto the CPU, a cache's tensors are no addresses for a kernel: its copy is made as ``from_buffers`` makes one."""
    import gemlite_b200
    shape = (4, 2, 16)
    cpu = [torch.zeros(*shape, 64, dtype=torch.uint8)] * 2 + [torch.zeros(shape)] * 2
    with pytest.raises(RuntimeError, match="CUDA"):
        gemlite_b200.QuantizedKVCache.from_buffers(*cpu)
