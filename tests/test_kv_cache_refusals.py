"""Arguments that the quantised KV cache refuses before anything is launched, without a GPU."""
import ctypes

import pytest
import torch

from attention_autotuner_b200 import _lib
from attention_autotuner_b200.ops.cache_interface import QuantizedKVCache, kv_cache_attn, kv_cache_read, kv_cache_write


@pytest.mark.parametrize("change,text", [
    (dict(bits=3), "bits"), (dict(bits=16), "bits"), (dict(head_dim=96), "head dimension"), (dict(head_dim=512), "head dimension"),
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=1 << 17), "page_size"), (dict(num_pages=0), "pages"),
    (dict(heads=0), "heads"), (dict(heads=65536), "heads"), (dict(dtype=torch.float32), "dtype"), (dict(device="cpu"), "CUDA device"),
    (dict(num_pages=2.0), "integer"), (dict(bits=True), "integer")])
def test_caches_that_cannot_be(change, text):
    with pytest.raises(ValueError, match=text):
        QuantizedKVCache(**{**dict(num_pages=4, heads=2, head_dim=64), **change})


def on_cpu():
    cache = object.__new__(QuantizedKVCache)
    cache.num_pages, cache.heads, cache.head_dim, cache.bits, cache.page_size, cache.dtype = 4, 2, 64, 4, 16, torch.float16
    cache.data = torch.zeros(4, 2, 1, 1152, dtype=torch.uint8)
    cache._form = (4, 64, 0)
    return cache


def test_calls_with_the_wrong_tensors():
    cache, table, n = on_cpu(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x, q = torch.zeros(1, 2, 5, 64).half(), torch.zeros(1, 4, 1, 64).half()
    for call, text in ((lambda: kv_cache_write(cache, x, x[:, :, :1], table, n), "v has shape"),
                       (lambda: kv_cache_write(cache, x.float(), x, table, n), "dtype"),
                       (lambda: kv_cache_write(cache, x, x, table.float(), n), "int32"),
                       (lambda: kv_cache_write(cache, x, x, table, n.long()), "int32"),
                       (lambda: kv_cache_write(cache, x, x, table, n, n[:0]), "count has shape"),
                       (lambda: kv_cache_write(None, x, x, table, n), "QuantizedKVCache"),
                       (lambda: kv_cache_attn(q[:, :3], cache, table, n), "multiple"),
                       (lambda: kv_cache_attn(q.expand(1, 4, 65, 64), cache, table, n), "at most 64"),
                       (lambda: kv_cache_attn(q[0], cache, table, n), "4-d"),
                       (lambda: kv_cache_attn(q, cache, table[:0], n), "not empty"),
                       (lambda: kv_cache_attn(q.expand(3, 4, 1, 64), cache, table, n), "sequences"),
                       (lambda: kv_cache_attn(q, cache, table, n), "not supported"),  # all is right but for the device
                       (lambda: kv_cache_read(cache, table, length=0), "length"),
                       (lambda: kv_cache_read(cache, table, n.short(), length=3), "int32")):
        with pytest.raises(ValueError, match=text):
            call()


def test_the_library_checks_before_it_looks_for_a_device():
    lib = _lib.load_kv()
    assert [lib.attn_b200_kv_block_bytes(b, d) for b, d in ((4, 64), (4, 128), (8, 128), (8, 256), (5, 64), (4, 96))] == [1152, 2176, 4224, 8320, 0, 0]
    good = dict(data=64, num_pages=4, heads=2, page_size=16, head_dim=64, bits=4, dtype=0)
    three = (ctypes.c_longlong * 3)(0, 64, 64)

    def write(table=64, stride=2, width=2, k=64, strides=three, B=1, L=1, **change):
        c = _lib.KVCacheStruct(**{**good, **change})
        return lib.attn_b200_kv_write(ctypes.byref(c), table, stride, width, 64, None, k, strides, 64, three, B, L, None)

    def attn(q=64, ws=64, B=1, group=1, Lq=1, scale=1.0, table_width=2):
        c = _lib.KVCacheStruct(**good)
        return lib.attn_b200_kv_attn(q, ctypes.byref(c), 64, table_width, table_width, 64, 64, None, ws, 0, B, group, Lq, scale, 0, None)

    # no workspace for tables of few positions, nor for sizes that are refused
    c = _lib.KVCacheStruct(**good)
    assert lib.attn_b200_kv_attn_workspace_bytes(ctypes.byref(c), 2, 1, 1, 1) == 0
    assert lib.attn_b200_kv_attn_workspace_bytes(ctypes.byref(c), 200, 0, 1, 1) == 0
    odd = (ctypes.c_longlong * 3)(0, 64, 63)
    for rc in (write(data=None), write(data=72), write(bits=5), write(head_dim=80), write(page_size=24), write(num_pages=0), write(dtype=2),
               write(table=None), write(stride=1), write(width=1 << 28, stride=1 << 28), write(k=None), write(k=66), write(strides=odd),
               write(B=0), write(B=65536), write(L=0), attn(q=None), attn(q=72), attn(ws=72), attn(B=4097), attn(group=0), attn(Lq=65),
               attn(scale=0.0), attn(scale=float("nan"))):
        assert rc in (1, 2), rc
        assert lib.attn_b200_kv_last_error().decode().startswith("kv_")
