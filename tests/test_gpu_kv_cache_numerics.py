"""Attention over the quantised KV cache where scores, values and their order are hard to hold: against plain 64-bit arithmetic with
the tolerances of test_gpu_kv_cache.py, unless a test derives its own."""
import math

import pytest
import torch
from test_gpu_kv_cache import DT, attention64, check_attn, held, i32, tables

from attention_autotuner_b200.ops.cache_interface import QuantizedKVCache, kv_cache_attn, kv_cache_write

pytestmark = pytest.mark.gpu


def one_sequence(k, v, bits, page, g):
    """A cache that holds k, v [1, H, L, d], and its table."""
    _, H, L, d = k.shape
    table, pages = tables(g, 1, -(-L // page))
    cache = QuantizedKVCache(pages, H, d, bits=bits, page_size=page, dtype=k.dtype)
    kv_cache_write(cache, k, v, table, i32(0))
    return cache, table


@pytest.mark.parametrize("shape", ["step", "slope", "even"])
@pytest.mark.parametrize("group", [2, 8, 16])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_rise_while_values_fall(bits, name, group, shape):
    """The position with the largest value comes first and has lost its weight when the reference of the exponentials has risen:
    at one blow, step by step with it, or in step, so that every position contributes as much."""
    dtype, d = DT[name], 64
    up, down = (12.0, -12.0) if name == "fp16" else (40.0, -4.0)
    for L in (512, 6000):
        g = torch.Generator("cuda").manual_seed(40 + L)
        x = torch.linspace(0, 1, L, device="cuda")
        if shape == "step":
            score, size = torch.where(x < 32 / L, -42.0, 0.0), torch.where(x == 0, up, down)
        else:
            size = up + (down - up) * x
            score = -42.0 * (1 - x) if shape == "slope" else -size * math.log(2)
        towards = torch.randn(d, generator=g, device="cuda")
        q = (towards + 0.05 * torch.randn(1, group, 1, d, generator=g, device="cuda")).to(dtype)
        k = (score[:, None] * towards / towards.norm() ** 2 + 0.02 * torch.randn(L, d, generator=g, device="cuda")).to(dtype)[None, None]
        v = (torch.randn(L, d, generator=g, device="cuda") * torch.exp2(size)[:, None]).to(dtype)[None, None]
        for order in (1, -1):
            kk, vv = (k, v) if order > 0 else (k.flip(2), v.flip(2))
            cache, table = one_sequence(kk, vv, bits, 64, g)
            o, lse = kv_cache_attn(q, cache, table, i32(L), None, False, 1.0, True)
            check_attn(o, lse, *attention64(q, held(kk, bits), held(vv, bits), i32(L), False, 1.0))
