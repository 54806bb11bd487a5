"""Attention over the quantised KV cache where scores, values and their order are hard to hold: against plain 64-bit arithmetic with
the tolerances of test_gpu_kv_cache.py, unless a test derives its own."""
import math

import pytest
import torch
from test_gpu_kv_cache import DT, FORMS, attention64, check_attn, held, i32, tables

from attention_autotuner_b200 import _lib
from attention_autotuner_b200.arch import B200
from attention_autotuner_b200.ops.attention_interface import flash_attn_func
from attention_autotuner_b200.ops.cache_interface import QuantizedKVCache, kv_cache_attn, kv_cache_read, kv_cache_write

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


@pytest.mark.parametrize("group", [2, 8, 16])
@pytest.mark.parametrize("bits", [4, 8])
def test_values_near_the_largest_of_bf16(bits, group):
    """Finite values whose weighted mean is finite: a few of 1e36, many of up to 3e38 (whose sum is not), rows of one value, and one of 1e36
    that comes first and has lost its weight, among values of 1e-20."""
    d = 64
    g = torch.Generator("cuda").manual_seed(50)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    towards = normal(d)
    for L, make in ((5, lambda: normal(5, d) * 1e36), (3000, lambda: 1e38 * (1 + 2 * torch.rand(3000, d, generator=g, device="cuda"))),
                    (400, lambda: torch.full((400, d), 3e38, device="cuda")), (512, None), (6000, None)):
        k = 0.1 * normal(L, d)
        if make is None:
            v = normal(L, d) * 1e-20
            v[0] = normal(d) * 1e36
            k[:32] -= 200 * towards / towards.norm() ** 2  # 2^-288 of the others' probability
        else:
            v = make()
        q = (towards + 0.05 * normal(1, group, 1, d)).bfloat16()
        k, v = k.bfloat16()[None, None], v.bfloat16()[None, None]
        cache, table = one_sequence(k, v, bits, 64, g)
        o, lse = kv_cache_attn(q, cache, table, i32(L), None, False, 1.0, True)
        want, want_lse, weight = attention64(q, held(k, bits), held(v, bits), i32(L), False, 1.0)
        assert o.isfinite().all()
        check_attn(o, lse, want, want_lse, weight)


@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("bits", [4, 8])
def test_long_sequences_with_values_at_one_end_of_their_range(bits, group):
    """One channel of V lies 40 above the others, so that these have the same few numbers everywhere and their sums grow all the way.
    The accumulators of 1024 positions take 128 products (of 16 positions, in two pieces), each of which may drop less than 2^-23 of a sum
    that grows to half of sum p range at most (numbers are added at even and subtracted at odd positions): 2^-18 of sum p range, here
    2^-18 / 0.54 < 2^-17 of sum p 0.54 range, next to the tolerance of check_attn."""
    L, B, d = 131072, 512, 64  # a head for every CTA: its four warps go over the whole sequence
    g = torch.Generator("cuda").manual_seed(60)
    k = 0.1 * torch.randn(1, 1, L, d, generator=g, device="cuda").half()
    v = torch.randn(1, 1, L, d, generator=g, device="cuda")
    v[..., 3] += 40
    v = v.half()
    cache, table = one_sequence(k, v, bits, 128, g)
    q = torch.randn(B, group, 1, d, generator=g, device="cuda").half()
    o = kv_cache_attn(q, cache, table.expand(B, -1), torch.full((B,), L, dtype=torch.int32, device="cuda"), None, False, d ** -0.5)
    some = q[::171, :, 0].transpose(0, 1)[None]  # [1, group, 3, d]
    want, _, weight = attention64(some, held(k, bits), held(v, bits), i32(L), False, d ** -0.5)
    got = o[::171, :, 0].transpose(0, 1)[None].double()
    size, spread = weight[..., :-1], weight[..., -1:]
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -14 * size + (2.0 ** -17 + 2.0 ** -22) * spread
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


@pytest.mark.parametrize("group", [2, 8, 16])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_values_that_cancel(bits, name, group):
    """Two positions with opposite values and nearly the same probability: the output is a small difference, whose own rounding hides
    nothing of how the probabilities went through the products (in two pieces: 2^-22 of the values; in one: up to 2^-12)."""
    dtype, d, B = DT[name], 128, 40
    g = torch.Generator("cuda").manual_seed(70)
    k = torch.randn(B, 1, 2, d, generator=g, device="cuda").to(dtype)
    v = torch.randn(B, 1, 1, d, generator=g, device="cuda").to(dtype)
    v = torch.cat([v, -v], 2)
    table, pages = tables(g, B, 1)
    cache = QuantizedKVCache(pages, 1, d, bits=bits, page_size=16, dtype=dtype)
    kv_cache_write(cache, k, v, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    q = (0.002 * torch.randn(B, group, 1, d, generator=g, device="cuda")).to(dtype)
    lengths = torch.full((B,), 2, dtype=torch.int32, device="cuda")
    o, lse = kv_cache_attn(q, cache, table, lengths, None, False, 1.0, True)
    want, _, weight = attention64(q, held(k, bits), held(v, bits), lengths, False, 1.0)
    size, spread = weight[..., :-1], weight[..., -1:]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -14 * size + 2.0 ** -22 * spread
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("group", [1, 8, 16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_with_outlying_channels(bits, name, d, group):
    """Sequences of one position, so that lse is the score: one channel of q is 40 to 80 and one of K 200, or of positive K 30, where the
    others are 1, which leaves few numbers for the others. A score is scale (ks sum q n + kz sum q), its products d / 16 sums of 16, each of which may
    drop less than 2^-23 of the largest partial sum, and eight roundings of 2^-24 for the rest, all relative to scale times
    M = sum |q| (n ks + |kz|); exp2 and log2 units add 2^-22 of the score."""
    dtype, B = DT[name], 64
    g = torch.Generator("cuda").manual_seed(80)
    for at, far in ((4, 200.0), (5, 200.0), (10, 30.0), (11, 30.0), (d - 1, 200.0)):  # nibbles of either kind
        q = torch.randn(B, group, 1, d, generator=g, device="cuda")
        q[..., at] = 40 * (1 + torch.rand(B, group, 1, generator=g, device="cuda"))
        k = torch.randn(B, 1, 1, d, generator=g, device="cuda")
        if far < 100:
            k = k.abs()
        k[..., (at + 13) % d] = far
        q, k = q.to(dtype), k.to(dtype)
        table, pages = tables(g, B, 1)
        cache = QuantizedKVCache(pages, 1, d, bits=bits, page_size=16, dtype=dtype)
        kv_cache_write(cache, k, k, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
        one = torch.ones(B, dtype=torch.int32, device="cuda")
        _, lse = kv_cache_attn(q, cache, table, one, None, False, d ** -0.5, True)
        hk = held(k, bits)
        want = (q.double() * hk).sum(-1) * d ** -0.5
        low = hk.amin(-1, keepdim=True)
        size = (q.double().abs() * (hk - low + low.abs())).sum(-1) * d ** -0.5
        tol = (d / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -22 * want.abs()
        assert ((lse.double() - want).abs() <= tol).all(), ((lse.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("bits,d,name", FORMS)
def test_values_read_back_are_rounded_once(bits, d, name):
    """Rows of positive values whose smallest is far below the step: about one product of a scale and a number in 2^8 lies half way between
    two 16-bit values, and the zero decides. Against zero + scale n in 64 bits (exact: 40 bits), rounded half to even by its bits;
    .to(dtype) would round to 32 bits on the way."""
    dtype, L = DT[name], 1000
    g = torch.Generator("cuda").manual_seed(90)
    x = torch.rand(1, 2, L, d, generator=g, device="cuda") * torch.exp2(torch.randint(0, 5, (1, 2, L, 1), generator=g, device="cuda").float()) + 0.5
    x[..., 7] = 2.0 ** (-14 if name == "fp16" else -24) * (1 + torch.rand(1, 2, L, generator=g, device="cuda"))
    x = x.to(dtype)
    cache, table = one_sequence(x, x.flip(1), bits, 64, g)
    k, v = kv_cache_read(cache, table, None, None, L)
    low, high = x.float().amin(-1, keepdim=True), x.float().amax(-1, keepdim=True)
    step = ((high - low) / torch.full_like(low, 2 ** bits - 1)).to(dtype).float()
    n = ((x.float() - low) / step).round().clamp(max=2 ** bits - 1)  # in fp32, as the format has it
    m, e = torch.frexp(low.double() + step.double() * n.double())
    digits = 2 / torch.finfo(dtype).eps
    want = torch.ldexp(torch.round(m * digits) / digits, e)
    assert torch.equal(k.double(), want) and torch.equal(v.double(), want.flip(1))


def test_tables_that_could_hold_more_than_the_kernels_count():
    """Rows of 32767 pages of 65536 positions for 40 sequences of ordinary lengths: several launches, each of which counts in 32 bits, and
    a page that does not exist is reported with its own sequence."""
    B, H, d, page, width = 40, 2, 64, 65536, 32767
    g = torch.Generator("cuda").manual_seed(100)
    L = 70000
    k, v = (torch.randn(2, H, L, d, generator=g, device="cuda").half() for _ in range(2))
    cache = QuantizedKVCache(4, H, d, bits=4, page_size=page)
    two = i32(2, 0, 1, 3).reshape(2, 2)
    kv_cache_write(cache, k, v, two, i32(0, 0))
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = two.repeat(B // 2, 1)
    lengths = torch.tensor([(0, 1, 33, 511, 5000, 65536, 65537, L)[i % 8] for i in range(B)], dtype=torch.int32, device="cuda")
    q = torch.randn(B, 3 * H, 1, d, generator=g, device="cuda").half()
    o, lse = kv_cache_attn(q, cache, table, lengths, None, True, 0.125, True)
    hk, hv = held(k, 4), held(v, 4)
    for b in range(B):
        at = slice(b, b + 1), slice(b % 2, b % 2 + 1)
        check_attn(o[at[0]], lse[at[0]], *attention64(q[at[0]], hk[at[1]], hv[at[1]], lengths[at[0]], True, 0.125))
    assert _lib.kv_status() == 0
    table[33, 0] = 4
    kv_cache_attn(q, cache, table, lengths)
    torch.cuda.synchronize()
    with pytest.raises(_lib.AttnB200Error, match="sequence 33"):
        kv_cache_attn(q, cache, table, lengths)
    assert _lib.kv_status() == 3


@pytest.mark.parametrize("size", [1.0, 2.0 ** 12, 2.0 ** 100])
@pytest.mark.parametrize("group", [1, 8, 16])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_of_any_size(bits, name, group, size):
    """Scores up to 1e10, where a step of fp32 is 1000: the largest takes all, and the output is its value, rounded."""
    if name == "fp16" and size > 2.0 ** 13:
        size = 1 / 4096
    dtype, d, B = DT[name], 128, 100
    g = torch.Generator("cuda").manual_seed(110)
    sign = torch.where(torch.rand(B, 1, 1, d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    q = 6e4 * sign * (0.5 + 0.5 * torch.rand(B, group, 1, d, generator=g, device="cuda"))
    k = 6e4 * sign * torch.tensor([0.2, 1.0, 0.5, -1.0], device="cuda")[:, None] * (0.9 + 0.1 * torch.rand(B, 1, 4, d, generator=g, device="cuda"))
    v = torch.randn(B, 1, 4, d, generator=g, device="cuda") * size
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    table, pages = tables(g, B, 1)
    cache = QuantizedKVCache(pages, 1, d, bits=bits, page_size=16, dtype=dtype)
    kv_cache_write(cache, k, v, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    lengths = torch.full((B,), 4, dtype=torch.int32, device="cuda")
    o, lse = kv_cache_attn(q, cache, table, lengths, None, False, d ** -0.5, True)
    want, want_lse, _ = attention64(q, held(k, bits), held(v, bits), lengths, False, d ** -0.5)
    assert want_lse.min() > 1e9
    hv = held(v, bits)[:, :, 1:2].expand_as(want)
    assert torch.equal(want, hv)
    # the value is put together of scale n and zero, each with a rounding of fp32 (the scale in pieces of 2^-22)
    rng = held(v, bits).amax(-1, keepdim=True)[:, :, 1:2] - held(v, bits).amin(-1, keepdim=True)[:, :, 1:2]
    half = torch.finfo(dtype).eps / 2 * want.abs().clamp(min=torch.finfo(dtype).smallest_normal)
    assert ((o.double() - want).abs() <= half + 2.0 ** -21 * rng).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -18 * want_lse).all()  # 16 products of 2^-23, a few roundings of 2^-24, of scores that do not cancel


def test_lse_of_one_position():
    """The score itself, to 2^-22 of it and of 1: sums of at most 64 products with 14 bits in all, a few of the last ones dropped."""
    d, B = 64, 512
    g = torch.Generator("cuda").manual_seed(120)
    q = torch.randint(-3, 4, (B, 1, 1, d), generator=g, device="cuda").half()
    k = torch.randint(0, 16, (B, 1, 1, d), generator=g, device="cuda").half()  # zero 0 and scale 1 where 0 and 15 occur
    k[..., 0], k[..., 1] = 0, 15
    table, pages = tables(g, B, 1)
    cache = QuantizedKVCache(pages, 1, d, bits=4, page_size=16)
    kv_cache_write(cache, k, k, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    _, lse = kv_cache_attn(q, cache, table, one, None, False, 2.0 ** -6, True)
    want = (q.double() * k.double()).sum(-1) * 2.0 ** -6
    assert ((lse.double() - want).abs() <= 2.0 ** -21 * (1 + want.abs())).all(), (lse.double() - want).abs().max().item()


def test_a_ragged_prompt_goes_on_sequence_by_sequence():
    """70 more positions behind 40 and 100, by flash_attn_func over what is read back of each. Probabilities and values rounded to
    bf16, as in the test of equal lengths."""
    B, H, group, d, new, scale = 2, 2, 4, 128, 70, 128 ** -0.5
    lens = [40, 100]
    g = torch.Generator("cuda").manual_seed(130)
    k, v = (torch.randn(B, H, 170, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(B, H * group, new, d, generator=g, device="cuda").bfloat16()
    table, pages = tables(g, B, 6)
    cache = QuantizedKVCache(pages, H, d, bits=8, page_size=32, dtype=torch.bfloat16)
    kv_cache_write(cache, k, v, table, i32(0, 0), i32(*lens))
    more = [torch.stack([x[b, :, n:n + new] for b, n in enumerate(lens)]) for x in (k, v)]
    kv_cache_write(cache, *more, table, i32(*lens))
    with pytest.raises(ValueError, match="of one length"):
        kv_cache_attn(q, cache, table, i32(*lens) + new, None, True, scale)
    for b, n in enumerate(lens):
        dk, dv = kv_cache_read(cache, table[b:b + 1], length=n + new)
        o = flash_attn_func(q[b:b + 1], dk.repeat_interleave(group, 1), dv.repeat_interleave(group, 1), B200(), True, scale)
        at = slice(b, b + 1), slice(None), slice(0, n + new)
        want, _, weight = attention64(q[b:b + 1], held(k[at], 8), held(v[at], 8), i32(n + new), True, scale)
        assert ((o.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * 2.0 ** -8 * weight[..., :-1]).all()


@pytest.mark.parametrize("group,Lq", [(1, 1), (2, 2), (3, 2), (4, 4)])
@pytest.mark.parametrize("bits,d,name", FORMS)
def test_sums_of_long_shares(bits, d, name, group, Lq):
    """Heads that each lie in a CTA or two, so that a warp goes over several times 1024 positions, with references that rise, values
    whose scales change from position to position, NaN in hidden places, and lengths that end anywhere."""
    dtype, B, L = DT[name], 700, 20000
    g = torch.Generator("cuda").manual_seed(140)
    k, v = (torch.randn(1, 1, L, d, generator=g, device="cuda") for _ in range(2))
    k *= torch.linspace(0.05, 1.5, L, device="cuda")[:, None]
    v *= torch.exp2(torch.randint(-6, 7, (L, 1), generator=g, device="cuda").float())
    k, v = k.to(dtype), v.to(dtype)
    v[:, :, -1] = math.nan
    cache, table = one_sequence(k, v, bits, 64, g)
    q = torch.randn(B, group, Lq, d, generator=g, device="cuda").to(dtype)
    lengths = torch.randint(0, L, (B,), generator=g, device="cuda", dtype=torch.int32)
    lengths[:3] = i32(L - 1, L - 1024, 4096)
    o, lse = kv_cache_attn(q, cache, table.expand(B, -1), lengths, None, True, d ** -0.5, True)
    assert o.isfinite().all()
    hk, hv = held(k, bits), held(v[:, :, :-1], bits)
    for b in (0, 1, 2, 350, 699):
        n = int(lengths[b])
        at = slice(b, b + 1)
        want = attention64(q[at], hk[:, :, :n], hv[:, :, :n], lengths[at], True, d ** -0.5)
        check_attn(o[at], lse[at], *want)
