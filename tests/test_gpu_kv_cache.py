"""The quantised KV cache (csrc/kv/, ops/cache_interface.py) against plain 64-bit arithmetic: what is written and read back bit
for bit, attention within the rounding of its output and of the probabilities.

Tolerance of attention, per element: half a step of the output type; bf16 outputs take a probability times a scale as one fp16 number
(half a step, 2^-11), fp16 outputs as two (2^-22), and that goes with numbers counted from the middle: at most 128 of 255 or 8 of 15
steps, 0.54 of the range of the row of V. The rest is fp32: scores of the sizes here (sums of at most 256 products below 2^6 in all)
are off by less than 2^-15, so each probability by as much of itself, and by that of the sum that they are divided by."""
import math

import pytest
import torch

from attention_autotuner_b200 import _lib
from attention_autotuner_b200.arch import B200
from attention_autotuner_b200.ops.attention_interface import flash_attn_func
from attention_autotuner_b200.ops.cache_interface import QuantizedKVCache, kv_cache_attn, kv_cache_read, kv_cache_write

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
FORMS = [(bits, d, name) for bits in (4, 8) for d in (64, 128, 256) for name in ("fp16", "bf16")]


def held(x, bits):
    """The values that a cache holds for the rows of x, in 64 bits (not rounded to its type)."""
    f = x.double()
    top = 2 ** bits - 1
    low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    step = ((high - low).float() / torch.full_like(low, top).float()).to(x.dtype).double()
    n = torch.where(step > 0, torch.round((f - low) / torch.where(step > 0, step, torch.ones_like(step))), torch.zeros_like(f))
    return low + step * n.clamp(max=top)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(seed, B, H, L, d, dtype):
    g = torch.Generator("cuda").manual_seed(seed)
    k = torch.randn(B, H, L, d, generator=g, device="cuda") + torch.randn(H, 1, d, generator=g, device="cuda")
    v = torch.randn(B, H, L, d, generator=g, device="cuda")
    return k.to(dtype), v.to(dtype), g


def tables(g, B, width, extra=3):
    """Pages of B sequences in no order, out of B * width + extra."""
    order = torch.randperm(B * width + extra, generator=g, device="cuda")[: B * width]
    return order.reshape(B, width).to(torch.int32).contiguous(), B * width + extra


def attention64(q, k, v, lengths, causal, scale):
    """o, lse and, behind one another, sum p |v| and sum p 0.54 range(v) in 64 bits; k, v [B, H, L, d] as held."""
    B, Hq, Lq, d = q.shape
    L, group = k.shape[2], Hq // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = q.double() @ kk.transpose(-1, -2) * scale
    i, j = torch.arange(Lq, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
    n = lengths.long()[:, None, None, None]
    seen = j < n
    if causal:
        seen = seen & (j <= i + n - Lq)
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    clean = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
    return p @ clean, lse, torch.cat([p @ clean.abs(), p @ (0.54 * (clean.amax(-1, keepdim=True) - clean.amin(-1, keepdim=True)))], -1)


def check_attn(o, lse, want, want_lse, weight):
    size, spread = weight[..., :-1], weight[..., -1:]
    tol = torch.finfo(o.dtype).eps / 2 * want.abs().clamp(min=torch.finfo(o.dtype).smallest_normal) + 2.0 ** -14 * size + (2.0 ** -11 if o.dtype == torch.bfloat16 else 2.0 ** -22) * spread
    bad = (o.double() - want).abs() > tol
    assert not bad.any(), ((o.double() - want).abs() / tol).max().item()
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and (o[none] == 0).all()
    assert (lse.double() - want_lse)[~none].abs().max().item() < 2.0 ** -12 if (~none).any() else True


def filled(seed, B, H, L, d, bits, page, dtype, lengths, junk=True):
    """A cache with L positions of B sequences, of which lengths count; every byte that was not written is 0xff (a NaN as a scale)."""
    k, v, g = make(seed, B, H, L, d, dtype)
    width = -(-L // page)
    table, pages = tables(g, B, width)
    cache = QuantizedKVCache(pages, H, d, bits=bits, page_size=page, dtype=dtype)
    if junk:
        cache.data.fill_(255)
    kv_cache_write(cache, k, v, table, torch.zeros_like(lengths), lengths)
    return cache, table, held(k, bits), held(v, bits), g


# ------------------------------------------------------------------------------------------------ writing and reading back
@pytest.mark.parametrize("bits,d,name", FORMS)
def test_written_positions_read_back_bit_for_bit(bits, d, name):
    """Ragged starts and counts, also inside a block of 16 and across pages; everything else stays as it was."""
    dtype, B, H, L, page = DT[name], 5, 3, 75, 16 if d == 64 else 64
    k, v, g = make(1, B, H, L, d, dtype)
    old_k, old_v, _ = make(2, B, H, 192, d, dtype)
    width = 192 // page
    table, pages = tables(g, B, width)
    cache = QuantizedKVCache(pages, H, d, bits=bits, page_size=page, dtype=dtype)
    every, zero = i32(*[192] * B), i32(*[0] * B)
    kv_cache_write(cache, old_k, old_v, table, zero)
    start, count = [0, 1, 15, 64, 117], [75, 74, 1, 0, 75]
    kv_cache_write(cache, k, v, table, i32(*start), i32(*count))
    want = []
    for x, old in ((k, old_k), (v, old_v)):
        full, new = held(old, bits), held(x, bits)
        for b in range(B):
            full[b, :, start[b]:start[b] + count[b]] = new[b, :, :count[b]]
        want.append(full.to(dtype))
    got = kv_cache_read(cache, table, zero, every, 192)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a window of it; rows behind the count are zeros
    gk, gv = kv_cache_read(cache, table, i32(*start), i32(*count), 80)
    for b in range(B):
        for have, w in ((gk, want[0]), (gv, want[1])):
            assert torch.equal(have[b, :, :count[b]], w[b, :, start[b]:start[b] + count[b]]) and (have[b, :, count[b]:] == 0).all()
    # without starts and counts
    assert torch.equal(kv_cache_read(cache, table, length=33)[0], want[0][:, :, :33])
    assert _lib.kv_status() == 0


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("name", ["fp16", "bf16"])
def test_rows_that_are_hard_to_hold(bits, name):
    dtype, d = DT[name], 128
    tiny = float(torch.finfo(dtype).smallest_normal)
    big = 6.0e4 if name == "fp16" else 1.0e38
    rows = torch.randn(12, d, generator=torch.Generator().manual_seed(5)).to(dtype)
    rows[0] = 0.75                     # one value: exact
    rows[1] = 0.0
    rows[2] = -0.0
    rows[3] = rows[3].float().mul(tiny).to(dtype)  # a scale that is subnormal, or zero
    rows[4] = torch.linspace(-big, big, d).to(dtype)
    rows[5, 7] = math.inf
    rows[6, 127] = -math.inf
    rows[7, 0] = math.nan
    rows[8] = torch.arange(d).to(dtype)            # ties: 127 / 15 and 127 / 255 steps
    rows[9] = (torch.arange(d) % 31).float().mul(0.5).to(dtype)  # range 15: a scale of 1, every other value half way
    rows[10] = rows[10] * 1e-3 + 100
    x = rows.cuda()[None, None]
    cache = QuantizedKVCache(2, 1, d, bits=bits, page_size=16, dtype=dtype)
    kv_cache_write(cache, x, x.flip(2), i32(1).reshape(1, 1), i32(2))
    k, v = kv_cache_read(cache, i32(1).reshape(1, 1), i32(2), None, 12)
    want = held(x, bits).to(dtype)
    for r in (5, 6, 7):
        want[0, 0, r] = math.nan
    same = (k == want) | (k.isnan() & want.isnan())
    assert same.all(), same.all(-1)
    assert torch.equal(k.isnan(), v.flip(2).isnan()) and torch.equal(k.nan_to_num(1.0), v.flip(2).nan_to_num(1.0))


@pytest.mark.parametrize("L", [1, 37])
def test_any_strides(L):
    """Projections laid out [B, L, H, d], one row for all heads, and views that start at odd elements."""
    B, H, d = 3, 4, 64
    g = torch.Generator("cuda").manual_seed(9)
    x = torch.randn(B, L, 2, H, d, generator=g, device="cuda").half()
    odd = torch.randn(B * H * L * d + 1, generator=g, device="cuda").half()[1:].reshape(B, H, L, d)
    wide = torch.randn(B, H, L, 2 * d, generator=g, device="cuda").half()[..., ::2]
    table, pages = tables(g, B, 4)
    for k, v in ((x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)), (x[:, :, 0, :1].transpose(1, 2).expand(B, H, L, d), odd), (wide, wide)):
        cache = QuantizedKVCache(pages, H, d, bits=4, page_size=16)
        kv_cache_write(cache, k, v, table, i32(0, 5, 20))
        gk, gv = kv_cache_read(cache, table, i32(0, 5, 20), None, L)
        assert torch.equal(gk, held(k, 4).half()) and torch.equal(gv, held(v, 4).half())
    # tables and lengths that are slices of something wider
    big = torch.full((B, 9), -1, dtype=torch.int32, device="cuda")
    big[:, 2:6] = table
    start = torch.stack([i32(0, 5, 20), i32(7, 7, 7)], 1)[:, 0]
    assert torch.equal(kv_cache_read(cache, big[:, 2:6], start, None, L)[0], gk)


# ------------------------------------------------------------------------------------------------ attention
# B, Hkv, group, Lq, causal, page, lengths: none, one, one short of, exactly and one past a block, a unit, a page; more queries
# than positions (rows that see nothing under the causal mask); every number of rows per pass; heads in one run and in many
ATTN = [
    (8, 2, 1, 1, False, 16, (0, 1, 15, 16, 17, 31, 32, 33)),
    (8, 1, 4, 1, True, 64, (63, 64, 65, 127, 128, 129, 1, 0)),
    (4, 2, 5, 1, False, 32, (100, 0, 257, 3)),
    (3, 3, 8, 1, True, 128, (511, 512, 77)),
    (4, 2, 1, 4, True, 16, (2, 4, 70, 35)),
    (3, 1, 3, 5, True, 32, (5, 1, 999)),
    (2, 2, 2, 8, True, 64, (8, 600)),
    (2, 1, 16, 3, True, 16, (40, 2)),
    (1, 1, 7, 64, True, 64, (200,)),
    (2, 1, 1, 33, False, 64, (129, 5)),
    (1, 2, 4, 1, False, 16, (5000,)),
    (2, 1, 8, 2, True, 64, (9001, 33)),
    (1, 1, 1, 1, False, 128, (30000,)),
    (19, 1, 16, 1, False, 64, (20, 0, 3) * 5 + (20000, 1, 2, 700)),
]


@pytest.mark.parametrize("bits,d,name", FORMS)
def test_attention_matches_64_bits(bits, d, name):
    dtype = DT[name]
    for i, (B, H, group, Lq, causal, page, lens) in enumerate(ATTN):
        L, lengths = max(lens), i32(*lens)
        cache, table, k, v, g = filled(20 + i, B, H, L, d, bits, page, dtype, lengths)
        q = torch.randn(B, H * group, Lq, d, generator=g, device="cuda").to(dtype)
        o, lse = kv_cache_attn(q, cache, table, lengths, B200(), causal, d ** -0.5, return_lse=True)
        check_attn(o, lse, *attention64(q, k, v, lengths, causal, d ** -0.5))
        assert torch.equal(o, kv_cache_attn(q, cache, table, lengths, B200(), causal, d ** -0.5))  # no lse, the same bits
    assert _lib.kv_status() == 0


@pytest.mark.parametrize("B", [33, 130, 1100, 4096])
def test_large_batches(B):
    """The search for a unit's sequence in steps of 32 and 1024; a third of the sequences are empty, one is long."""
    g = torch.Generator("cuda").manual_seed(B)
    lengths = torch.randint(0, 40, (B,), generator=g, device="cuda", dtype=torch.int32) * (torch.arange(B, device="cuda") % 3 > 0)
    lengths[B // 2] = 700
    k, v, _ = make(B, B, 1, 48, 64, torch.float16)
    table = torch.arange(B * 3, device="cuda", dtype=torch.int32).reshape(B, 3).repeat(1, 15)  # positions repeat after 48
    cache = QuantizedKVCache(3 * B, 1, 64, bits=4, page_size=16)
    kv_cache_write(cache, k, v, table, torch.zeros_like(lengths))
    q = torch.randn(B, 2, 1, 64, generator=g, device="cuda").half()
    o, lse = kv_cache_attn(q, cache, table, lengths.int(), return_lse=True)
    hk, hv = held(k, 4), held(v, 4)
    check_attn(o, lse, *attention64(q, hk.repeat(1, 1, 15, 1), hv.repeat(1, 1, 15, 1), lengths, False, 0.125))


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_growing_peaks_and_scales(bits, name):
    """Scores that grow along the keys move the reference at every unit; scales of V from 2^-10 to 2^12 move theirs. Queries of
    very different sizes, one of them zero, share a tile."""
    dtype, L, d = DT[name], 1500, 128
    k, v, g = make(3, 1, 2, L, d, dtype)
    k = (k.float() * torch.linspace(0.05, 3.0, L, device="cuda")[:, None]).to(dtype)
    v = (v.float() * torch.exp2(torch.linspace(-10, 12, L, device="cuda"))[:, None]).to(dtype)
    table, pages = tables(g, 1, 24)
    cache = QuantizedKVCache(pages, 2, d, bits=bits, page_size=64, dtype=dtype)
    kv_cache_write(cache, k, v, table, i32(0))
    for group, order in ((4, 1), (4, -1), (8, 1)):
        q = torch.randn(1, 2 * group, 1, d, generator=g, device="cuda") * torch.tensor([1.0, 1e-3, 0.0, 4.0] * (group // 2), device="cuda")[None, :, None, None]
        q = q.to(dtype)
        if order < 0:  # the peak comes first, and most of what follows is small against it
            kv_cache_write(cache, k.flip(2), v.flip(2), table, i32(0))
        o, lse = kv_cache_attn(q, cache, table, i32(L), None, False, d ** -0.5, True)
        hk, hv = (held(x.flip(2) if order < 0 else x, bits) for x in (k, v))
        want, want_lse, weight = attention64(q, hk, hv, i32(L), False, d ** -0.5)
        check_attn(o, lse, want, want_lse, weight)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("group", [2, 8])
def test_large_values_without_weight(bits, group):
    """Values 2^40 times the others in a place that one of two queries does not see, and where the probability is 2^-60: what is
    left of the row is as exact as without them."""
    d, L = 64, 300
    k, v, g = make(17, 1, 1, L, d, torch.bfloat16)
    q = torch.randn(1, group, 2, d, generator=g, device="cuda").bfloat16()
    v[:, :, L - 1] *= 2.0 ** 40                                     # the last position: query 0 does not see it
    k[:, :, 100] = (-30 * q[0, 0, 0] / q[0, 0, 0].float().norm()).bfloat16()  # query 0 of head 0: a score far below the others
    v[:, :, 100] *= 2.0 ** 40
    cache = QuantizedKVCache(5, 1, d, bits=bits, page_size=64, dtype=torch.bfloat16)
    table = i32(3, 1, 4, 0, 2).reshape(1, 5)
    kv_cache_write(cache, k, v, table, i32(0))
    o, lse = kv_cache_attn(q, cache, table, i32(L), None, True, 1.0, True)
    want, want_lse, weight = attention64(q, held(k, bits), held(v, bits), i32(L), True, 1.0)
    check_attn(o[:, :1, :1], lse[:, :1, :1], want[:, :1, :1], want_lse[:, :1, :1], weight[:, :1, :1])
    check_attn(o, lse, want, want_lse, weight)


def test_values_beyond_the_range_of_fp16():
    """bf16 keys, values and queries of 2^-60 and 2^60: scales and zeros are applied in fp32."""
    for up in (-60, 60):
        k, v, g = make(4, 1, 1, 300, 64, torch.bfloat16)
        q = torch.randn(1, 4, 1, 64, generator=g, device="cuda").bfloat16()
        k2, v2, q2 = (x.float().mul(2.0 ** u).bfloat16() for x, u in ((k, up), (v, -up), (q, -up)))
        out = []
        for kk, vv, qq in ((k, v, q), (k2, v2, q2)):
            cache = QuantizedKVCache(5, 1, 64, bits=4, page_size=64, dtype=torch.bfloat16)
            table = i32(4, 2, 0, 1, 3).reshape(1, 5)
            kv_cache_write(cache, kk, vv, table, i32(0))
            out.append(kv_cache_attn(qq, cache, table, i32(300)))
        assert torch.equal(out[0].float().mul(2.0 ** -up), out[1].float())  # powers of two: the same numbers


@pytest.mark.parametrize("group", [2, 8])
def test_infinities_and_nan_stay_where_they_are_seen(group):
    """A position that holds NaN takes the rows that see it and no other; in hidden places and behind the length it has no effect."""
    d, H, L, Lq = 64, 2, 70, 3
    cache, table, k, v, g = filled(31, 2, H, L, d, 4, 16, torch.float16, i32(L, L))
    q = torch.randn(2, H * group, Lq, d, generator=g, device="cuda").half()
    clean = kv_cache_attn(q, cache, table, i32(L, L), None, True)
    bad = torch.full((2, H, 1, d), math.nan, device="cuda").half()
    fine = torch.randn(2, H, 1, d, generator=g, device="cuda").half()
    kv_cache_write(cache, bad, fine, table, i32(L - 2, L - 2), i32(1, 0))  # K of position 68 of sequence 0: queries 1 and 2 see it
    o = kv_cache_attn(q, cache, table, i32(L, L), None, True)
    assert torch.equal(o[:, :, 0], clean[:, :, 0]) and torch.equal(o[1], clean[1]) and o[0, :, 1:].isnan().all()
    kv_cache_write(cache, fine, bad * math.inf, table, i32(L - 2, L - 2), i32(1, 0))  # and V
    o = kv_cache_attn(q, cache, table, i32(L, L), None, True)
    assert torch.equal(o[:, :, 0], clean[:, :, 0]) and torch.equal(o[1], clean[1]) and o[0, :, 1:].isnan().all()
    short = kv_cache_attn(q, cache, table, i32(L - 2, L - 2), None, False)
    assert short.isfinite().all()
    qbad = q.clone()
    qbad[0, 0, 1, 5] = math.inf
    o = kv_cache_attn(qbad, cache, table, i32(L - 2, L - 2), None, False)
    assert o[0, 0, 1].isnan().all()
    qbad[0, 0, 1] = q[0, 0, 1]
    o[0, 0, 1] = short[0, 0, 1]
    assert torch.equal(o, short)


def test_offsets_past_32_bits():
    """Pages behind 4 GB of a cache, read by several sequences at once."""
    page, d, H = 128, 128, 8
    per_page = H * page // 16 * 4224
    pages = (9 << 29) // per_page + 2
    cache = QuantizedKVCache(pages, H, d, bits=8, page_size=page)
    k, v, g = make(6, 2, H, 200, d, torch.float16)
    table = i32(pages - 1, 0, pages - 2, 1).reshape(2, 2)
    kv_cache_write(cache, k, v, table, i32(0, 0))
    gk, gv = kv_cache_read(cache, table, None, None, 200)
    assert torch.equal(gk, held(k, 8).half()) and torch.equal(gv, held(v, 8).half())
    q = torch.randn(3, H, 1, d, generator=g, device="cuda").half()
    three = torch.cat([table, table[:1]])  # the first sequence twice
    lengths = i32(200, 130, 200)
    o, lse = kv_cache_attn(q, cache, three, lengths, None, False, d ** -0.5, True)
    pick = torch.tensor([0, 1, 0], device="cuda")
    check_attn(o, lse, *attention64(q, held(k, 8)[pick], held(v, 8)[pick], lengths, False, d ** -0.5))


# ------------------------------------------------------------------------------------------------ as a program uses them
def test_a_prompt_its_continuation_and_decoding():
    """A prompt in two pieces, the second with dense attention over what is read back; then tokens one by one, and a draft."""
    B, H, group, d, page, dtype, scale = 3, 2, 4, 128, 16, torch.bfloat16, 128 ** -0.5
    k, v, g = make(8, B, H, 100, d, dtype)
    q = torch.randn(B, H * group, 100, d, generator=g, device="cuda").to(dtype)
    table, pages = tables(g, B, 7)
    cache = QuantizedKVCache(pages, H, d, bits=8, page_size=page, dtype=dtype)
    cache.data.fill_(255)
    hk, hv = held(k, 8), held(v, 8)
    zero = i32(0, 0, 0)
    kv_cache_write(cache, k[:, :, :60], v[:, :, :60], table, zero)
    kv_cache_write(cache, k[:, :, 60:90], v[:, :, 60:90], table, zero + 60)
    dk, dv = kv_cache_read(cache, table, None, None, 90)
    o = flash_attn_func(q[:, :, 60:90], dk.repeat_interleave(group, 1), dv.repeat_interleave(group, 1), B200(), True, scale)
    want, _, weight = attention64(q[:, :, 60:90], hk[:, :, :90], hv[:, :, :90], zero + 90, True, scale)
    assert ((o.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * 2.0 ** -8 * weight[..., :-1]).all()  # P and the values rounded to bf16
    for n in range(90, 96):
        kv_cache_write(cache, k[:, :, n:n + 1], v[:, :, n:n + 1], table, zero + n)
        o, lse = kv_cache_attn(q[:, :, n:n + 1], cache, table, zero + n + 1, B200(), True, scale, True)
        check_attn(o, lse, *attention64(q[:, :, n:n + 1], hk[:, :, :n + 1], hv[:, :, :n + 1], zero + n + 1, True, scale))
    kv_cache_write(cache, k[:, :, 96:], v[:, :, 96:], table, zero + 96)
    o, lse = kv_cache_attn(q[:, :, 96:], cache, table, zero + 100, B200(), True, scale, True)
    check_attn(o, lse, *attention64(q[:, :, 96:], hk, hv, zero + 100, True, scale))


def test_captured_steps_see_new_tables_and_lengths():
    """Two graphs over one cache, each with the workspace of its capture, replayed with other values and side by side."""
    B, H, d, page = 4, 2, 64, 16
    k, v, g = make(12, B, H, 400, d, torch.float16)
    table, pages = tables(g, B, 25)
    cache = QuantizedKVCache(pages, H, d, bits=4, page_size=page)
    kv_cache_write(cache, k, v, table, i32(0, 0, 0, 0))
    hk, hv = held(k, 4), held(v, 4)
    q = torch.randn(B, 4 * H, 1, d, generator=g, device="cuda").half()
    new = torch.randn(B, H, 1, d, generator=g, device="cuda").half()
    lengths, tab = i32(10, 0, 399, 1), table.clone()
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            kv_cache_attn(q, cache, tab, lengths)  # first call outside the capture
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(kv_cache_attn(q, cache, tab, lengths, return_lse=True))
            graphs.append(graph)
    torch.cuda.synchronize()
    for lens in ((10, 0, 399, 1), (400, 400, 400, 400), (0, 0, 0, 0), (17, 33, 1, 250)):
        lengths.copy_(i32(*lens))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = attention64(q, hk, hv, lengths, False, 0.125)
        for o, lse in outs:
            check_attn(o, lse, *want)
    # other pages in the table; and a captured write
    tab.copy_(table.flip(0))
    lengths.copy_(i32(300, 300, 300, 300))
    graphs[0].replay()
    torch.cuda.synchronize()
    check_attn(*outs[0], *attention64(q, hk.flip(0), hv.flip(0), lengths, False, 0.125))
    start = i32(3, 3, 3, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_cache_write(cache, new, new, table, start)
    start.copy_(i32(9, 200, 17, 399))
    graph.replay()
    torch.cuda.synchronize()
    got = kv_cache_read(cache, table, start, None, 1)[0]
    assert torch.equal(got, held(new, 4).half())
    assert torch.equal(kv_cache_read(cache, table, i32(3, 3, 3, 3), None, 1)[0], hk[:, :, 3:4].half())  # as before the capture


def test_a_captured_step_behind_copies_and_another_stream():
    """What stands in front of the cache's kernels in a graph may be a copy, a fill, or the join of two streams."""
    B, H, d = 2, 2, 128
    cache, table, k, v, g = filled(18, B, H, 200, d, 4, 64, torch.float16, i32(200, 150))
    q_in, new_in = (torch.randn(B, n, 1, d, generator=g, device="cuda").half() for n in (8, 2))
    q, new, lengths = torch.empty_like(q_in), torch.empty_like(new_in), i32(0, 0)
    host = torch.tensor([200, 150], dtype=torch.int32).pin_memory()
    side, main = torch.cuda.Stream(), torch.cuda.Stream()

    def step():
        lengths.copy_(host, non_blocking=True)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            new.copy_(new_in)
            torch.mul(q_in, 0.5, out=q)
        main.wait_stream(side)
        kv_cache_write(cache, new, new, table, lengths - 1)
        return kv_cache_attn(q, cache, table, lengths)

    with torch.cuda.stream(main):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            o = step()
    for n in ((200, 150), (180, 2), (1, 199)):
        host.copy_(torch.tensor(n, dtype=torch.int32))
        new_in.normal_(generator=g)
        q_in.normal_(generator=g)
        torch.cuda.synchronize()
        with torch.cuda.stream(main):
            graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            k[b, :, n[b] - 1] = held(new_in[b, :, 0], 4)
            v[b, :, n[b] - 1] = held(new_in[b, :, 0], 4)
        want = attention64(q_in * 0.5, k, v, lengths, False, 0.125)
        keep = torch.tensor([x <= (200, 150)[b] for b, x in enumerate(n)], device="cuda")  # positions behind 150 of sequence 1 were not written
        check_attn(o[keep], want[1][keep], *(x[keep] for x in want))


def test_lengths_that_the_kernel_before_wrote():
    """Both kernels of a call see what the launch in front of it wrote, here for 200 calls without a pause."""
    B, H, d = 3, 2, 64
    start = i32(900, 0, 2000)
    cache, table, k, v, g = filled(16, B, H, 2300, d, 4, 64, torch.float16, i32(2300, 2300, 2300))
    q = torch.randn(B, 4 * H, 1, d, generator=g, device="cuda").half()
    lengths, outs = start.clone(), []
    for _ in range(200):
        lengths.add_(1)
        outs.append(kv_cache_attn(q, cache, table, lengths))
    for i in (0, 1, 57, 199):
        n = start + i + 1
        check_attn(outs[i], attention64(q, k, v, n, False, 0.125)[1], *attention64(q, k, v, n, False, 0.125))
        assert torch.equal(outs[i], kv_cache_attn(q, cache, table, n))


def test_calls_on_another_stream_and_from_threads():
    import threading
    B, H, d = 2, 4, 128
    lengths = i32(3000, 1234)
    cache, table, k, v, g = filled(14, B, H, 3000, d, 4, 64, torch.bfloat16, lengths)
    q = torch.randn(B, 4 * H, 1, d, generator=g, device="cuda").bfloat16()
    want = kv_cache_attn(q, cache, table, lengths)
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [kv_cache_attn(q, cache, table, lengths) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            results[i] = all(torch.equal(o, want) for o in out)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == [True] * 4


# ------------------------------------------------------------------------------------------------ tables that cannot be
def test_bad_tables_and_lengths_are_left_out_and_reported():
    d, H = 64, 2
    lengths = i32(40, 40)
    cache, table, k, v, g = filled(15, 2, H, 40, d, 4, 16, torch.float16, lengths)
    q = torch.randn(2, H, 1, d, generator=g, device="cuda").half()
    before = cache.data.clone()
    for page in (-1, cache.num_pages, 2 ** 31 - 1):
        bad = table.clone()
        bad[0, 1] = page
        # attention over the other positions
        o, lse = kv_cache_attn(q, cache, bad, lengths, None, False, 0.125, True)
        keep = torch.tensor([*range(16), *range(32, 40)], device="cuda")
        w0 = attention64(q[:1], k[:1, :, keep], v[:1, :, keep], i32(24), False, 0.125)
        w1 = attention64(q[1:], k[1:], v[1:], lengths[1:], False, 0.125)
        check_attn(o, lse, *(torch.cat(x) for x in zip(w0, w1)))
        with pytest.raises(_lib.AttnB200Error, match="page"):
            torch.cuda.synchronize()
            kv_cache_attn(q, cache, table, lengths)
        assert _lib.kv_status() == 3 and _lib.kv_status() == 0
        rk, _ = kv_cache_read(cache, bad, None, lengths, 40)
        assert (rk[0, :, 16:32] == 0).all() and torch.equal(rk[0, :, 32:], k[0, :, 32:].half()) and torch.equal(rk[1], k[1].half())
        assert _lib.kv_status() == 3
        kv_cache_write(cache, q[:, :, :, :].expand(2, H, 16, d), q.expand(2, H, 16, d), bad, i32(16, 16), i32(16, 0))
        assert _lib.kv_status() == 3 and torch.equal(cache.data, before)
    # lengths, starts and counts out of range
    o, lse = kv_cache_attn(q, cache, table, i32(-5, 4000), None, False, 0.125, True)
    assert _lib.kv_status() == 4 and (o[0] == 0).all()
    for start, count in ((-1, 1), (0, 17), (0, -2), (48, 1), (2 ** 31 - 1, 1)):
        kv_cache_write(cache, q.expand(2, H, 16, d)[:, :, :, :], q.expand(2, H, 16, d), table, i32(start, 0), i32(count, 0))
        status = _lib.kv_status()
        assert status == 4, (start, count, status)
        kv_cache_read(cache, table, i32(start, 0), i32(count, 0), 16)
        assert _lib.kv_status() == 4
    # a place of the batch that is not in use may hold anything
    kv_cache_write(cache, q, q, table, i32(-7, 2 ** 31 - 1), i32(0, 0))
    assert _lib.kv_status() == 0
    kv_cache_attn(q, cache, table, lengths)
    assert _lib.kv_status() == 0


def test_refusals_on_the_device():
    cache = QuantizedKVCache(4, 2, 64, bits=4, page_size=16)
    table, lengths = i32(0, 1).reshape(1, 2), i32(20)
    x = torch.zeros(1, 2, 20, 64, device="cuda").half()
    q = torch.zeros(1, 4, 1, 64, device="cuda").half()
    ok = dict(q=q, cache=cache, page_table=table, lengths=lengths)
    for change, text in ((dict(q=q.bfloat16()), "dtype"), (dict(q=q[:, :3]), "multiple"), (dict(q=q[..., :32]), "shape"),
                         (dict(q=q.expand(1, 4, 65, 64)), "at most 64"), (dict(q=q.cpu()), "is on cpu"), (dict(page_table=table.long()), "int32"),
                         (dict(page_table=table[0]), "2-d"), (dict(lengths=lengths.long()), "int32"), (dict(lengths=i32(1, 2)), "shape"),
                         (dict(lengths=None), "tensor"), (dict(lengths=lengths.cpu()), "is on cpu"), (dict(cache=None), "QuantizedKVCache"),
                         (dict(q=q.clone().requires_grad_()), "forward only"), (dict(q=None), "4-d")):
        with pytest.raises(ValueError, match=text):
            kv_cache_attn(**{**ok, **change})
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(_lib.AttnB200Error, match="scale"):
            kv_cache_attn(q, cache, table, lengths, softmax_scale=scale)
    ok = dict(cache=cache, k=x, v=x, page_table=table, start=i32(0))
    for change, text in ((dict(v=x[:, :, :5]), "shape"), (dict(k=x[:, :1], v=x[:, :1]), "heads"), (dict(k=x.float()), "dtype"),
                         (dict(start=None), "start"), (dict(count=torch.ones(1, device="cuda")), "int32"), (dict(k=x[:, :, :0], v=x[:, :, :0]), "shape"),
                         (dict(v=x.clone().requires_grad_()), "forward only"), (dict(k=x.cpu()), "is on cpu")):
        with pytest.raises(ValueError, match=text):
            kv_cache_write(**{**ok, **change})
    with torch.no_grad():
        kv_cache_write(cache, x.clone().requires_grad_(), x, table, i32(0))
    for length in (0, -1, 1.5, True, None):
        with pytest.raises(ValueError, match="length"):
            kv_cache_read(cache, table, length=length)
    # the C ABI: a workspace that is missing, too small or misaligned
    import ctypes
    lib, c, big = _lib.load_kv(), cache.struct(), torch.zeros(1, 64, dtype=torch.int32, device="cuda")
    need = lib.attn_b200_kv_attn_workspace_bytes(ctypes.byref(c), 64, 1, 2, 1)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    for at, size in ((None, 0), (None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert lib.attn_b200_kv_attn(q.data_ptr(), ctypes.byref(c), big.data_ptr(), 64, 64, lengths.data_ptr(), q.data_ptr(), None, at, size, 1, 2, 1,
                                     0.125, 0, torch.cuda.current_stream().cuda_stream) == 1
    many = torch.zeros(4097, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.AttnB200Error, match="4097"):
        kv_cache_attn(q.expand(4097, 4, 1, 64), cache, many, torch.zeros(4097, dtype=torch.int32, device="cuda"))
