"""Performance cases of the quantised KV cache: writing it, reading it back, and attention over it.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU, as a serving program has them before the call
    run(state)           one pass: the plain form in 32 bits, or (own) the package's operators
    work(case)           bytes and operations one pass cannot do without
    exact(case, seed)    what run returns, from the definition in 64 bits

A position of a head is held as whole numbers n of 4 or 8 bits with two 16-bit numbers, K and V apart: zero is the smallest
of its d values, scale the range over 2^bits - 1, n = (x - zero) / scale rounded to the nearest, half to even; the value is
zero + scale n. Positions live in pages that a table names for each sequence.

A case is a dict: ``op`` (attn, write, read), the sizes B, Hq, Hkv, Lq, L, d, ``bits``, ``page``, the data type, ``ragged``
(sequences of many lengths, one of them empty, or all of L positions) and ``causal`` for attn. ``write`` writes up to Lq new
positions of each sequence behind the L that are there and reads the same positions back, ``read`` reads up to L.
"""
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, B, Hq, Hkv, Lq, L, d, bits, page, dtype, ragged, causal=False):
    return dict(name=name, op=op, B=B, Hq=Hq, Hkv=Hkv, Lq=Lq, L=L, d=d, bits=bits, page=page, dtype=dtype, ragged=ragged, causal=causal)


def listed():
    return [
        # a decoding step of the smallest benchmark configuration: latency
        _case("attn_token_small", "attn", 2, 4, 4, 1, 512, 64, 4, 16, "fp16", False),
        # a decoding step of a serving batch, grouped heads, sequences between empty and 8192
        _case("attn_token_batch", "attn", 32, 32, 8, 1, 8192, 128, 4, 64, "bf16", True),
        # the decoding configuration of the dense operator (a head of K and V for each of Q), in 8 bits
        _case("attn_token_16k", "attn", 2, 16, 16, 1, 16384, 128, 8, 128, "bf16", False),
        # a draft of four tokens looked over at once, causal among themselves
        _case("attn_draft", "attn", 16, 32, 8, 4, 4096, 128, 8, 32, "fp16", True, True),
        # a few long documents, the largest read
        _case("attn_token_long", "attn", 8, 32, 8, 1, 131072, 128, 4, 64, "fp16", False),
        # one long document of a model with wide heads and one head of K and V
        _case("attn_token_wide", "attn", 1, 8, 1, 1, 50001, 256, 4, 16, "bf16", False),
        # the token that every sequence of a batch adds per step
        _case("write_token", "write", 64, 8, 8, 1, 1000, 128, 4, 64, "bf16", False),
        # the cache of one long prompt, 8 bits
        _case("write_prompt", "write", 1, 16, 16, 16384, 0, 128, 8, 128, "bf16", False),
        # prompts of odd lengths that go on behind what is there, head dimension 64
        _case("write_ragged", "write", 4, 12, 12, 1500, 333, 64, 4, 16, "fp16", True),
        # a short prompt's cache read back for its next piece
        _case("read_short", "read", 1, 8, 8, 1, 500, 128, 4, 64, "fp16", False),
        # the caches of a ragged batch read back for a dense pass
        _case("read_ragged", "read", 4, 16, 16, 1, 2999, 128, 4, 64, "bf16", True),
        # one long cache read back whole, 8 bits
        _case("read_long", "read", 1, 16, 16, 1, 16384, 128, 8, 128, "fp16", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    op = rng.choice(("attn", "attn", "attn", "attn", "write", "read"))
    dtype, bits, page = rng.choice(("fp16", "bf16")), rng.choice((4, 4, 8)), rng.choice((16, 32, 64, 128))
    d = rng.choice((64, 128, 128, 256))
    B, Hkv = _log_int(rng, 1, 96), rng.choice((1, 2, 4, 8, 16))
    ragged = rng.choice((False, True))
    if op == "attn":
        Lq = rng.choice((1, 1, 1, 2, 3, 5, 8))
        group = rng.choice((1, 2, 4, 5, 8, 16))
        return _case("", op, B, Hkv * group, Hkv, Lq, _log_int(rng, 16, 65536), d, bits, page, dtype, ragged, rng.choice((True, Lq == 1)))
    if op == "write":
        Lq = rng.choice((1, _log_int(rng, 2, 16384)))
        return _case("", op, B, Hkv, Hkv, Lq, rng.choice((0, _log_int(rng, 1, 5000))), d, bits, page, dtype, ragged)
    return _case("", op, B, Hkv, Hkv, 1, _log_int(rng, 1, 16384), d, bits, page, dtype, ragged)


def draw(rng):
    limit = {"attn": 3.0e8, "write": 1.3e8, "read": 1.3e8}  # bytes: below the largest listed case of each kind
    while True:
        case = _draw_once(rng)
        padded = case["B"] * case["Hkv"] * (case["L"] + case["Lq"]) * case["d"]  # what the plain form holds in 32 bits
        w = work(case)
        if w["bytes"] <= limit[case["op"]] and w["flops"] <= 1.5e10 and padded <= 1.0e9:
            del case["name"]
            return case


def _lengths(case):
    """Positions of each sequence that are there (attn, read), or that come in (write)."""
    B, most = case["B"], case["Lq"] if case["op"] == "write" else case["L"]
    if not case["ragged"]:
        return [most] * B
    rng = random.Random(B * 1000003 + most)
    lens = [_log_int(rng, max(1, most // 64), most) for _ in range(B)]
    if B >= 3:
        lens[B // 2] = 0  # a place of the batch that no request has taken
    lens[-1] = most
    return lens


def _inputs(case, seed):
    """q, k, v in their 16-bit type: channels of K about means of their own, a few of them far out; k and v are what the cache holds or, for write, is given."""
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator("cuda").manual_seed(seed)
    B, Hq, Hkv, d = case["B"], case["Hq"], case["Hkv"], case["d"]
    n = case["Lq"] if case["op"] == "write" else case["L"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    mean = normal(Hkv, 1, d)
    mean[:, :, ::29] *= 4.0
    q = normal(B, Hq, case["Lq"], d).to(dt)
    k = torch.empty(B, Hkv, n, d, device="cuda", dtype=dt)
    v = torch.empty(B, Hkv, n, d, device="cuda", dtype=dt)
    for b in range(B):
        k[b] = normal(Hkv, n, d) + mean
        v[b] = normal(Hkv, n, d)
    start = [case["L"] if case["op"] == "write" else 0] * B
    pages = -(-(n + start[0]) // case["page"])
    order = torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).reshape(B, pages)
    return q, k, v, start, order


def _quantise(x, bits):
    """Whole numbers (uint8), scales and zeros (16 bits) of the rows of x."""
    f = x.float()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    most = torch.full_like(lo, 2 ** bits - 1)
    scale, zero = ((hi - lo) / most).to(x.dtype), lo.to(x.dtype)
    s = scale.float()
    n = torch.where(s > 0, (f - zero.float()) / s, torch.zeros_like(f)).round().clamp(0, 2 ** bits - 1)
    return n.to(torch.uint8), scale, zero


def _values(n, scale, zero):
    return zero.float() + scale.float() * n.float()


def prepare(case, seed):
    q, k, v, start, table = _inputs(case, seed)
    B, Hkv, d, page, bits = (case[x] for x in ("B", "Hkv", "d", "page", "bits"))
    lens = _lengths(case)
    dev = q.device
    used = torch.tensor([-(-(s + n) // page) for s, n in zip(start, lens)], device=dev)
    table = torch.where(torch.arange(table.shape[1], device=dev)[None] < used[:, None], table, torch.full_like(table, -1))
    num_pages = table.numel()
    st = dict(op=case["op"], bits=bits, page=page, causal=case["causal"], scale=d ** -0.5, table=table, n=k.shape[2],
              start=torch.tensor(start, device=dev, dtype=torch.int32), count=torch.tensor(lens, device=dev, dtype=torch.int32))
    if own:
        from attention_autotuner_b200.arch import B200
        from attention_autotuner_b200.ops.cache_interface import QuantizedKVCache, kv_cache_write
        st["arch"] = B200()
        st["cache"] = QuantizedKVCache(num_pages, Hkv, d, bits=bits, page_size=page, dtype=q.dtype, device=dev)
        if case["op"] != "write":
            kv_cache_write(st["cache"], k, v, table, st["start"], st["count"])
    else:
        for x in ("k", "v"):
            st[x + "n"] = torch.zeros(num_pages + 1, Hkv, page, d, device=dev, dtype=torch.uint8)
            st[x + "s"], st[x + "z"] = (torch.zeros(num_pages + 1, Hkv, page, 1, device=dev, dtype=q.dtype) for _ in range(2))
        if case["op"] != "write":
            for b in range(B):
                _plain_write({**st, "table": table[b:b + 1], "start": st["start"][b:b + 1], "count": st["count"][b:b + 1]},
                             k[b:b + 1], v[b:b + 1])
    if case["op"] == "attn":
        st["q"] = q
    elif case["op"] == "write":
        st["k"], st["v"] = k, v
    return st


def _places(st, length):
    """Of positions start + i, i < length: page, place in the page, and whether i < count."""
    i = torch.arange(length, device=st["table"].device)[None]
    pos = st["start"].long()[:, None] + i
    there = i < st["count"].long()[:, None]
    pages = st["table"].long().gather(1, (pos // st["page"]).clamp(max=st["table"].shape[1] - 1)).clamp(min=0)
    return pages, pos % st["page"], there


def _plain_write(st, k, v):
    pages, rows, there = _places(st, k.shape[2])
    pages = torch.where(there, pages, torch.full_like(pages, st["kn"].shape[0] - 1))  # the last page takes what is in no sequence
    for x, name in ((k, "k"), (v, "v")):
        parts = _quantise(x, st["bits"])
        for part, which in zip(parts, "nsz"):
            st[name + which][pages, :, rows] = part.transpose(1, 2)


def _plain_values(st, length):
    """K and V of positions start + i in 32 bits [B, Hkv, length, d], and whether i < count [B, length]."""
    pages, rows, there = _places(st, length)
    return [_values(*(st[x + part][pages, :, rows].transpose(1, 2) for part in "nsz")) for x in "kv"] + [there]


def _plain_attn(st):
    k, v, there = _plain_values(st, st["n"])
    q = st["q"].float()
    B, Hq, Lq, d = q.shape
    Hkv = k.shape[1]
    rows = q.reshape(B, Hkv, Hq // Hkv * Lq, d)
    s = (rows @ k.transpose(-1, -2) * st["scale"]).reshape(B, Hkv, Hq // Hkv, Lq, -1)
    seen = there[:, None, None, None, :]
    if st["causal"]:
        i, j = torch.arange(Lq, device=q.device)[:, None], torch.arange(st["n"], device=q.device)[None]
        seen = seen & (j <= i + (st["count"].long()[:, None, None] - Lq))[:, None, None]
    s = torch.where(seen, s, torch.full((), -math.inf, device=q.device))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p.reshape(B, Hkv, -1, st["n"]) @ v
    return o.reshape(B, Hq, Lq, d).to(st["q"].dtype)


def run(st):
    if own:
        from attention_autotuner_b200.ops.cache_interface import kv_cache_attn, kv_cache_read, kv_cache_write
        if st["op"] == "attn":
            return kv_cache_attn(st["q"], st["cache"], st["table"], st["count"], st["arch"], st["causal"], st["scale"])
        if st["op"] == "write":
            kv_cache_write(st["cache"], st["k"], st["v"], st["table"], st["start"], st["count"])
        return kv_cache_read(st["cache"], st["table"], st["start"], st["count"], st["n"])
    if st["op"] == "attn":
        return _plain_attn(st)
    if st["op"] == "write":
        _plain_write(st, st["k"], st["v"])
    k, v, there = _plain_values(st, st["n"])
    dtype = st["ks"].dtype
    zero = torch.zeros((), device=k.device)
    return tuple(torch.where(there[:, None, :, None], x, zero).to(dtype) for x in (k, v))


def work(case):
    """Bytes: the positions that are there in their packed form, every 16-bit input and output once (a written cache counts as
    one output). Operations: two products over the positions that are seen; quantising counts none."""
    B, Hq, Hkv, Lq, d, bits = (case[x] for x in ("B", "Hq", "Hkv", "Lq", "d", "bits"))
    lens = _lengths(case)
    packed = sum(lens) * Hkv * 2 * (d * bits // 8 + 4)
    if case["op"] == "attn":
        seen = sum(max(0, min(n, i + n - Lq + 1)) if case["causal"] else n for n in lens for i in range(Lq))
        return dict(bytes=packed + 4 * B * Hq * Lq * d, flops=4 * Hq * seen * d)
    given = sum(lens) * Hkv * d * 4
    returned = B * (Lq if case["op"] == "write" else case["L"]) * Hkv * d * 4
    return dict(bytes=packed + returned + (given if case["op"] == "write" else 0), flops=0)


def exact(case, seed):
    q, k, v, _, _ = _inputs(case, seed)
    dt, top = q.dtype, float(2 ** case["bits"] - 1)

    def held(x):  # [Hkv, n, d] of one sequence: the values that its numbers stand for
        x = x.double()
        low = x.min(-1, keepdim=True).values
        step = ((x.max(-1, keepdim=True).values - low) / torch.tensor([top], device=x.device, dtype=x.dtype)).to(dt).double()
        return low + step * torch.clamp(torch.round((x - low) / torch.where(step == 0, torch.inf, step)), 0.0, top)

    outs = []
    for b, n in enumerate(_lengths(case)):
        if case["op"] != "attn":
            both = []
            for x in (k[b], v[b]):
                full = torch.zeros(x.shape, device=x.device, dtype=torch.float64)
                full[:, :n] = held(x[:, :n])
                both.append(full)
            outs.append(both)
            continue
        Hq, Lq, d = q.shape[1:]
        o = torch.zeros(Hq, Lq, d, device=q.device, dtype=torch.float64)
        kb, vb = held(k[b, :, :n]), held(v[b, :, :n])
        for i in range(Lq):
            m = max(0, n - Lq + 1 + i) if case["causal"] else n
            if m == 0:
                continue
            rows = q[b, :, i].double().unflatten(0, (case["Hkv"], -1))  # [Hkv, group, d]
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", rows, kb[:, :m]) * d ** -0.5, dim=-1)
            o[:, i] = torch.einsum("hgn,hnd->hgd", p, vb[:, :m]).flatten(0, 1)
        outs.append(o)
    if case["op"] == "attn":
        return torch.stack(outs)
    return tuple(torch.stack([pair[i] for pair in outs]) for i in range(2))
