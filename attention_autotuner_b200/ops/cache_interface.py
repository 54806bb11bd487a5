"""A quantised, paged KV cache for decoding, and attention over it. No counterpart in the reference, whose operators read dense
16-bit K and V (python/ops/attention_interface.py:11-35).

    cache = QuantizedKVCache(num_pages, heads, head_dim, bits=4, page_size=64, dtype=torch.float16, device="cuda")
    kv_cache_write(cache, k, v, page_table, start, count=None)          # positions start[b] + i, i < count[b]
    o = kv_cache_attn(q, cache, page_table, lengths, device_type, causal=False, softmax_scale=None, return_lse=False)
    k, v = kv_cache_read(cache, page_table, start, count, length)       # dense again, for flash_attn_func over equal lengths

A position of a head of K or V is held as whole numbers n of 4 or 8 bits with a scale and a zero of the cache's type and stands for
``zero + scale * n``: zero is the smallest of the head_dim values, scale their range over 2^bits - 1 rounded to the type, n the
nearest whole number (half to even). A row with an infinity or a NaN stands for NaN. 2 (head_dim bits / 8 + 4) bytes per position
and head instead of 4 head_dim: 136 instead of 512 at 4 bits and head dimension 128.

``page_table`` int32 [B, width]: entry i of row b is the page of positions [i page_size, (i + 1) page_size) of sequence b; entries
behind the positions in use are never read. ``start``, ``count`` and ``lengths`` are int32 [B]. All four are CUDA tensors that the
kernels read when they run, so a captured CUDA graph sees the values of its replay. What is out of range in them (a page that does
not exist, positions behind the table's last entry, negative numbers) is left out (not written, read back as zeros, not attended
to) and makes later calls raise AttnB200Error until ``_lib.kv_status()`` has reported and cleared it. A page may stand in several
rows for reading; two rows that write the same position leave a mixture. Forward only. Everything runs on the current stream of
the cache's device."""
import torch

from .. import _lib
from ._checks import check_like
from ._native import kv_ops

MAX_QUERIES = 64  # new positions of a sequence in one kv_cache_attn call
_CODES = {torch.float16: 0, torch.bfloat16: 1}


def _fail(msg):
    raise ValueError(msg)


class QuantizedKVCache:
    """``num_pages`` pages of ``page_size`` positions (a power of two from 16 on) of ``heads`` heads; head_dim 64, 128 or 256.
    ``data`` holds them, uint8 [num_pages, heads, page_size / 16, block bytes] and uninitialised: nothing is read that was not
    written. K, V and queries have the cache's ``dtype``. Make it before a stream capture begins."""

    def __init__(self, num_pages, heads, head_dim, bits=4, page_size=64, dtype=torch.float16, device="cuda"):
        for name, x in (("num_pages", num_pages), ("heads", heads), ("head_dim", head_dim), ("bits", bits), ("page_size", page_size)):
            if not isinstance(x, int) or isinstance(x, bool):
                _fail(f"QuantizedKVCache: {name} must be an integer, got {x!r}")
        if dtype not in _CODES:
            _fail(f"QuantizedKVCache: dtype must be float16 or bfloat16, got {dtype}")
        if bits not in (4, 8):
            _fail(f"QuantizedKVCache: bits must be 4 or 8, got {bits}")
        if head_dim not in (64, 128, 256):
            _fail(f"QuantizedKVCache: head dimension must be 64, 128 or 256, got {head_dim}")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            _fail(f"QuantizedKVCache: page_size must be a power of two from 16 to 65536, got {page_size}")
        if not 0 < num_pages < 2 ** 31 or not 0 < heads <= 65535:
            _fail(f"QuantizedKVCache: {num_pages} pages of {heads} heads are not supported")
        device = torch.device(device)
        if device.type != "cuda":
            _fail(f"QuantizedKVCache: the cache must live on a CUDA device (there is no CPU path), got {device}")
        kv_ops()
        lib = _lib.load_kv()
        self.num_pages, self.heads, self.head_dim, self.bits, self.page_size, self.dtype = num_pages, heads, head_dim, bits, page_size, dtype
        block = lib.attn_b200_kv_block_bytes(bits, head_dim)
        self.data = torch.empty(num_pages, heads, page_size // 16, block, dtype=torch.uint8, device=device)
        with torch.cuda.device(self.data.device):
            _lib.check_kv(lib.attn_b200_kv_prepare())
        self._form = (bits, head_dim, _CODES[dtype])

    @property
    def device(self):
        return self.data.device

    def struct(self):
        """The cache as the C ABI takes it (include/attn_b200_kv.h)."""
        bits, head_dim, code = self._form
        return _lib.KVCacheStruct(self.data.data_ptr(), self.num_pages, self.heads, self.page_size, head_dim, bits, code)


def _check_cache(op, cache, page_table):
    if not isinstance(cache, QuantizedKVCache):
        _fail(f"{op}: cache must be a QuantizedKVCache, got {type(cache).__name__}")
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.numel() == 0:
        _fail(f"{op}: page_table must be a 2-d tensor [batch, pages of a sequence] that is not empty")
    if page_table.dtype != torch.int32:
        _fail(f"{op}: page_table has dtype {page_table.dtype}, expected torch.int32")
    if page_table.device != cache.device:
        _fail(f"{op}: page_table is on {page_table.device}, the cache on {cache.device}")


def _check_values(op, name, t, cache, page_table):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        _fail(f"{op}: {name} must be a 4-d tensor [batch, heads, length, head_dim]")
    if t.dtype != cache.dtype:
        _fail(f"{op}: {name} has dtype {t.dtype}, the cache {cache.dtype}")
    if t.device != cache.device:
        _fail(f"{op}: {name} is on {t.device}, the cache on {cache.device}")
    if t.shape[0] != page_table.shape[0] or t.shape[3] != cache.head_dim or min(t.shape) == 0:
        _fail(f"{op}: {name} has shape {tuple(t.shape)}; page_table has {page_table.shape[0]} sequences, the cache head dimension "
              f"{cache.head_dim}")
    if torch.is_grad_enabled() and t.requires_grad or torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        _fail(f"{op}: {name} requires a gradient, and the KV cache is forward only: call it under torch.no_grad() or detach")


def _check_per_sequence(op, page_table, **tensors):
    for name, t in tensors.items():
        if t is not None:
            check_like(op, name, t, page_table.shape[:1], torch.int32, page_table.device)


def kv_cache_write(cache, k, v, page_table, start, count=None):
    """Quantises k, v [B, heads, L, head_dim] and writes position i < count[b] (all L without ``count``) of sequence b as its position
    start[b] + i. Any strides; no copy where channels are dense and rows start at multiples of 16 bytes."""
    if isinstance(cache, QuantizedKVCache):
        if kv_ops().kv_write(cache.data, *cache._form, page_table, start, count, k, v):
            return
    op = "kv_cache_write"
    _check_cache(op, cache, page_table)
    _check_values(op, "k", k, cache, page_table)
    _check_values(op, "v", v, cache, page_table)
    if k.shape[1] != cache.heads:
        _fail(f"{op}: k has {k.shape[1]} heads, the cache {cache.heads}")
    if k.shape != v.shape:
        _fail(f"{op}: v has shape {tuple(v.shape)}, k has {tuple(k.shape)}")
    if start is None:
        _fail(f"{op}: start must be a tensor")
    _check_per_sequence(op, page_table, start=start, count=count)
    _fail(f"{op}: not supported: k {tuple(k.shape)}, page_table {tuple(page_table.shape)}, data {tuple(cache.data.shape)}")


def kv_cache_read(cache, page_table, start=None, count=None, length=None):
    """K and V [B, heads, length, head_dim] of positions start[b] + i (from 0 without ``start``), rounded to the cache's dtype; rows
    i >= count[b] are zeros. For a prompt that goes on behind what the cache holds by more than 64 positions: flash_attn_func takes them
    with each head repeated for the heads of q that share it. It has no lengths and would attend to the zeros, so sequences of
    different lengths go through it one at a time (``page_table[b:b + 1]``, ``length`` of that sequence)."""
    op = "kv_cache_read"
    if not isinstance(length, int) or isinstance(length, bool) or not 0 < length <= 1 << 30:
        _fail(f"{op}: length must be a positive integer, got {length!r}")
    if isinstance(cache, QuantizedKVCache):
        out = kv_ops().kv_read(cache.data, *cache._form, page_table, start, count, length)
        if out is not None:
            return out
    _check_cache(op, cache, page_table)
    _check_per_sequence(op, page_table, start=start, count=count)
    _fail(f"{op}: not supported: page_table {tuple(page_table.shape)}, data {tuple(cache.data.shape)}")


def kv_cache_attn(q, cache, page_table, lengths, device_type=None, causal=False, softmax_scale=None, return_lse=False):
    """flash_attn_func over the first lengths[b] positions of each sequence, for up to 64 queries: q [B, Hq, Lq, head_dim], Hq a
    multiple of the cache's heads (query heads h Hq/heads ... share head h). With ``causal`` the queries are the last Lq positions:
    query i sees j <= i + lengths[b] - Lq. A query that sees nothing gets 0 (lse -inf). ``softmax_scale=None`` is 0.125, as there.
    The values zero + scale * n are used as they are, without a rounding to 16 bits. Up to 4096 sequences. ``device_type`` stands where
    flash_attn_func has it and is not used: there is no tile configuration to look up."""
    scale = 0.125 if softmax_scale is None else softmax_scale
    if isinstance(cache, QuantizedKVCache):
        out = kv_ops().kv_attn(cache.data, *cache._form, page_table, lengths, q, scale, causal, return_lse)
        if out is not None:
            return out
    op = "kv_cache_attn"
    _check_cache(op, cache, page_table)
    _check_values(op, "q", q, cache, page_table)
    if q.shape[1] % cache.heads != 0:
        _fail(f"{op}: q has {q.shape[1]} heads, not a multiple of the cache's {cache.heads}")
    if q.shape[2] > MAX_QUERIES:
        _fail(f"{op}: {q.shape[2]} queries of a sequence, at most {MAX_QUERIES} (longer prompts: kv_cache_read and "
              "flash_attn_func, for sequences of one length)")
    if lengths is None:
        _fail(f"{op}: lengths must be a tensor")
    _check_per_sequence(op, page_table, lengths=lengths)
    _fail(f"{op}: not supported: q {tuple(q.shape)}, page_table {tuple(page_table.shape)}, data {tuple(cache.data.shape)}")
