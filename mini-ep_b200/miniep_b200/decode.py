"""The operators of a decode step around the expert-parallel layer, as CUDA
kernels: writing new tokens into the key/value cache, attention over it, and
sampling the next token.

  * ``KVCache``: keys and values of a batch for every layer, in the model
    dtype or quantised to e4m3 with one fp32 scale a row;
  * ``norm_rope_store``: head norms, rotation and the cache write in one pass;
  * ``cache_attention``: attention of new tokens over a row's cache and, with a
    ``SharedPrefix``, over a prefix that all rows share;
  * ``sample_tokens`` / ``Sampler``: temperature, top-k, top-p and min-p from
    given uniform numbers.

Tensors are CUDA tensors on one device, whichever is current; work goes to
that device's current stream and nothing synchronises. The operators are for
inference: a tensor that requires grad is refused while grad mode is on.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from ._lib import MEPError, check

_DTYPES = {torch.float32: _lib.MEP_F32, torch.bfloat16: _lib.MEP_BF16}
_CACHE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.MEP_E4M3}


def _need(cond: bool, msg: str):
    if not cond:
        raise MEPError(msg)


def _tensor(t, name: str, device, dtype=None):
    """Refuses what is not a CUDA tensor on `device` (None: any) of `dtype`."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise MEPError(f"{name} must be a CUDA tensor")
    if device is not None and t.get_device() != device.index:
        raise MEPError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype is not dtype:
        raise MEPError(f"{name} must be {dtype}, not {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise MEPError(f"{name} requires grad: this operator has no backward pass")


def _rows(t):
    """`t` (batch, tokens, heads, head_dim) itself where the kernels' 16-byte
    accesses fit its strides, else a copy; its address and strides."""
    b, n, h, one = t.stride()
    p = t.data_ptr()
    if one != 1 or (p | (b | n | h) * t.element_size()) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        b, n, h, _ = t.stride()
        p = t.data_ptr()
    return t, p, b, n, h


def _flat(t):
    """Contiguous and on a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() & 15 == 0 else t.clone()


class _on:
    """Calls into the library with the tensors' device current."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


class KVCache:
    """Keys and values (layers, batch, kv_heads, capacity, head_dim),
    contiguous CUDA tensors the caller owns. In the model dtype, or quantised:
    torch.float8_e4m3fn codes with fp32 scales (layers, batch, kv_heads,
    capacity); `dtype` is then the model dtype that `read` answers in."""

    def __init__(self, k, v, k_scale=None, v_scale=None, dtype=None):
        _tensor(k, "k", None)
        _tensor(v, "v", k.device, k.dtype)
        _need(k.dtype in _CACHE_DTYPES, f"a cache is fp32, bf16 or e4m3, not {k.dtype}")
        _need(k.dim() == 5 and k.shape == v.shape,
              "k and v must both be (layers, batch, kv_heads, capacity, head_dim)")
        self.quantized = k.dtype == torch.float8_e4m3fn
        dtype = dtype or (torch.bfloat16 if self.quantized else k.dtype)
        _need(dtype in _DTYPES, f"the model dtype is fp32 or bf16, not {dtype}")
        _need(self.quantized or dtype == k.dtype,
              f"a {k.dtype} cache cannot serve a {dtype} model")
        _need((k_scale is not None) == self.quantized and (v_scale is not None) == self.quantized,
              "k_scale and v_scale go with an e4m3 cache, and only with one")
        parts = [k, v]
        if self.quantized:
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                _tensor(t, name, k.device, torch.float32)
                _need(t.shape == k.shape[:-1], f"{name} must be {tuple(k.shape[:-1])}")
            parts += [k_scale, v_scale]
        for t in parts:
            _need(t.is_contiguous() and t.data_ptr() % 16 == 0,
                  "cache tensors must be contiguous and start on a 16-byte boundary")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.dtype, self.device = dtype, k.device
        self.layers, self.batch, self.kv_heads, self.capacity, self.head_dim = k.shape
        self._code = _CACHE_DTYPES[k.dtype]
        # every layer starts on a 16-byte boundary too: a row is a multiple of
        # 16 bytes (head_dim is one of 16), and scales are read one at a time
        step = [t[0].numel() * t.element_size() if self.layers else 0 for t in parts]
        at = [t.data_ptr() for t in parts] + [0] * (4 - len(parts))
        step += [0] * (4 - len(parts))
        self._ptrs = [tuple(p + l * d for p, d in zip(at, step)) for l in range(self.layers)]

    @classmethod
    def empty(cls, layers: int, batch: int, kv_heads: int, capacity: int, head_dim: int,
              dtype=torch.bfloat16, quantized: bool = False, device="cuda") -> "KVCache":
        """A zeroed cache of its own tensors."""
        shape = (layers, batch, kv_heads, capacity, head_dim)
        store = torch.float8_e4m3fn if quantized else dtype
        k, v = (torch.zeros(shape, dtype=store, device=device) for _ in range(2))
        ks = vs = None
        if quantized:
            ks, vs = (torch.zeros(shape[:-1], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs, dtype)

    def layer(self, layer: int) -> tuple:
        _need(0 <= layer < self.layers, f"layer {layer} outside [0, {self.layers})")
        return self._ptrs[layer]

    def read(self, layer: int, start: int, end: int):
        """Columns [start, end) of one layer, (batch, kv_heads, end - start,
        head_dim) each, in the model dtype: a view of a cache that holds it,
        code * scale rounded once of a quantised one."""
        return self._read(layer, 0, self.batch, start, end)

    def _read(self, layer: int, first: int, rows: int, start: int, end: int):
        """`read` of batch rows [first, first + rows)."""
        kp, vp, ksp, vsp = self.layer(layer)
        _need(0 <= start <= end <= self.capacity,
              f"columns [{start}, {end}) outside the cache's {self.capacity}")
        if not self.quantized:
            return tuple(t[layer, first:first + rows, :, start:end] for t in (self.k, self.v))
        shape = (2, rows, self.kv_heads, end - start, self.head_dim)
        out = torch.empty(shape, dtype=self.dtype, device=self.device)
        k, v = out[0], out[1]
        skip = first * self.kv_heads * self.capacity  # cached rows before them
        at = skip * self.head_dim
        with _on(self.device) as stream:
            check(_lib.lib().mep_kv_read(_DTYPES[self.dtype], rows, self.kv_heads,
                                         self.head_dim, kp + at, vp + at, ksp + 4 * skip,
                                         vsp + 4 * skip, self.capacity, start, end - start,
                                         k.data_ptr(), v.data_ptr(), stream),
                  None, "KVCache.read")
        return k, v


class SharedPrefix:
    """Keys and values of a prefix all rows of a batch share: (layers,
    kv_heads, columns, head_dim) each, rotated, in the model dtype."""

    def __init__(self, k, v):
        _tensor(k, "prefix k", None)
        _tensor(v, "prefix v", k.device, k.dtype)
        _need(k.dtype in _DTYPES, f"a prefix is fp32 or bf16, not {k.dtype}")
        _need(k.dim() == 4 and k.shape == v.shape,
              "prefix k and v must both be (layers, kv_heads, columns, head_dim)")
        for t in (k, v):
            _need(t.is_contiguous() and t.data_ptr() % 16 == 0,
                  "prefix tensors must be contiguous and start on a 16-byte boundary")
        self.k, self.v = k, v
        self.layers, self.kv_heads, self.columns, self.head_dim = k.shape
        step = k[0].numel() * k.element_size() if self.layers else 0
        self._ptrs = [(k.data_ptr() + l * step, v.data_ptr() + l * step)
                      for l in range(self.layers)]

    @classmethod
    def from_cache(cls, cache: KVCache, row: int, columns: int) -> "SharedPrefix":
        """A copy of the first `columns` columns of one row, of every layer
        (read back to the model dtype from a quantised cache)."""
        _need(0 <= row < cache.batch, f"row {row} outside [0, {cache.batch})")
        got = [cache._read(l, row, 1, 0, columns) for l in range(cache.layers)]
        return cls(torch.cat([k for k, _ in got]).contiguous(),
                   torch.cat([v for _, v in got]).contiguous())


def _column(col, device):
    """(host column or -1, device pointer or 0)."""
    if isinstance(col, torch.Tensor):
        _tensor(col, "col", device, torch.int64)
        _need(col.numel() == 1, "col must hold one column")
        return -1, col.data_ptr()
    col = int(col)
    _need(0 <= col < 1 << 62, f"column {col} does not fit the cache")
    return col, 0


def _heads(q, cache: KVCache):
    _tensor(q, "q", cache.device, cache.dtype)
    if q.dim() != 4 or q.shape[0] != cache.batch or q.shape[3] != cache.head_dim:
        raise MEPError(f"q {tuple(q.shape)} must be (batch, tokens, heads, head_dim) and fit a "
                       f"cache of batch {cache.batch}, head_dim {cache.head_dim}")
    return q.shape


def norm_rope_store(q, k, v, cos, sin, positions, cache: KVCache, layer: int, col, *,
                    q_norm=None, k_norm=None, eps: float = 1e-6):
    """Optional RMS norm of each q and k head, rotation, and the cache write of
    new tokens, in one pass. q: (B, T, Hq, D); k, v: (B, T, Hk, D), any
    strides; cos, sin: (rows, D) fp32 or model dtype; positions: (B, T) int64
    (broadcast over B allowed). Token t's K (rotated) and V go to column
    col + t of `cache`'s `layer`, quantised if the cache is; `col` is an int
    or a one-element int64 device tensor (columns outside the cache are then
    not written). Returns the rotated q, (B, T, Hq, D) contiguous."""
    B, T, Hq, D = _heads(q, cache)
    dev, dt, Hk = cache.device, cache.dtype, cache.kv_heads
    _tensor(k, "k", dev, dt)
    _tensor(v, "v", dev, dt)
    if k.shape != (B, T, Hk, D) or v.shape != (B, T, Hk, D):
        raise MEPError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be {(B, T, Hk, D)}")
    _tensor(cos, "cos", dev)
    _tensor(sin, "sin", dev, cos.dtype)
    _need(cos.dtype is torch.float32 or cos.dtype is dt, f"cos and sin must be fp32 or {dt}")
    rows = cos.shape[0] if cos.dim() == 2 else -1
    _need(cos.shape == (rows, D) and sin.shape == (rows, D), f"cos and sin must be (rows, {D})")
    _tensor(positions, "positions", dev, torch.int64)
    pb, pt = positions.stride() if positions.dim() == 2 else (0, 0)
    if positions.shape != (B, T):
        _need(positions.shape == (1, T), f"positions must be {(B, T)}, not {tuple(positions.shape)}")
        pb = 0
    qn = kn = 0
    if q_norm is not None:
        _tensor(q_norm, "q_norm", dev, dt)
        _need(q_norm.shape == (D,), f"q_norm must be ({D},)")
        q_norm = _flat(q_norm)
        qn = q_norm.data_ptr()
    if k_norm is not None:
        _tensor(k_norm, "k_norm", dev, dt)
        _need(k_norm.shape == (D,), f"k_norm must be ({D},)")
        k_norm = _flat(k_norm)
        kn = k_norm.data_ptr()
    cos, sin = _flat(cos), _flat(sin)
    q, *qs = _rows(q)
    k, *ks = _rows(k)
    v, *vs = _rows(v)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    args = _lib.STORE_ARGS.pack(
        _DTYPES[dt], cache._code, B, T, Hq, Hk, D, *qs, *ks, *vs, qn, kn, eps, cos.data_ptr(),
        sin.data_ptr(), _DTYPES[cos.dtype], rows, positions.data_ptr(), pb, pt, out.data_ptr(),
        *cache.layer(layer), cache.capacity, *_column(col, dev))
    with _on(dev) as stream:
        rc = _lib.lib().mep_norm_rope_store(args, stream)
    check(rc, None, "norm_rope_store")
    return out


@lru_cache(maxsize=4096)
def _attention_workspace(*sizes) -> int:
    n = C.c_int64()
    check(_lib.lib().mep_cache_attention_workspace(*sizes, C.byref(n)), None, "cache_attention")
    return n.value


def cache_attention(q, cache: KVCache, layer: int, col, scale: float, *, lengths=None,
                    prompt_cols: int = 0, prefix: SharedPrefix | None = None):
    """Attention of new tokens over `cache`'s `layer`: q (B, T, Hq, D) rotated,
    any strides; query head h reads K/V head h // (Hq // Hk). Query t of row b
    sees the own columns c <= col + t with c < lengths[b] or c >= prompt_cols
    (`lengths` (B,) int64: the row's prompt inside the padded prompt columns;
    None: every c <= col + t), and all of `prefix`. `col` is an int or a
    one-element int64 device tensor. Returns (B, T, Hq, D) contiguous; zeros
    for a query that sees nothing. What a column holds that none of the call's
    queries of its row sees does not matter (NaN included); with T > 1, a NaN
    in a column that a later query sees reaches the row's earlier ones too."""
    B, T, Hq, D = _heads(q, cache)
    dev, dt, Hk = cache.device, cache.dtype, cache.kv_heads
    lens = 0
    if lengths is not None:
        _tensor(lengths, "lengths", dev, torch.int64)
        _need(lengths.shape == (B,), f"lengths must be ({B},), not {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
        lens = lengths.data_ptr()
    P = pk = pv = 0
    if prefix is not None:
        if prefix.k.dtype is not dt or prefix.k.get_device() != dev.index:
            raise MEPError(f"the prefix must be {dt} on {dev}")
        _need(prefix.kv_heads == Hk and prefix.head_dim == D,
              "the prefix and the cache have different heads")
        _need(0 <= layer < prefix.layers, f"layer {layer} outside the prefix's {prefix.layers}")
        P, (pk, pv) = prefix.columns, prefix._ptrs[layer]
    _need(0 <= prompt_cols < 1 << 62, "prompt_cols must not be negative, up to 2^62 - 1")
    host, devcol = _column(col, dev)
    dc, code = _DTYPES[dt], cache._code
    nbytes = _attention_workspace(dc, code, B, T, Hq, Hk, D, cache.capacity, host, P)
    q, *qs = _rows(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    args = _lib.ATTENTION_ARGS.pack(
        dc, code, B, T, Hq, Hk, D, *qs, *cache.layer(layer), cache.capacity, lens, prompt_cols,
        host, devcol, pk, pv, P, scale, out.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes)
    with _on(dev) as stream:
        rc = _lib.lib().mep_cache_attention(args, stream)
    check(rc, None, "cache_attention")
    return out


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *,
                  return_logprobs: bool = False):
    """Next token of each row of `logits` (B, V) from one uniform number each
    (u: (B,) fp32 in [0, 1)): (B,) int64, and with `return_logprobs` the drawn
    tokens' log probabilities among the kept ones (fp32). Tokens are ordered by
    (logit descending, id ascending), w = exp((l - lmax) / temperature); kept
    are the first top_k (0: all), of those the ones whose preceding mass is
    below top_p of their mass, of those w >= min_p; the token is the first id,
    ascending, whose running kept weight exceeds u times its sum. Temperature 0
    (or NaN) takes the best token (lowest id). Each of temperature, top_p, min_p (fp32)
    and top_k (int32) is a number or a (B,) device tensor. A row whose logits
    are all -inf or NaN gives token -1."""
    _tensor(logits, "logits", None)
    dev = logits.device
    _need(logits.dtype in _DTYPES, f"logits are fp32 or bf16, not {logits.dtype}")
    _need(logits.dim() == 2 and logits.shape[1] > 0, "logits must be (rows, vocab)")
    B, V = logits.shape
    _tensor(u, "u", dev, torch.float32)
    _need(u.shape == (B,), f"u must be ({B},), not {tuple(u.shape)}")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    u = u.contiguous()
    ptrs, nums, keep = [], [], []
    for name, x, dt, num in (("temperature", temperature, torch.float32, float),
                             ("top_k", top_k, torch.int32, int),
                             ("top_p", top_p, torch.float32, float),
                             ("min_p", min_p, torch.float32, float)):
        if isinstance(x, torch.Tensor):
            _tensor(x, name, dev, dt)
            _need(x.shape == (B,), f"{name} must be a number or ({B},)")
            x = x.contiguous()
            keep.append(x)
            ptrs.append(x.data_ptr())
            nums.append(num(1))
        else:
            ptrs.append(None)
            # an integer far below 0 stays below it in 32 bits
            nums.append(max(min(num(x), 0x7fffffff), -1) if dt == torch.int32 else num(x))
    tokens = torch.empty(B, dtype=torch.int64, device=dev)
    logprobs = torch.empty(B, dtype=torch.float32, device=dev) if return_logprobs else None
    with _on(dev) as stream:
        check(_lib.lib().mep_sample(_DTYPES[logits.dtype], logits.data_ptr(), B, V,
                                    logits.stride(0), u.data_ptr(), *ptrs, *nums,
                                    tokens.data_ptr(),
                                    None if logprobs is None else logprobs.data_ptr(), stream),
              None, "sample_tokens")
    return (tokens, logprobs) if return_logprobs else tokens


@dataclass
class Sampler:
    """Filters of `sample_tokens` with a source of its uniform numbers: a
    generator on the logits' device, seeded with `seed` at the first draw. The
    same seed gives the same sequence of draws."""
    temperature: object = 1.0
    top_k: object = 0
    top_p: object = 1.0
    min_p: object = 0.0
    seed: int = 0

    def __post_init__(self):
        self._gen = None

    def uniform(self, *shape, device):
        """The next uniform numbers of the sequence."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if self._gen is None or self._gen.device != device:
            self._gen = torch.Generator(device=device)
            self._gen.manual_seed(self.seed)
        return torch.rand(*shape, generator=self._gen, device=device)

    def __call__(self, logits, u=None):
        if u is None:
            u = self.uniform(logits.shape[0], device=logits.device)
        return sample_tokens(logits, u, self.temperature, self.top_k, self.top_p, self.min_p)
