"""The decode-step operators on a B200 against plain 64-bit forms: cache write
with head norms and rotation, reading a quantised cache back, attention over
the cache and a shared prefix, sampling."""
import math

import pytest
import torch

import decode_ref as R
from gpu_util import require_gpu
from miniep_b200 import (KVCache, MEPError, Sampler, SharedPrefix, _lib, cache_attention,
                         norm_rope_store, sample_tokens)

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def within(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), (got.double() - ref).abs().max().item(),
                           ((got.double() - ref).abs() / tol).max().item())


# ------------------------------------------------------------- cache write
STORE = [  # B, T, Hq, Hk, D, cap, col
    (1, 1, 16, 8, 64, 9, 4), (3, 1, 4, 2, 64, 5, 0), (2, 37, 32, 8, 128, 40, 3),
    (5, 2, 12, 4, 32, 17, 15), (2, 3, 24, 4, 80, 8, 1), (1, 70, 2, 2, 16, 70, 0),
    (2, 5, 8, 1, 112, 11, 2), (33, 1, 6, 3, 48, 4, 3)]


@pytest.mark.parametrize("shape", STORE, ids=str)
@pytest.mark.parametrize("dtype,quant", [(BF, False), (BF, True), (F32, False), (F32, True)],
                         ids=["bf16", "bf16-e4m3", "f32", "f32-e4m3"])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_store(shape, dtype, quant, norm):
    B, T, Hq, Hk, D, cap, col = shape
    g = gen(hash(shape) % 1000)
    qkv = randn(g, B, T, Hq + 2 * Hk, D, dtype=dtype, std=3.0)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    cos, sin = R.rope_tables(3000, D, F32 if D != 80 else dtype)
    pos = torch.randint(0, 3000, (B, T), generator=g, device="cuda")
    qn = 1 + randn(g, D, dtype=dtype, std=0.2) if norm else None
    kn = 1 + randn(g, D, dtype=dtype, std=0.2) if norm and D != 32 else None
    cache = KVCache.empty(2, B, Hk, cap, D, dtype, quantized=quant)
    before = [t.clone() for t in (cache.k, cache.v)]
    out = norm_rope_store(q, k, v, cos, sin, pos, cache, 1, col, q_norm=qn, k_norm=kn, eps=1e-5)
    assert out.shape == (B, T, Hq, D) and out.is_contiguous()
    ref, mag = R.rotated(q, qn, cos, sin, pos, 1e-5)
    within(out, ref, R.rotated_tol(ref, mag, dtype))
    kr, vr = cache.read(1, col, col + T)
    ref, mag = (t.transpose(1, 2) for t in R.rotated(k, kn, cos, sin, pos, 1e-5))
    vt = v.transpose(1, 2).double()
    if quant:
        within(kr, ref, R.quantised_tol(ref, mag, dtype))
        within(vr, vt, R.quantised_tol(vt, vt.abs(), dtype))
        # reading back is code * scale, rounded once
        window = (1, slice(None), slice(None), slice(col, col + T))
        for got, codes, scale in ((kr, cache.k, cache.k_scale), (vr, cache.v, cache.v_scale)):
            exact = R.dequantised(codes[window], scale[window])
            within(got, exact, R.HALF[dtype] * exact.abs())
    else:
        within(kr, ref, R.rotated_tol(ref, mag, dtype))
        assert torch.equal(vr, v.transpose(1, 2))
    # nothing else is written
    for t, was in zip((cache.k, cache.v), before):
        t = t.clone()
        t[1, :, :, col:col + T] = was[1, :, :, col:col + T]
        assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


def test_store_strides_positions_and_streams():
    """Heads-major inputs, positions broadcast over rows, another stream."""
    g = gen(1)
    B, T, Hq, Hk, D = 3, 6, 8, 4, 64
    q = randn(g, B, Hq, T, D, dtype=BF).transpose(1, 2)
    k = randn(g, T, B, Hk, D, dtype=BF).transpose(0, 1)
    v = randn(g, B, T, Hk, D + 1, dtype=BF)[..., 1:]  # rows off the 16-byte grid
    cos, sin = R.rope_tables(64, D)
    pos = torch.arange(7, 7 + T, device="cuda")[None]
    cache = KVCache.empty(1, B, Hk, 8, D, BF)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = norm_rope_store(q, k, v, cos, sin, pos, cache, 0, 2)
    s.synchronize()
    ref, mag = R.rotated(q, None, cos, sin, pos.expand(B, T), 0.0)
    within(out, ref, R.rotated_tol(ref, mag, BF))
    assert torch.equal(cache.v[0, :, :, 2:], v.transpose(1, 2))
    assert not cache.v[0, :, :, :2].any()


def test_store_column_on_the_device():
    """A device column advances under replays; columns outside the cache and
    positions outside the tables touch nothing outside them."""
    g = gen(2)
    B, T, Hq, Hk, D, cap = 2, 2, 4, 2, 64, 5
    q, k, v = (randn(g, B, T, h, D, dtype=BF) for h in (Hq, Hk, Hk))
    cos, sin = R.rope_tables(16, D)
    pos = torch.zeros(B, T, dtype=torch.long, device="cuda")
    for quant in (False, True):
        cache = KVCache.empty(1, B, Hk, cap, D, BF, quantized=quant)
        col = torch.zeros(1, dtype=torch.long, device="cuda")
        graph = torch.cuda.CUDAGraph()
        norm_rope_store(q, k, v, cos, sin, pos, cache, 0, col)
        with torch.cuda.graph(graph):
            norm_rope_store(q, k, v, cos, sin, pos, cache, 0, col)
        want = cache.read(0, 0, T)[1].clone()
        for c in (-1, 1, 4, 5, 1 << 40):
            cache.k.zero_(), cache.v.zero_()
            col.fill_(c)
            graph.replay()
            got = cache.read(0, 0, cap)[1] if not quant else None
            codes = cache.v[0].float()
            for t in range(T):
                if 0 <= c + t < cap:
                    assert codes[:, :, c + t].any()
                    if got is not None:
                        assert torch.equal(got[:, :, c + t], want[:, :, t])
            rest = [x for x in range(cap) if not c <= x < c + T]
            assert not codes[:, :, rest].any()
    pos[1, 1] = 16
    pos[0, 0] = -1
    cache = KVCache.empty(1, B, Hk, cap, D, BF)
    out = norm_rope_store(q, k, v, cos, sin, pos, cache, 0, 0)
    nan = out.isnan().all(-1).all(-1)
    assert nan.tolist() == [[True, False], [False, True]]
    assert cache.k[0, 0, :, 0].isnan().all() and not cache.k[0, 0, :, 1].isnan().any()
    assert not cache.v.isnan().any()


@pytest.mark.parametrize("heads", [(8, 8, 64), (6, 6, 16), (1, 1, 128), (7, 7, 80), (5, 5, 48)],
                         ids=str)
@pytest.mark.parametrize("B,T", [(2, 3), (4, 1900)], ids=str)
def test_store_quantised_rows_of_zeros_among_others(heads, B, T):
    """Rows of zeros and of numbers too small to scale in one pass of a warp
    with others, lanes without a row, one pass a warp and several."""
    Hq, Hk, D = heads
    g = gen(D + T)
    q, k, v = (randn(g, B, T, h, D, dtype=BF, std=2.0) for h in (Hq, Hk, Hk))
    for x in (k, v):
        kind = torch.randint(0, 3, x.shape[:3], generator=g, device="cuda")
        x[kind == 1] = 0
        x[kind == 2] *= torch.where(torch.rand(int((kind == 2).sum()), 1, generator=g,
                                               device="cuda") < 0.5, 2.0 ** -110, 1.0).to(BF)
    cos, sin = R.rope_tables(64, D)
    pos = torch.randint(0, 64, (B, T), generator=g, device="cuda")
    cache = KVCache.empty(1, B, Hk, T + 2, D, BF, quantized=True)
    norm_rope_store(q, k, v, cos, sin, pos, cache, 0, 1)
    kr, vr = cache.read(0, 1, 1 + T)
    ref, mag = (t.transpose(1, 2) for t in R.rotated(k, None, cos, sin, pos, 0.0))
    vt = v.transpose(1, 2).double()
    for got, codes, scale, want, size in ((kr, cache.k, cache.k_scale, ref, mag),
                                          (vr, cache.v, cache.v_scale, vt, vt.abs())):
        tiny = want.abs().amax(-1) < 2.0 ** -100
        assert not got[tiny].any() and not scale[0, :, :, 1:1 + T][tiny].any()
        assert not codes[0, :, :, 1:1 + T].float()[tiny].any()
        want = want.masked_fill(tiny[..., None], 0.0)
        within(got, want, R.quantised_tol(want, size.masked_fill(tiny[..., None], 0.0), BF))


def test_store_quantised_extremes():
    """Rows of zeros, of tiny and of huge numbers; a NaN stays one."""
    D = 64
    rows = torch.zeros(6, 1, 1, D)
    rows[1] = 2.0 ** -101
    rows[2] = 2.0 ** -99
    rows[3] = 3e38
    rows[4, 0, 0, 5] = 7.0
    rows[5, 0, 0, 3] = math.nan
    rows[5, 0, 0, 4] = 1.0
    rows = rows.cuda()
    cos, sin = torch.ones(1, D, device="cuda"), torch.zeros(1, D, device="cuda")
    cache = KVCache.empty(1, 6, 1, 1, D, F32, quantized=True)
    norm_rope_store(rows, rows, rows, cos, sin, torch.zeros(6, 1, dtype=torch.long, device="cuda"),
                    cache, 0, 0)
    for x in cache.read(0, 0, 1):
        x = x[:, 0, 0].cpu()
        assert not x[0].any() and not x[1].any()
        assert (x[2] / 2.0 ** -99 - 1).abs().max() <= 8 * R.FP32
        assert (x[3] / 3e38 - 1).abs().max() <= 8 * R.FP32
        assert abs(x[4, 5] / 7 - 1) <= 8 * R.FP32 and x[4].count_nonzero() == 1
        assert x[5, 3].isnan() and x[5, 4] == 1.0


def test_read_many_heads():
    """More (row, head) pairs than a grid dimension holds."""
    B, Hk, D = 8200, 8, 16
    x = randn(gen(40), 1, B, Hk, 2, D)
    codes, scale = R.quantise(x)
    cache = KVCache(codes, codes, scale, scale, dtype=F32)
    for got in cache.read(0, 1, 2):
        want = R.dequantised(codes, scale)[0, :, :, 1:2]
        within(got, want, R.HALF[F32] * want.abs())


@pytest.mark.parametrize("quant", [False, True], ids=["plain", "e4m3"])
def test_prefix_from_a_row_of_a_cache(quant):
    """One row's columns of every layer, from a layout whose rows lie off the
    16-byte grid of the scales; the other rows cost no memory."""
    g = gen(41)
    for L, B, Hk, cap, D, columns in ((3, 5, 3, 7, 48, 5), (1, 2, 1, 1, 16, 1), (2, 3, 2, 4, 64, 0),
                                      (4, 64, 8, 1024, 64, 1000)):
        k, v = randn(g, L, B, Hk, cap, D), randn(g, L, B, Hk, cap, D)
        if quant:
            (kc, ks), (vc, vs) = R.quantise(k), R.quantise(v)
            cache = KVCache(kc, vc, ks, vs, dtype=BF)
        else:
            cache = KVCache(k.to(BF), v.to(BF))
        del k, v
        row = B - 1
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        prefix = SharedPrefix.from_cache(cache, row, columns)
        # the result, and what it is gathered from
        took = torch.cuda.max_memory_allocated() - before
        assert took <= 3 * (2 * L * Hk * columns * D * 2) + L * 4096 + 4096
        assert prefix.k.shape == (L, Hk, columns, D)
        for l in range(L):
            want = cache.read(l, 0, columns)
            assert torch.equal(prefix.k[l], want[0][row]) and torch.equal(prefix.v[l], want[1][row])


def test_store_and_read_of_nothing():
    cache = KVCache.empty(1, 0, 2, 4, 64, BF, quantized=True)
    q, k = torch.empty(0, 1, 4, 64, dtype=BF, device="cuda"), torch.empty(0, 1, 2, 64, dtype=BF, device="cuda")
    cos, sin = R.rope_tables(4, 64)
    pos = torch.empty(0, 1, dtype=torch.long, device="cuda")
    assert norm_rope_store(q, k, k, cos, sin, pos, cache, 0, 1).shape == (0, 1, 4, 64)
    cache = KVCache.empty(1, 2, 2, 4, 64, BF, quantized=True)
    q, k = torch.empty(2, 0, 4, 64, dtype=BF, device="cuda"), torch.empty(2, 0, 2, 64, dtype=BF, device="cuda")
    pos = torch.empty(2, 0, dtype=torch.long, device="cuda")
    assert norm_rope_store(q, k, k, cos, sin, pos, cache, 0, 4).shape == (2, 0, 4, 64)
    assert cache.read(0, 3, 3)[0].shape == (2, 2, 0, 64)
    assert cache_attention(q, cache, 0, 4, 1.0).shape == (2, 0, 4, 64)


# --------------------------------------------------------------- attention
HEADS = [(16, 8, 64), (4, 2, 64), (32, 8, 128), (12, 4, 32), (24, 4, 80), (8, 1, 128),
         (40, 1, 64), (3, 3, 16), (6, 2, 48), (4, 4, 112)]
SPANS = [  # B, T, prompt, new, minimum length
    (1, 1, 0, 1, 0), (1, 1, 256, 1, 256), (3, 1, 100, 7, 0), (2, 3, 64, 5, 1), (2, 1, 1000, 60, 3),
    (5, 16, 16, 0, 1), (2, 70, 70, 0, 5), (1, 1, 5000, 1, 5000)]
KINDS = [(BF, False), (BF, True), (F32, False), (F32, True)]
KIND_IDS = ["bf16", "bf16-e4m3", "f32", "f32-e4m3"]


def make(g, heads, span, dtype, quant, P=0, std=2.0, layers=2):
    Hq, Hk, D = heads
    B, T, prompt, new, lo = span
    cap = prompt + new + 3
    q = randn(g, B, T, Hq, D, dtype=dtype, std=std)
    k, v = randn(g, layers, B, Hk, cap, D), randn(g, layers, B, Hk, cap, D)
    lengths = torch.randint(lo, prompt + 1, (B,), generator=g, device="cuda")
    if quant:
        (k, ks), (v, vs) = R.quantise(k), R.quantise(v)
        cache = KVCache(k, v, ks, vs, dtype=dtype)
        kd, vd = R.dequantised(k, ks), R.dequantised(v, vs)
    else:
        cache = KVCache(k.to(dtype), v.to(dtype))
        kd, vd = cache.k.double(), cache.v.double()
    prefix = SharedPrefix(randn(g, layers, Hk, P, D, dtype=dtype),
                          randn(g, layers, Hk, P, D, dtype=dtype)) if P else None
    return q, cache, kd, vd, lengths, prompt + new - T, prefix


def attend_case(seed, heads, span, dtype, quant, P=0, use_lengths=True):
    g = gen(seed)
    q, cache, kd, vd, lengths, col, prefix = make(g, heads, span, dtype, quant, P)
    B, T, prompt = span[0], span[1], span[2]
    D = heads[2]
    scale = 1 / math.sqrt(D)
    if not use_lengths:
        lengths = None
    got = cache_attention(q, cache, 1, col, scale, lengths=lengths, prompt_cols=prompt,
                          prefix=prefix)
    keep = R.visible(T, cache.capacity, col, lengths, prompt, B, "cuda")
    out, spread, size, n = R.attention(q, kd[1], vd[1], keep, scale,
                                       *((prefix.k[1], prefix.v[1]) if P else ()))
    within(got, out, R.attention_tol(out, spread, size, n, dtype, D, quant))
    return got


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("span", SPANS, ids=str)
def test_attention(span, heads, dtype, quant):
    attend_case(3, heads, span, dtype, quant)


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("heads", HEADS[:6], ids=str)
@pytest.mark.parametrize("span,P", [((1, 1, 4, 1, 0), 1), ((4, 1, 33, 5, 1), 509),
                                    ((70, 1, 9, 2, 0), 128), ((3, 48, 48, 0, 9), 127),
                                    ((2, 1, 600, 9, 1), 1300), ((33, 5, 5, 0, 1), 257)], ids=str)
def test_attention_with_prefix(span, P, heads, dtype, quant):
    attend_case(4, heads, span, dtype, quant, P)


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("heads,span", [((4, 2, 64), (2, 1024, 1024, 0, 5)),
                                        ((8, 2, 128), (2, 333, 333, 0, 1)),
                                        ((6, 1, 80), (1, 1021, 1500, 300, 900))], ids=str)
@pytest.mark.parametrize("P", [0, 200])
def test_attention_of_whole_prompts(P, heads, span, dtype, quant):
    """What a prefill asks for: every token of ragged prompts at once over the
    prompt's own columns, and a later part of one over what was there before."""
    attend_case(12, heads, span, dtype, quant, P)


def test_attention_without_lengths():
    for P in (0, 77):
        attend_case(5, (16, 8, 64), (3, 4, 130, 9, 1), BF, True, P, use_lengths=False)


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
def test_attention_masked_places_hold_anything(dtype, quant):
    """NaN and infinities in columns that no query of the row sees (padding,
    columns not yet written) change nothing; a row that sees nothing is zero."""
    heads, span = (8, 2, 64), (4, 2, 90, 6, 0)
    for P in (0, 40):
        g = gen(6)
        q, cache, kd, vd, lengths, col, prefix = make(g, heads, span, dtype, quant, P)
        lengths[0], lengths[1] = 0, 90
        prompt = 90 + 6 + 1  # beyond every visible column: row 0 sees no own key
        args = dict(lengths=lengths, prompt_cols=prompt, prefix=prefix)
        keep = R.visible(2, cache.capacity, col, lengths, prompt, 4, "cuda")
        out, spread, size, n = R.attention(q, kd[1], vd[1], keep, 0.1,
                                           *((prefix.k[1], prefix.v[1]) if P else ()))
        hidden = ~keep.any(1)[:, None].expand(-1, 2, -1)
        for t in (cache.k, cache.v):
            t[1].view(torch.uint8 if quant else dtype)[hidden] = 0x7f if quant else math.nan
        if quant:
            cache.k_scale[1][hidden] = math.inf
            cache.v_scale[1][hidden] = math.nan
        got = cache_attention(q, cache, 1, col, 0.1, **args)
        within(got, out, R.attention_tol(out, spread, size, n, dtype, 64, quant))
        if not P:
            assert not got[0].any()


def test_attention_large_scores_and_signs():
    """Scores far apart (one key takes all) and a negative scale."""
    for dtype in (BF, F32):
        g = gen(7)
        q, cache, kd, vd, lengths, col, _ = make(g, (8, 4, 64), (2, 1, 300, 2, 200), dtype, False,
                                                 std=30.0)
        for scale in (1.0, -1.0):
            got = cache_attention(q, cache, 0, col, scale, lengths=lengths, prompt_cols=300)
            keep = R.visible(1, cache.capacity, col, lengths, 300, 2, "cuda")
            out, spread, size, n = R.attention(q, kd[0], vd[0], keep, scale)
            within(got, out, R.attention_tol(out, spread, size, n, dtype, 64, False))


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("heads,T", [((8, 2, 64), 1), ((8, 1, 128), 1), ((12, 1, 32), 1),
                                     ((8, 2, 64), 24), ((4, 2, 80), 3)], ids=str)
@pytest.mark.parametrize("gap", [6, 14, 17, 21, 28, 45])
def test_attention_weights_far_below_the_largest(gap, heads, T, dtype, quant):
    """A key far above the others in score and far below them in value (at the
    first, a middle or the last column): what the others weigh still counts, in
    equal and in unequal measure. Where the values grow as the weights fall, the
    same in turn."""
    Hq, Hk, D = heads
    g = gen(gap + T)
    B, n, scale = 6, 700, 0.125
    q = (1 + 0.05 * randn(g, B, T, Hq, D)).to(dtype)
    k, v = 0.02 * randn(g, 1, B, Hk, n, D), randn(g, 1, B, Hk, n, D)
    v.abs_()  # nothing cancels
    at = [0, 3, 350, 500, n - T, 0]
    for b in range(B):
        k[0, b, :, at[b]] = gap / (D * scale)
        v[0, b, :, at[b]] *= (0.0, 2.0 ** -60, 2.0 ** -75, 0.0, 2.0 ** -60, 1e-3)[b]
    # the last row: a tenth of the others is larger by what it lies lower
    k[0, -1, :, 7::10] = -gap / (D * scale)
    v[0, -1, :, 7::10] *= math.exp(gap)
    if quant:
        (k, ks), (v, vs) = R.quantise(k), R.quantise(v)
        cache = KVCache(k, v, ks, vs, dtype=dtype)
        kd, vd = R.dequantised(k, ks), R.dequantised(v, vs)
    else:
        cache = KVCache(k.to(dtype), v.to(dtype))
        kd, vd = cache.k.double(), cache.v.double()
    col = n - T
    got = cache_attention(q, cache, 0, col, scale)
    keep = R.visible(T, n, col, None, 0, B, "cuda")
    out, spread, size, m = R.attention(q, kd[0], vd[0], keep, scale)
    within(got, out, R.attention_tol(out, spread, size, m, dtype, D, quant))


@pytest.mark.parametrize("dtype,quant", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("heads,T", [((8, 2, 64), 1), ((8, 1, 128), 2), ((12, 1, 32), 1),
                                     ((8, 2, 64), 24), ((4, 2, 80), 3)], ids=str)
@pytest.mark.parametrize("by", [10, 16, 22, 28])
def test_attention_queries_with_one_large_value(by, heads, T, dtype, quant):
    """One value of a query 2^by times the others, where the keys are zero: the
    others decide, with all their bits."""
    Hq, Hk, D = heads
    g = gen(by + T)
    B, n = 3, 300
    q = randn(g, B, T, Hq, D)
    q[..., 5] = 2.0 ** by
    q = q.to(dtype)
    k, v = randn(g, 1, B, Hk, n, D), randn(g, 1, B, Hk, n, D)
    k[..., 5] = 0
    if quant:
        (k, ks), (v, vs) = R.quantise(k), R.quantise(v)
        cache = KVCache(k, v, ks, vs, dtype=dtype)
        kd, vd = R.dequantised(k, ks), R.dequantised(v, vs)
    else:
        cache = KVCache(k.to(dtype), v.to(dtype))
        kd, vd = cache.k.double(), cache.v.double()
    got = cache_attention(q, cache, 0, n - T, 0.5)
    keep = R.visible(T, n, n - T, None, 0, B, "cuda")
    out, spread, size, m = R.attention(q, kd[0], vd[0], keep, 0.5)
    within(got, out, R.attention_tol(out, spread, size, m, dtype, D, quant))


@pytest.mark.parametrize("heads", [(16, 8, 64), (32, 8, 128), (4, 2, 16), (8, 8, 80)], ids=str)
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_attention_prefix_with_growing_scores(heads, scale):
    """A large batch behind a prefix whose later keys weigh more and more (each
    step of keys raises the maximum far beyond the last), or less and less."""
    Hq, Hk, D = heads
    for B, P, up in ((160, 700, True), (160, 700, False), (300, 65, True)):
        g = gen(B + P)
        q = randn(g, B, 1, Hq, D, dtype=BF).abs()
        grow = torch.linspace(0.0, 40.0, P, device="cuda")
        kp = randn(g, 1, Hk, P, D) * 0.3 + (grow if up else grow.flip(0))[:, None] * 8 / D
        prefix = SharedPrefix(kp.to(BF), randn(g, 1, Hk, P, D, dtype=BF))
        cache = KVCache(randn(g, 1, B, Hk, 4, D, dtype=BF), randn(g, 1, B, Hk, 4, D, dtype=BF))
        got = cache_attention(q, cache, 0, 2, scale, prefix=prefix)
        keep = R.visible(1, 4, 2, None, 0, B, "cuda")
        out, spread, size, n = R.attention(q, cache.k[0], cache.v[0], keep, scale, prefix.k[0],
                                           prefix.v[0])
        within(got, out, R.attention_tol(out, spread, size, n, BF, D, False))


@pytest.mark.parametrize("quant", [False, True], ids=["plain", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_attention_scale_zero_weighs_every_seen_column_alike(dtype, quant):
    """Masked columns stay out at a scale of 0, one of -0, and one so small that
    it vanishes against small queries."""
    for heads, span, P in (((8, 4, 64), (2, 1, 300, 2, 200), 0),
                           ((8, 4, 64), (2, 3, 70, 5, 1), 37),
                           ((16, 8, 64), (160, 1, 5, 2, 1), 333)):
        g = gen(17)
        q, cache, kd, vd, lengths, col, prefix = make(g, heads, span, dtype, quant, P)
        B, T, prompt = span[:3]
        kp, vp = (None, None) if prefix is None else (prefix.k[0], prefix.v[0])
        keep = R.visible(T, cache.capacity, col, lengths, prompt, B, "cuda")
        for scale, by in ((0.0, 1.0), (-0.0, 1.0), (1e-30, 1e-30)):
            x = q * by
            got = cache_attention(x, cache, 0, col, scale, lengths=lengths, prompt_cols=prompt,
                                  prefix=prefix)
            out, spread, size, n = R.attention(x, kd[0], vd[0], keep, scale, kp, vp)
            within(got, out, R.attention_tol(out, spread, size, n, dtype, heads[2], quant))


def test_attention_prefix_far_larger_than_a_run():
    """Key tiles dealt over all SMs, tiles cut between them, tails of a tile."""
    for heads, B, P in (((2, 1, 64), 64, 20001), ((16, 8, 64), 1100, 333), ((8, 1, 128), 33, 4097)):
        attend_case(11, heads, (B, 1, 5, 2, 0), BF, True, P)


@pytest.mark.parametrize("heads,B,P,last", [((16, 8, 64), 300, 1300, 3),
                                            ((32, 8, 128), 200, 2500, 4),
                                            ((32, 8, 128), 1500, 700, 7),
                                            ((8, 1, 128), 33, 4097, 3)], ids=str)
def test_attention_prefix_that_gives_up_leaves_no_finite_row(heads, B, P, last):
    """Loads that stop early, as after a wait that ran out: every row is NaN or,
    where all its keys had been read, what it is without; nothing is left in
    flight, and the next call is whole."""
    Hq, Hk, D = heads
    g = gen(B)
    q = randn(g, B, 1, Hq, D, dtype=BF)
    cache = KVCache(randn(g, 1, B, Hk, 6, D, dtype=BF), randn(g, 1, B, Hk, 6, D, dtype=BF))
    prefix = SharedPrefix(randn(g, 1, Hk, P, D, dtype=BF), randn(g, 1, Hk, P, D, dtype=BF))
    want = cache_attention(q, cache, 0, 3, 0.1, prefix=prefix)
    assert torch.isfinite(want.float()).all()
    try:
        for loads in (0, 1, 2, 3, last):  # the workspace holds the last call's sums
            _lib.lib().mep_debug_prefix_loads(loads)
            got = cache_attention(q, cache, 0, 3, 0.1, prefix=prefix)
            _lib.lib().mep_debug_prefix_loads(-1)
            nan = got.isnan()
            assert torch.equal(nan.any(-1), nan.all(-1))
            lost = nan.all(-1)
            assert lost.all() if loads == 0 else lost.any()
            assert torch.equal(got[~lost], want[~lost])
            again = cache_attention(q, cache, 0, 3, 0.1, prefix=prefix)
            assert torch.equal(again, want)
    finally:
        _lib.lib().mep_debug_prefix_loads(-1)


@pytest.mark.parametrize("quant", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("P", [0, 300])
def test_attention_replayed_with_a_device_column(P, quant):
    """Two captured graphs, each with its own workspace, replayed in turn on
    two streams while the column advances, against eager calls."""
    span = (3, 1, 500, 40, 1)
    sets = []
    for seed in (8, 9):
        q, cache, _, _, lengths, _, prefix = make(gen(seed), (16, 8, 64), span, BF, quant, P)
        col = torch.full((1,), 500, dtype=torch.long, device="cuda")
        call = lambda c, q=q, cache=cache, lengths=lengths, prefix=prefix: cache_attention(  # noqa: E731
            q, cache, 1, c, 0.125, lengths=lengths, prompt_cols=500, prefix=prefix)
        call(col)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(col)
        sets.append((call, graph, out, col, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for c in (500, 501, 520, 539):
        for _, graph, _, col, s in sets:
            with torch.cuda.stream(s):
                col.fill_(c)
                graph.replay()
        torch.cuda.synchronize()
        for call, _, out, _, _ in sets:
            want = call(c)
            # another split of the columns may sum in another order
            d = (out.float() - want.float()).abs()
            assert (d <= 2 * R.HALF[BF] * want.float().abs() + 2.0 ** -8).all()


def test_attention_repeats_bit_for_bit():
    q, cache, _, _, lengths, col, prefix = make(gen(10), (16, 8, 64), (8, 1, 3000, 60, 1), BF, True,
                                                700)
    first = cache_attention(q, cache, 0, col, 0.125, lengths=lengths, prompt_cols=3000,
                            prefix=prefix)
    for _ in range(5):
        again = cache_attention(q, cache, 0, col, 0.125, lengths=lengths, prompt_cols=3000,
                                prefix=prefix)
        assert torch.equal(first, again)


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^32 bytes (and 2^32 elements in e4m3): the last
    row and head read their own columns."""
    free, _ = torch.cuda.mem_get_info()
    if free < 14 << 30:
        pytest.skip("needs 14 GB of free memory")
    B, Hk, D, cap = 9, 8, 64, 1 << 20
    codes = torch.zeros(1, B, Hk, cap, D, dtype=torch.uint8, device="cuda")
    k = codes.view(torch.float8_e4m3fn)
    scale = torch.ones(1, B, Hk, cap, device="cuda")
    cache = KVCache(k, k, scale, scale, dtype=BF)
    assert k.numel() > 1 << 32
    start = cap - 4
    for b in range(B):
        codes[0, b, :, start:] = torch.tensor(b + 1.0).to(torch.float8_e4m3fn).view(torch.uint8)
    q = torch.zeros(B, 1, 16, D, dtype=BF, device="cuda")
    got = cache_attention(q, cache, 0, cap - 1, 1.0, lengths=torch.zeros(B, dtype=torch.long, device="cuda"),
                          prompt_cols=start)
    want = torch.tensor([float(torch.tensor(b + 1.0).to(torch.float8_e4m3fn)) for b in range(B)])
    assert torch.equal(got[:, 0, 15, 63].float().cpu(), want)
    assert torch.equal(cache.read(0, cap - 1, cap)[0][:, 7, 0, 63].float().cpu(), want)


# ---------------------------------------------------------------- sampling
def draw_rows(logits, u, temperature, top_k, top_p, min_p):
    tok, lp = sample_tokens(logits, u, temperature, top_k, top_p, min_p, return_logprobs=True)
    B = logits.shape[0]
    # numbers reach the kernel in fp32
    pick = lambda x, i: x[i].item() if isinstance(x, torch.Tensor) else \
        x if isinstance(x, int) else torch.tensor(x).item()  # noqa: E731
    rows, us = logits.float().cpu().tolist(), u.cpu().tolist()
    undecided = 0
    for i in range(B):
        want, logp, margin = R.sample(rows[i], us[i], *(pick(x, i) for x in
                                                        (temperature, top_k, top_p, min_p)))
        # weights and sums are exact to V * 2^-44 of the best token's weight
        if margin <= len(rows[i]) * 2.0 ** -43:
            undecided += 1
            continue
        assert tok[i].item() == want, (i, margin)
        # the logarithm's fp32 rounding, and weights to 2^-43 of themselves
        # above 2^-16 of the best (2^-27 over all that can be drawn here)
        if math.isfinite(logp):
            assert abs(lp[i].item() - logp) <= 2 * R.FP32 * abs(logp) + 2.0 ** -24
        else:
            assert lp[i].item() == logp
    assert undecided <= B // 8
    return tok


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1),
           (0.8, 40, 0.95, 0.02), (0.0, 5, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (2.0, 3000, 0.3, 0.0),
           (1.0, 1 << 30, 0.999, 0.0), (0.05, 20, 0.9, 0.0), (5.0, 0, 0.99, 0.001),
           (1.0, 0, 1e-6, 0.0), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("filt", FILTERS, ids=str)
def test_sample(filt, dtype):
    for B, V in ((4, 1), (7, 37), (3, 1024), (5, 4099), (2, 49155)):
        g = gen(V)
        logits = randn(g, B, V, dtype=dtype, std=3.0)
        u = torch.rand(B, generator=g, device="cuda")
        draw_rows(logits, u, *filt)


def test_sample_rows_of_their_own_and_strides():
    g = gen(20)
    B, V = 24, 5003
    for dtype in (BF, F32):
        whole = randn(g, B, V + 13, dtype=dtype, std=2.5)
        logits = whole[:, 5:5 + V]  # odd start and row stride
        u = torch.rand(B, generator=g, device="cuda")
        t = torch.linspace(0, 2, B, device="cuda")
        k = torch.randint(0, 200, (B,), generator=g, device="cuda", dtype=torch.int32)
        p = 0.2 + torch.rand(B, generator=g, device="cuda")
        m = 0.2 * torch.rand(B, generator=g, device="cuda")
        draw_rows(logits, u, t, k, p, m)
        wide = randn(g, V, B, dtype=dtype).T  # vocabulary not contiguous
        draw_rows(wide, u, t, k, p, m)


@pytest.mark.parametrize("filt", [(1.0, 0, 1.0, 0.0), (3.0, 5000, 0.9, 0.0), (4.0, 0, 0.9, 1e-4),
                                  (1.0, 20000, 1.0, 0.0), (9.0, 30000, 0.5, 0.0)], ids=str)
def test_sample_wide_rows_and_nuclei(filt):
    """Thousands of tokens kept, vocabularies past what a CTA keeps on chip."""
    for V, dtype in ((40001, F32), (262147, BF), (700001, BF), (400003, F32)):
        g = gen(V)
        logits = randn(g, 2, V, dtype=dtype, std=2.0)
        draw_rows(logits, torch.rand(2, generator=g, device="cuda"), *filt)
    tied = torch.randint(0, 3, (4, 30011), generator=gen(1), device="cuda").float()
    draw_rows(tied, torch.rand(4, generator=gen(2), device="cuda"), *filt)


def test_sample_small_and_large_logits():
    """16-bit rows around zero (values below 2^-9 and the border among them),
    all negative, far from zero, and wider than the table of values."""
    for V in (300, 20011):
        for scale, shift in ((1e-3, 0.0), (4e-3, 0.0), (0.05, 0.0), (1.0, -9.0), (1.0, 300.0),
                             (900.0, 0.0), (30.0, 5000.0), (1e-6, 2e-3), (10.0, 100.0)):
            g = gen(V)
            logits = (randn(g, 3, V) * scale + shift).to(BF)
            u = torch.rand(3, generator=g, device="cuda")
            for filt in ((1.0, 0, 1.0, 0.0), (0.5, 100, 0.7, 0.0), (0.7, 0, 0.6, 1e-3),
                         (1e-3, 0, 0.9, 0.0), (2.0, 150, 1.0, 0.2)):
                draw_rows(logits, u, *filt)


@pytest.mark.parametrize("top,temps", [(5.0, (3.7, 3.85)), (-100.0, (0.7, 0.79))], ids=str)
def test_sample_values_past_the_end_of_the_table(top, temps):
    """16-bit rows whose smallest weights lie near -127, with tokens below them
    (finite ones, -inf, NaN) and, where the best is positive, around zero."""
    inf, nan = math.inf, math.nan
    pool = [top, top - 1, top - 2, -119.0, -123.5, -126.0, -127.0, -127.5, -128.0, -200.0, -inf,
            nan, -nan]
    if top > 0:
        pool += [1e-4, -1e-4, 1.9e-3, -1.9e-3, 2e-3, 0.0, -0.0, 1.0, -1.0]
    for B, V in ((3, 9001), (150, 4200)):
        g = gen(V)
        at = torch.randint(0, len(pool), (B, V), generator=g, device="cuda")
        logits = torch.tensor(pool, device="cuda").to(BF)[at]
        u = torch.rand(B, generator=g, device="cuda")
        for temp in temps:
            for k, p in (((0, 1.0), (300, 1.0), (V // 2, 0.9), (V - 1, 1.0), (V + 5, 0.9999999),
                          (0, 0.9999999), (0, 0.3)) if B == 3 else ((V // 2, 0.9), (0, 1.0))):
                draw_rows(logits, u, temp, k, p, 0.0)


def test_sample_every_row_count():
    """Row counts that change how many CTAs share a row."""
    for B in (1, 9, 18, 37, 74, 150, 300):
        g = gen(B)
        logits = randn(g, B, 8200, dtype=BF, std=2.0)
        draw_rows(logits, torch.rand(B, generator=g, device="cuda"), 0.9, 30, 0.9, 0.0)


@pytest.mark.parametrize("rows,V", [(1, 32705), (1, 32770), (36, 32770), (1, 32768), (37, 16346),
                                    (73, 16384), (73, 16420), (74, 8177), (147, 8180),
                                    (147, 8184)], ids=str)
@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "shifted"])
def test_sample_last_run_of_a_row_shorter_than_the_others(rows, V, aligned):
    """Unfiltered 16-bit rows whose runs lie about 4096 ids, the row's last run
    below it and the others not: all CTAs of a row go the same way."""
    g = gen(V + rows)
    pad = (-V) % 8 if aligned else 9 + V % 2  # an odd row stride: every start there is
    whole = randn(g, rows, V + pad, dtype=BF, std=2.0)
    logits = whole[:, :V] if aligned else whole[:, 1:1 + V]
    u = torch.rand(rows, generator=g, device="cuda")
    for filt in ((1.0, 0, 1.0, 0.0), (0.8, 0, 1.0, 0.01)):
        draw_rows(logits, u, *filt)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_sample_short_runs_on_several_ctas(dtype):
    """Rows just long enough for several CTAs each, whose first pass is over at
    once, in many calls: the largest logit comes from every CTA's run."""
    for rows, V in ((1, 1024), (37, 1025), (74, 1024), (147, 2047), (9, 8192), (36, 8193)):
        g = gen(V)
        for i in range(20):
            logits = randn(g, rows, V, dtype=dtype)
            at = torch.randint(0, V, (rows,), generator=g, device="cuda")
            logits[torch.arange(rows, device="cuda"), at] = 60.0  # the others' share: V e^-54
            u = torch.rand(rows, generator=g, device="cuda") * 0.999
            assert torch.equal(sample_tokens(logits, u, 0.0), at)
            assert torch.equal(sample_tokens(logits, u, 1.0), at)
            assert torch.equal(sample_tokens(logits, u, 1.0, 3, 0.9), at)


def test_sample_ties_take_the_lowest_ids():
    """Equal logits: exact shares, kept from the lowest id up."""
    for V in (16, 1000, 40000):
        logits = torch.zeros(8, V, device="cuda")
        u = torch.tensor([0.0, 0.1251, 0.2501, 0.3751, 0.5001, 0.6251, 0.7501, 0.9999],
                         device="cuda")
        n = V // 2
        tok = sample_tokens(logits, u, 1.0, 0, 0.5)
        assert tok.tolist() == [int(x * n) for x in u.tolist()]
        tok = sample_tokens(logits, u, 1.0, n, 0.5)
        assert tok.tolist() == [int(x * (n // 2)) for x in u.tolist()]
        assert sample_tokens(logits, u, 0.0).tolist() == [0] * 8
        logits[:, V // 4:] += 1  # ties at the border of top_k
        tok = sample_tokens(logits, u, 1.0, 8)
        assert tok.tolist() == [V // 4 + int(x * 8) for x in u.tolist()]
    x = torch.zeros(1, 64, device="cuda")
    x[0, ::2] = -0.0  # equal to +0
    assert sample_tokens(x, torch.tensor([0.999], device="cuda"), 1.0, 4).item() == 3


def test_sample_infinities_nan_and_bounds():
    inf, nan = math.inf, math.nan
    rows = [([-inf] * 5, -1), ([nan] * 5, -1), ([nan, -inf, 1.0, nan, -inf], 2),
            ([0.0, inf, 1.0, inf, nan], 3), ([-inf, -3e38, -inf, -inf, -inf], 1),
            ([3e38, -3e38, 0, 0, 0], 0)]
    for dtype in (F32, BF):
        logits = torch.tensor([r for r, _ in rows]).to(dtype).cuda()
        u = torch.full((len(rows),), 0.75, device="cuda")
        for filt in ((1.0, 0, 1.0, 0.0), (1.0, 2, 0.9, 0.1), (0.3, 4, 1.0, 0.0)):
            tok, lp = sample_tokens(logits, u, *filt, return_logprobs=True)
            assert tok.tolist() == [t for _, t in rows]
            assert lp[0].item() == -inf and lp[3].item() == pytest.approx(math.log(0.5), rel=1e-6)
        assert sample_tokens(logits, u, 0.0).tolist() == [-1, -1, 2, 1, 1, 0]
    logits = torch.zeros(4, 10, device="cuda")
    u = torch.tensor([0.0, 1.0, 2.0, nan], device="cuda")
    assert sample_tokens(logits, u).tolist() == [0, 9, 9, 0]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [5, 3001, 70001])
def test_sample_infinite_logits_at_any_temperature(V, dtype):
    """+inf logits share the mass even where 34 temperatures pass fp32's range,
    and finite ones share it alike where the temperature is infinite."""
    inf = math.inf
    logits = randn(gen(V), 8, V, dtype=dtype)
    at = torch.tensor([1, V // 2, V - 2], device="cuda")
    logits[:4, at] = inf
    u = torch.tensor([0.0, 0.34, 0.67, 0.99] * 2, device="cuda")
    for t in (1.0, 1e37, 3e38, inf):
        temp = torch.full((8,), t, device="cuda")
        for k, p, m in ((0, 1.0, 0.0), (0, 1.0, 0.3), (3, 1.0, 0.0), (0, 0.9999, 0.0),
                        (4, 0.9999, 0.0)):
            tok, lp = sample_tokens(logits, u, temp, k, p, m, return_logprobs=True)
            assert tok[:4].tolist() == [at[0].item(), at[1].item(), at[2].item(), at[2].item()]
            assert ((lp[:4] + math.log(3)).abs() <= 2 * R.FP32 * math.log(3)).all()
        if t == inf:  # every finite logit weighs the same
            want = (u[4:].double() * V).floor().long()
            assert torch.equal(sample_tokens(logits, u, temp)[4:], want)


def test_sample_row_values_outside_their_ranges():
    """Per-row values cannot be refused without waiting for them: each has a
    meaning (temperature below 0 or NaN: greedy; top_k below 0: all; top_p not
    above 0: the best token; min_p above 1: as 1; NaN: no filter)."""
    nan = math.nan
    for dtype, V in ((F32, 700), (BF, 700), (BF, 70000)):
        logits = randn(gen(V), 8, V, dtype=dtype)
        ids = torch.arange(V, device="cuda")
        best = torch.where(logits == logits.amax(1, keepdim=True), ids, V).amin(1)
        u = torch.full((8,), 0.999, device="cuda")
        ones = torch.ones(8, device="cuda")
        zero = torch.zeros(8, dtype=torch.int32, device="cuda")
        for t, k, p, m in ((-ones, zero, ones, 0 * ones), (nan * ones, zero, ones, 0 * ones),
                           (ones, zero, -ones, 0 * ones), (ones, zero, 0 * ones, 0 * ones)):
            assert torch.equal(sample_tokens(logits, u, t, k, p, m), best)
        free = sample_tokens(logits, u)
        for k, p, m in ((zero - 3, ones, 0 * ones), (zero, nan * ones, 0 * ones),
                        (zero, 2 * ones, -ones), (zero, ones, nan * ones)):
            assert torch.equal(sample_tokens(logits, u, ones, k, p, m), free)
        assert torch.equal(sample_tokens(logits, u, ones, zero, ones, 7 * ones),
                           sample_tokens(logits, u, 1.0, 0, 1.0, 1.0))


def test_sampler_draws_on():
    """One seed, one sequence, whichever way the device is named."""
    a, b = Sampler(seed=5), Sampler(seed=5)
    x = a.uniform(3, device="cuda"), a.uniform(3, device="cuda")
    y = b.uniform(3, device="cuda:0"), b.uniform(3, device=torch.device("cuda", 0))
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    assert not torch.equal(x[0], x[1])


def test_sample_replays_and_repeats():
    g = gen(30)
    logits = randn(g, 16, 49155, dtype=BF, std=2.0)
    u = torch.rand(16, generator=g, device="cuda")
    filt = (0.9, 100, 0.9, 0.01)
    sample_tokens(logits, u, *filt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok = sample_tokens(logits, u, *filt)
    for _ in range(3):
        logits.copy_(randn(g, 16, 49155, std=2.0))
        u.copy_(torch.rand(16, generator=g, device="cuda"))
        graph.replay()
        assert torch.equal(tok, sample_tokens(logits, u, *filt))
    assert sample_tokens(logits[:0], u[:0]).shape == (0,)


def test_sample_shares_follow_the_probabilities():
    """Over a grid of u every kept token is drawn in its share, off by at most
    one grid point at each of its two borders."""
    n = 4096
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tok = sample_tokens(logits.expand(n, 5), u)
    share = torch.bincount(tok, minlength=5).double() / n
    want = torch.softmax(logits.double(), 0)
    assert ((share - want).abs() <= 2 / n).all()


def test_refusals_on_the_gpu():
    cache = KVCache.empty(2, 2, 2, 8, 64, BF)
    q = torch.zeros(2, 1, 4, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 1, 2, 64, dtype=BF, device="cuda")
    cos, sin = R.rope_tables(8, 64)
    pos = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    store = lambda **kw: norm_rope_store(*[kw.get(n, d) for n, d in (  # noqa: E731
        ("q", q), ("k", k), ("v", k), ("cos", cos), ("sin", sin), ("pos", pos), ("cache", cache),
        ("layer", 0), ("col", 0))], q_norm=kw.get("q_norm"))
    store()
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:1]), dict(k=k[:, :, :1]),
                dict(v=k.cpu()), dict(cos=cos[:, :32]), dict(cos=cos.half()), dict(pos=pos.int()),
                dict(pos=pos.expand(2, 3)), dict(layer=2), dict(layer=-1), dict(col=8),
                dict(col=-1), dict(col=torch.zeros(1, device="cuda")), dict(q_norm=cos[0]),
                dict(q=torch.zeros(2, 1, 3, 64, dtype=BF, device="cuda")),
                dict(q=q.clone().requires_grad_())):
        with pytest.raises(MEPError):
            store(**bad)
    with torch.no_grad():
        store(q=q.clone().requires_grad_())
    n = torch.zeros(2, dtype=torch.long, device="cuda")
    cache_attention(q, cache, 0, 0, 1.0, lengths=n)
    prefix = SharedPrefix(*[torch.zeros(1, 2, 3, 64, dtype=BF, device="cuda")] * 2)
    other = SharedPrefix(*[torch.zeros(1, 1, 3, 64, dtype=BF, device="cuda")] * 2)
    for args, kw in (((q, cache, 0, 8, 1.0), {}), ((q, cache, 0, 0, 1.0), dict(lengths=n.int())),
                     ((q, cache, 0, 0, 1.0), dict(lengths=n[:1])),
                     ((q, cache, 1, 0, 1.0), dict(prefix=prefix)),
                     ((q, cache, 0, 0, 1.0), dict(prefix=other)),
                     ((q, cache, 0, 0, 1.0), dict(lengths=n, prompt_cols=-1)),
                     ((q.float(), cache, 0, 0, 1.0), {})):
        with pytest.raises(MEPError):
            cache_attention(*args, **kw)
    e4 = cache.k.to(torch.float8_e4m3fn)
    s = torch.zeros(2, 2, 2, 8, device="cuda")
    for args in ((cache.k, cache.v[:1]), (cache.k, cache.v.float()), (e4, e4), (e4, e4, s, s[:1]),
                 (cache.k, cache.v, s, s), (cache.k.half(), cache.v.half()),
                 (cache.k.transpose(1, 2), cache.v.transpose(1, 2)), (e4, e4, s, s, torch.half)):
        with pytest.raises(MEPError):
            KVCache(*args)
    with pytest.raises(MEPError):
        cache.read(0, 5, 9)
    with pytest.raises(MEPError):
        SharedPrefix.from_cache(cache, 2, 4)
    small = KVCache.empty(1, 1, 1, 4, 24, BF)
    with pytest.raises(MEPError, match="head_dim"):
        cache_attention(torch.zeros(1, 1, 1, 24, dtype=BF, device="cuda"), small, 0, 0, 1.0)
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for args in ((x.half(), u), (x[0], u), (x, u[:1]), (x, u.double()), (x, u.cpu()), (x, u, -1.0),
                 (x, u, math.inf), (x, u, math.nan), (x, u, 1.0, -1), (x, u, 1.0, 0, 0.0),
                 (x, u, 1.0, 0, 1.0, 1.5), (x, u, u.double()), (x, u, u[:1]), (x, u, 1.0, u)):
        with pytest.raises(MEPError):
            sample_tokens(*args)


@pytest.mark.parametrize("col", [-1, 1 << 62, (1 << 63) - 1, 1 << 63, 1 << 70, -(1 << 63) - 1])
def test_columns_past_64_bits_are_refused(col):
    cache = KVCache.empty(1, 2, 2, 8, 64, BF)
    q, k = (torch.zeros(2, 1, h, 64, dtype=BF, device="cuda") for h in (4, 2))
    cos, sin = R.rope_tables(8, 64)
    pos = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    with pytest.raises(MEPError):
        norm_rope_store(q, k, k, cos, sin, pos, cache, 0, col)
    with pytest.raises(MEPError):
        cache_attention(q, cache, 0, col, 1.0)
    with pytest.raises(MEPError):
        cache_attention(q, cache, 0, 0, 1.0, prompt_cols=col)


@pytest.mark.parametrize("k", [-1, -(1 << 31) - 1, 5 - (1 << 32), 5 - (1 << 64)])
def test_negative_top_k_is_refused(k):
    with pytest.raises(MEPError, match="top_k"):
        sample_tokens(torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda"), 1.0, k)
