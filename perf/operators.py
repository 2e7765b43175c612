"""The decode-step operators of miniep_b200 as measured cases: norm_rope_store
(with KVCache.read), cache_attention over a row's own cache, cache_attention
with a shared prefix, and sample_tokens, each beside its plain form in torch.

``own`` chooses the side: False computes the plain form (elementary torch
operations in 32 bits, 64 where a border decides), True calls the framework.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ELT = {"bf16": 2, "f32": 4}
E4M3_MAX = 448.0
# a K or V row whose largest magnitude is below this is stored as zeros
TINY = 2.0 ** -100


def _framework():
    root = str(Path(__file__).resolve().parents[1] / "mini-ep_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import miniep_b200
    return miniep_b200


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence, one token: what a single user's decode step waits for
        dict(name="store one token", op="store", B=1, T=1, Hq=16, Hk=8, D=64, dtype="bf16",
             quant=False, norm=False, cap=289, col=256, maxpos=4096),
        # a decode step of 64 sequences into a quantised cache, heads normalised
        dict(name="store step e4m3", op="store", B=64, T=1, Hq=16, Hk=8, D=64, dtype="bf16",
             quant=True, norm=True, cap=1152, col=1027, maxpos=4096),
        # prompts of an odd length written to a quantised cache and read back
        # for the prompt's own attention
        dict(name="store prompts e4m3", op="store", B=16, T=1021, Hq=32, Hk=8, D=128,
             dtype="bf16", quant=True, norm=True, cap=1153, col=0, maxpos=32768),
        # one sequence over a short context
        dict(name="attend one row", op="attend", B=1, T=1, Hq=16, Hk=8, D=64, dtype="bf16",
             quant=False, prompt=256, new=1, minlen=256, P=0),
        # the 64-sequence decode workload, half way through its 128 new tokens,
        # ragged prompts, quantised cache
        dict(name="attend 64 rows e4m3", op="attend", B=64, T=1, Hq=16, Hk=8, D=64, dtype="bf16",
             quant=True, prompt=1024, new=65, minlen=512, P=0),
        # long contexts: 1 GB of keys and values a step
        dict(name="attend long", op="attend", B=8, T=1, Hq=32, Hk=8, D=128, dtype="bf16",
             quant=False, prompt=32700, new=68, minlen=30000, P=0),
        # few rows behind a short common prompt, fp32 (the parity dtype)
        dict(name="prefix few rows f32", op="prefix", B=4, T=1, Hq=16, Hk=8, D=64, dtype="f32",
             quant=False, prompt=33, new=5, minlen=1, P=509),
        # a batch decoding behind one long common prompt, own columns quantised
        dict(name="prefix 64 rows", op="prefix", B=64, T=1, Hq=16, Hk=8, D=64, dtype="bf16",
             quant=True, prompt=100, new=29, minlen=20, P=4096),
        # the rows' own prompts prefilled behind the common one
        dict(name="prefix prompts", op="prefix", B=32, T=48, Hq=32, Hk=8, D=128, dtype="bf16",
             quant=False, prompt=48, new=0, minlen=9, P=4099),
        # one sequence sampling with the usual top-k and top-p
        dict(name="sample one row", op="sample", B=1, V=49155, dtype="bf16", mode="top_k_top_p"),
        # a batch whose rows ask for different filters, fp32 logits
        dict(name="sample 64 mixed", op="sample", B=64, V=49155, dtype="f32", mode="mixed"),
        # a large batch and vocabulary with a nucleus filter alone
        dict(name="sample 256 top_p", op="sample", B=256, V=100003, dtype="bf16", mode="top_p"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _heads(rng):
    """(Hq, Hk, D): the shapes of the framework's models and generic ones."""
    return rng.choice([(16, 8, 64), (4, 2, 64), (32, 8, 128), (8, 8, 64), (16, 2, 128),
                       (12, 4, 32), (24, 4, 80), (8, 1, 128)])


def _drawn(rng):
    op = rng.choice(["store", "attend", "prefix", "sample"])
    if op == "sample":
        return dict(op=op, B=_log_int(rng, 1, 256), V=_log_int(rng, 500, 100003),
                    dtype=rng.choice(["bf16", "f32"]),
                    mode=rng.choice(["plain", "greedy", "top_k", "top_p", "min_p", "top_k_top_p",
                                     "mixed"]))
    Hq, Hk, D = _heads(rng)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    quant = rng.random() < 0.5
    if op == "store":
        T = 1 if rng.random() < 0.4 else _log_int(rng, 2, 1021)
        col = _log_int(rng, 1, 2000)
        return dict(op=op, B=_log_int(rng, 1, 256), T=T, Hq=Hq, Hk=Hk, D=D, dtype=dtype,
                    quant=quant, norm=rng.random() < 0.5, cap=col + T + _log_int(rng, 1, 100),
                    col=col, maxpos=rng.choice([4096, 32768]))
    if op == "attend":
        T = 1 if rng.random() < 0.7 else _log_int(rng, 2, 16)
        prompt = _log_int(rng, 1, 32700)
        new = _log_int(rng, T, 128)
        return dict(op=op, B=_log_int(rng, 1, 128), T=T, Hq=Hq, Hk=Hk, D=D, dtype=dtype,
                    quant=quant, prompt=prompt, new=new, minlen=_log_int(rng, 1, prompt), P=0)
    if rng.random() < 0.3:  # the rows' prompts behind the prefix
        T = _log_int(rng, 2, 128)
        prompt, new = T, 0
    else:
        T, prompt, new = 1, _log_int(rng, 1, 1024), _log_int(rng, 1, 128)
    return dict(op=op, B=_log_int(rng, 1, 128), T=T, Hq=Hq, Hk=Hk, D=D, dtype=dtype, quant=quant,
                prompt=prompt, new=new, minlen=_log_int(rng, 1, prompt),
                P=_log_int(rng, 1, 16411))


def draw(rng):
    """A case of the same ranges, none costlier than its operator's largest listed one."""
    while True:
        c = _drawn(rng)
        most = [work(x) for x in listed() if x["op"] == c["op"]]
        w = work(c)
        # in 32 bits a product costs more than in 16: an eighth of the products there
        flops = w["flops"] * (8 if c["dtype"] == "f32" else 1)
        if w["bytes"] <= max(m["bytes"] for m in most) and \
                flops <= max(m["flops"] for m in most):
            return c


# ------------------------------------------------------------------ geometry
def _lengths(case):
    """The rows' prompt lengths, before prepare() shuffles them: from minlen to
    the padded length in even steps, so their sum does not hang on the seed."""
    B, lo, hi = case["B"], case["minlen"], case["prompt"]
    if B == 1:
        return [hi]
    return [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _col(case):
    """Cache column of the first query's own token."""
    return case["prompt"] + case["new"] - case["T"]


def _visible(case):
    """(own columns any query of row b sees, own keys over all its queries), summed over rows."""
    T, prompt, col = case["T"], case["prompt"], _col(case)
    cols = keys = 0
    for n in _lengths(case):
        seen = [min(n, col + t + 1) + max(0, col + t + 1 - prompt) for t in range(T)]
        cols += seen[-1]
        keys += sum(seen)
    return cols, keys


def work(case):
    e = ELT[case["dtype"]]
    if case["op"] == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * e + case["B"] * 32, "flops": 4 * n}
    B, T, Hq, Hk, D = (case[k] for k in ("B", "T", "Hq", "Hk", "D"))
    row = D + 4 if case["quant"] else D * e  # one cached row: codes and their scale
    if case["op"] == "store":
        n = B * T
        by = n * (2 * Hq + 2 * Hk) * D * e + 2 * n * Hk * row + n * 8
        by += min(n, case["maxpos"]) * 2 * D * 4
        if case["quant"]:
            by += 2 * n * Hk * (row + D * e)
        return {"bytes": by, "flops": 8 * n * (Hq + Hk) * D}
    cols, keys = _visible(case)
    by = 2 * B * T * Hq * D * e + 2 * cols * Hk * row + 2 * case["P"] * Hk * D * e
    return {"bytes": by, "flops": 4 * D * Hq * (keys + B * T * case["P"])}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _quantise(x):
    """(codes e4m3, scales fp32) of rows along the last dimension."""
    x = x.float()
    a = x.abs().amax(-1)
    some = a >= TINY
    scale = torch.where(some, a / E4M3_MAX, torch.zeros_like(a))
    inv = torch.where(some, E4M3_MAX / a, torch.zeros_like(a))
    return (x * inv.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def _rope_tables(maxpos, D, theta=10000.0):
    """(maxpos, D) fp32 cosines and sines, angles in 64 bits."""
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    ang = torch.arange(maxpos, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat((ang, ang), dim=1)
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "sample":
        B, V = case["B"], case["V"]
        # a language model's logits: a broad body and a few strong candidates
        x = torch.randn(B, V, generator=g, device="cuda") * 2.0
        hot = torch.randint(0, V, (B, 24), generator=g, device="cuda")
        x.scatter_add_(1, hot, 4.0 + 5.0 * torch.rand(B, 24, generator=g, device="cuda"))
        s["logits"] = x.to(dt)
        s["u"] = torch.rand(B, generator=g, device="cuda")
        ones, mode = torch.ones(B, device="cuda"), case["mode"]
        s["temperature"] = 0.8 * ones
        s["top_k"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["top_p"], s["min_p"] = ones.clone(), 0.0 * ones
        if mode == "greedy":
            s["temperature"] = 0.0 * ones
        if mode in ("top_k", "top_k_top_p"):
            s["top_k"] += 50
        if mode in ("top_p", "top_k_top_p"):
            s["top_p"] = 0.95 * ones
        if mode == "min_p":
            s["min_p"] = 0.05 * ones
        if mode == "mixed":
            s["temperature"] = 0.25 * torch.randint(0, 7, (B,), generator=g, device="cuda").float()
            s["top_k"] = torch.tensor([0, 1, 40, 1000], device="cuda", dtype=torch.int32)[
                torch.randint(0, 4, (B,), generator=g, device="cuda")]
            s["top_p"] = 0.5 + 0.5 * torch.rand(B, generator=g, device="cuda")
            s["top_p"][torch.rand(B, generator=g, device="cuda") < 0.3] = 1.0
            s["min_p"] = 0.1 * torch.rand(B, generator=g, device="cuda")
            s["min_p"][torch.rand(B, generator=g, device="cuda") < 0.5] = 0.0
        return s
    B, T, Hq, Hk, D = (case[k] for k in ("B", "T", "Hq", "Hk", "D"))
    if case["op"] == "store":
        # one projection's output, cut into its heads as a program cuts it
        qkv = _randn(g, (B, T, Hq + 2 * Hk, D), dt)
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        s["cos"], s["sin"] = _rope_tables(case["maxpos"], D)
        first = torch.randint(0, case["maxpos"] - T + 1, (B, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(T, device="cuda")
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = 1 + _randn(g, (D,), dt, 0.1)
            s["k_norm"] = 1 + _randn(g, (D,), dt, 0.1)
        shape = (1, B, Hk, case["cap"], D)
        store = torch.float8_e4m3fn if case["quant"] else dt
        s["k_cache"] = torch.zeros(shape, device="cuda", dtype=store)
        s["v_cache"] = torch.zeros(shape, device="cuda", dtype=store)
        s["k_scale"] = torch.zeros(shape[:-1], device="cuda") if case["quant"] else None
        s["v_scale"] = torch.zeros(shape[:-1], device="cuda") if case["quant"] else None
        return s
    s["q"] = _randn(g, (B, T, Hq, D), dt, 2.0)
    s["scale"] = 1.0 / math.sqrt(D)
    s["col"] = _col(case)
    n = torch.tensor(_lengths(case), device="cuda")
    s["lengths"] = n[torch.randperm(B, generator=g, device="cuda")]
    shape = (1, B, Hk, case["prompt"] + case["new"], D)
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g, device="cuda", dtype=dt)
        s[name + "_scale"] = None
        if case["quant"]:
            x, s[name + "_scale"] = _quantise(x)
        s[name + "_cache"] = x
        if case["P"]:
            s[name + "_prefix"] = torch.randn((1, Hk, case["P"], D), generator=g, device="cuda",
                                              dtype=dt)
    return s


# ------------------------------------------------------------------ plain forms
def _rotated(x, w, cos, sin, eps=1e-6):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()
    a, b = x.chunk(2, dim=-1)
    return x * cos + torch.cat((-b, a), dim=-1) * sin


def _plain_store(s):
    dt, col, T = s["q"].dtype, s["col"], s["T"]
    cos, sin = s["cos"][s["positions"]].unsqueeze(2), s["sin"][s["positions"]].unsqueeze(2)
    q = _rotated(s["q"], s["q_norm"], cos, sin).to(dt)
    k = _rotated(s["k"], s["k_norm"], cos, sin).transpose(1, 2)
    v = s["v"].transpose(1, 2)
    window = slice(col, col + T)
    if not s["quant"]:
        s["k_cache"][0, :, :, window] = k.to(dt)
        s["v_cache"][0, :, :, window] = v
        return {"q": q, "k": s["k_cache"][0, :, :, window], "v": s["v_cache"][0, :, :, window]}
    out = {"q": q}
    for name, x in (("k", k), ("v", v)):
        codes, scale = _quantise(x)
        s[name + "_cache"][0, :, :, window] = codes
        s[name + "_scale"][0, :, :, window] = scale
        out[name] = (s[name + "_cache"][0, :, :, window].float()
                     * s[name + "_scale"][0, :, :, window].unsqueeze(-1)).to(dt)
    return out


def _plain_attend(s):
    B, T, Hq, Hk, D = (s[k] for k in ("B", "T", "Hq", "Hk", "D"))
    G = Hq // Hk
    n = s["k_cache"].shape[3]
    k, v = s["k_cache"][0].float(), s["v_cache"][0].float()
    if s["quant"]:
        k, v = k * s["k_scale"][0].unsqueeze(-1), v * s["v_scale"][0].unsqueeze(-1)
    q = s["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4)  # B Hk G T D
    score = (q.reshape(B, Hk, G * T, D) @ k.transpose(2, 3)).view(B, Hk, G, T, n) * s["scale"]
    c = torch.arange(n, device="cuda")
    own_prompt = (c < s["lengths"][:, None]) | (c >= s["prompt"])  # B n
    past = c <= s["col"] + torch.arange(T, device="cuda")[:, None]  # T n
    seen = (own_prompt[:, None] & past)[:, None, None]  # B 1 1 T n
    score = score.masked_fill(~seen, -math.inf)
    if s["P"]:
        kp, vp = s["k_prefix"][0].float(), s["v_prefix"][0].float()  # Hk P D
        qp = q.permute(1, 0, 2, 3, 4).reshape(Hk, B * G * T, D)
        sp = (qp @ kp.transpose(1, 2)).mul_(s["scale"])
        sp = sp.view(Hk, B, G, T, s["P"]).permute(1, 0, 2, 3, 4)
        top = torch.maximum(score.amax(-1, keepdim=True), sp.amax(-1, keepdim=True))
    else:
        top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(B, Hk, G * T, n) @ v).view(B, Hk, G, T, D)
    if s["P"]:
        pp = (sp - top).exp()
        total = total + pp.sum(-1, keepdim=True)
        pp = pp.permute(1, 0, 2, 3, 4).reshape(Hk, B * G * T, s["P"])
        o = o + (pp @ vp).view(Hk, B, G, T, D).permute(1, 0, 2, 3, 4)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties: lowest id first
    t = s["temperature"].double()[:, None]
    rank = torch.arange(V, device=x.device)
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    w = torch.where(t > 0, w, (rank == 0).double())
    k = s["top_k"][:, None]
    w = w * ((k <= 0) | (rank < k))
    run = w.cumsum(1)
    before = torch.cat((torch.zeros_like(run[:, :1]), run[:, :-1]), dim=1)
    top_p = s["top_p"].double()[:, None]
    w = w * ((top_p >= 1) | (before < top_p * run[:, -1:]))
    w = w * (w >= s["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, w)  # back to the order of ids
    run = w.cumsum(1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(1)
    last = V - 1 - (w > 0).flip(1).int().argmax(1)
    token = torch.minimum(token, last)
    logprob = torch.log(w.gather(1, token[:, None]) / run[:, -1:])[:, 0]
    return {"tokens": token, "logprobs": logprob.float()}


# ------------------------------------------------------------------ run
def _cache(s, F):
    """The handle that a program keeps for its cache (no copy)."""
    if "handle" not in s:
        s["handle"] = F.KVCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                dtype=s["q"].dtype)
    return s["handle"]


def _own(s):
    F = _framework()
    if s["op"] == "sample":
        token, logprob = F.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"],
                                         s["top_p"], s["min_p"], return_logprobs=True)
        return {"tokens": token, "logprobs": logprob}
    cache = _cache(s, F)
    if s["op"] == "store":
        q = F.norm_rope_store(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], cache, 0,
                              s["col"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        end = s["col"] + s["T"]
        if s["quant"]:
            k, v = cache.read(0, s["col"], end)
        else:
            k, v = s["k_cache"][0, :, :, s["col"]:end], s["v_cache"][0, :, :, s["col"]:end]
        return {"q": q, "k": k, "v": v}
    prefix = None
    if s["P"]:
        if "prefix" not in s:
            s["prefix"] = F.SharedPrefix(s["k_prefix"], s["v_prefix"])
        prefix = s["prefix"]
    return F.cache_attention(s["q"], cache, 0, s["col"], s["scale"], lengths=s["lengths"],
                             prompt_cols=s["prompt"], prefix=prefix)


def run(state):
    if own:
        return _own(state)
    if state["op"] == "store":
        return _plain_store(state)
    if state["op"] == "sample":
        return _plain_sample(state)
    return _plain_attend(state)


# ------------------------------------------------------------------ exact
def _e4m3_grid(x):
    """Nearest e4m3 values (ties to even) of |x| <= 448, in 64 bits."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6)
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, e)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_store(s):
    D, half = s["D"], s["D"] // 2
    out = {}
    for name in ("q", "k", "v"):
        x = s[name].double()
        w = s.get(name + "_norm")
        if name != "v":
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
            c = s["cos"].double()[s["positions"]][:, :, None]
            n = s["sin"].double()[s["positions"]][:, :, None]
            lo, hi = x[..., :half], x[..., half:]
            x = torch.cat((lo * c[..., :half] - hi * n[..., :half],
                           hi * c[..., half:] + lo * n[..., half:]), dim=-1)
        if name != "q":
            x = x.transpose(1, 2)
            if s["quant"]:
                a = x.abs().amax(-1, keepdim=True) / E4M3_MAX
                x = torch.where(a > 0, _e4m3_grid(x / a.clamp_min(1e-300)) * a, 0 * x)
        out[name] = x
    return out


def _exact_attend(s):
    B, T, Hq, Hk, D = (s[k] for k in ("B", "T", "Hq", "Hk", "D"))
    G = Hq // Hk
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    n = s["k_cache"].shape[3]
    lens = s["lengths"].tolist()
    for b in range(B):
        # the row's visible columns: its prompt, then what it wrote after the padded prompts
        cols = torch.tensor([c for c in range(n) if c < lens[b] or c >= s["prompt"]],
                            device="cuda", dtype=torch.long)
        late = cols[None, :] > s["col"] + torch.arange(T, device="cuda")[:, None]  # T, columns
        for h in range(Hk):
            k, v = s["k_cache"][0, b, h].double()[cols], s["v_cache"][0, b, h].double()[cols]
            if s["quant"]:
                k = k * s["k_scale"][0, b, h].double()[cols, None]
                v = v * s["v_scale"][0, b, h].double()[cols, None]
            hide = late
            if s["P"]:
                k = torch.cat((s["k_prefix"][0, h].double(), k))
                v = torch.cat((s["v_prefix"][0, h].double(), v))
                hide = torch.cat((torch.zeros(T, s["P"], dtype=torch.bool, device="cuda"), late), 1)
            x = s["q"][b, :, h * G:(h + 1) * G].double() @ k.T * s["scale"]  # T G keys
            x = x.masked_fill(hide[:, None], -math.inf)
            some = torch.isfinite(x).any(-1, keepdim=True)
            p = torch.softmax(torch.where(some, x, torch.zeros_like(x)), dim=-1)
            out[b, :, h * G:(h + 1) * G] = torch.where(some, p @ v, torch.zeros_like(p @ v))
    return out


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    u, temp, top_p, min_p = (s[k].double().cpu().numpy()
                             for k in ("u", "temperature", "top_p", "min_p"))
    top_k = s["top_k"].cpu().numpy()
    tokens, logprobs = [], []
    for row in range(logits.shape[0]):
        x = logits[row]
        if temp[row] == 0:
            tokens.append(int(np.argmax(x)))
            logprobs.append(0.0)
            continue
        ids = np.argsort(-x, kind="stable")
        if top_k[row] > 0:
            ids = ids[:top_k[row]]
        w = np.exp((x[ids] - x[ids[0]]) / temp[row])
        if top_p[row] < 1:
            mass = np.cumsum(w)
            n = 1 + int(np.searchsorted(mass[:-1], top_p[row] * mass[-1], side="left"))
            ids, w = ids[:n], w[:n]
        ids, w = ids[w >= min_p[row]], w[w >= min_p[row]]
        by_id = np.argsort(ids)
        ids, w = ids[by_id], w[by_id]
        mass = np.cumsum(w)
        at = min(int(np.searchsorted(mass, u[row] * mass[-1], side="right")), len(ids) - 1)
        tokens.append(int(ids[at]))
        logprobs.append(math.log(w[at] / mass[-1]))
    return {"tokens": torch.tensor(tokens), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_attend(s)
