"""Plain 64-bit forms of the decode-step operators and the error bounds their
tests use (not collected as tests).

Half a rounding step relative to the value: bf16 2^-8, fp32 2^-24, e4m3 2^-4
(2^-10 absolute below its smallest normal number).
"""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FP32 = 2.0 ** -24


def rope_tables(rows, D, dtype=torch.float32, theta=10000.0, device="cuda"):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    ang = torch.cat((ang, ang), 1)
    return ang.cos().to(dtype).to(device), ang.sin().to(dtype).to(device)


def rotated(x, w, cos, sin, positions, eps):
    """(r, magnitude): the rotated head rows in 64 bits and |y c| + |y' s|."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    h = x.shape[-1] // 2
    other = torch.cat((-x[..., h:], x[..., :h]), -1)
    return x * c + other * s, (x * c).abs() + (other * s).abs()


def rotated_tol(ref, mag, dtype):
    """One rounding to `dtype`, and fp32 before it: a sum of D <= 128 squares
    in 8 + 4 steps, rsqrtf (2 ulp), two products for the norm, two products and
    a sum for the rotation, each within 2^-24 of its terms: below 32 of them."""
    return HALF[dtype] * ref.abs() + 32 * FP32 * mag


def quantised_tol(x, mag, dtype):
    """e4m3 rounding of the row scaled to 448, its dequantisation (two fp32
    roundings and two of the scale) and one rounding to `dtype`."""
    a = x.abs().amax(-1, keepdim=True)
    return (2.0 ** -4 + HALF[dtype] * 1.07 + 8 * FP32) * x.abs() + 2.0 ** -10 * a / 448 \
        + 34 * FP32 * (mag + a)


def visible(T, n, col, lengths, prompt, B, device):
    """(B, T, n) keep-mask of the own columns."""
    c = torch.arange(n, device=device)
    past = c <= col + torch.arange(T, device=device)[:, None]
    if lengths is None:
        return past[None].expand(B, T, n)
    return past[None] & ((c < lengths[:, None]) | (c >= prompt))[:, None]


def attention(q, k, v, keep, scale, kp=None, vp=None):
    """(out, tol terms): 64-bit attention of q (B, T, Hq, D) over k, v (B, Hk,
    n, D) in the columns `keep` (B, T, n), behind the shared kp, vp (Hk, P, D)."""
    B, T, Hq, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    q = q.double().view(B, T, Hk, G, D)
    k, v = k.double(), v.double()
    hidden = ~keep.any(1)[:, None, :, None]  # columns nobody sees: whatever they hold
    k, v = k.masked_fill(hidden, 0.0), v.masked_fill(hidden, 0.0)
    mask = keep[:, :, None, None]
    if kp is not None:
        k = torch.cat((kp.double()[None].expand(B, -1, -1, -1), k), 2)
        v = torch.cat((vp.double()[None].expand(B, -1, -1, -1), v), 2)
        mask = torch.cat((mask.new_ones(B, T, 1, 1, kp.shape[1]), mask), -1)
    s = torch.einsum("btkgd,bknd->btkgn", q, k) * scale
    s = s.masked_fill(~mask, -math.inf)
    some = mask.any(-1, keepdim=True)
    p = torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1) * mask
    out = torch.einsum("btkgn,bknd->btkgd", p, v).reshape(B, T, Hq, D)
    spread = torch.einsum("btkgn,bknd->btkgd", p, v.abs()).reshape(B, T, Hq, D)
    size = torch.einsum("btkgd,bknd->btkgn", q.abs(), k.abs()).masked_fill(~mask, 0).amax(-1)
    size = (size * abs(scale)).reshape(B, T, Hq, 1) if size.numel() else 0.0
    return out, spread, size, k.shape[2]


def attention_tol(out, spread, size, n, dtype, D, quantized):
    """|error| of an output, with a = sum p |v|:
      * its rounding to `dtype`;
      * each p rounded once to 16 bits before it meets v (bf16 models: 2^-8;
        fp32: split operands, 2^-20 left);
      * each score off by (D + 8) 2^-23 of scale * sum |q k| (D products summed
        in fp32 or split into two parts, the scales, the base-2 exponent), which
        moves numerator and denominator alike: twice;
      * the two sums of n terms in fp32: n 2^-24 each, plus 2^-20 for the
        exponential and the joining of partial sums.
    A quantised cache adds nothing: the reference reads the same codes, whose
    scales enter as factors (counted in the 8)."""
    p = HALF[dtype] if dtype == torch.bfloat16 else 2.0 ** -20
    score = (D + 8) * 2.0 ** -23 * size
    return HALF[dtype] * out.abs() + (p + 2 * torch.expm1(torch.as_tensor(score)) +
                                      2 * n * FP32 + 2.0 ** -20) * spread + 1e-30


def dequantised(codes, scale):
    return codes.double() * scale.double()[..., None]


def quantise(x):
    """(codes, scales) of rows along the last dimension."""
    x = x.float()
    a = x.abs().amax(-1)
    some = a >= 2.0 ** -100
    scale = torch.where(some, a / 448, torch.zeros_like(a))
    inv = torch.where(some, 448 / a, torch.zeros_like(a))
    return (x * inv[..., None]).to(torch.float8_e4m3fn), scale


def sample(logits, u, temperature, top_k, top_p, min_p):
    """(token, logprob, margin) of one row, lists and 64-bit floats: margin is
    the distance of u from the nearest border of the drawn token's share, and of
    top_p and min_p from theirs (a token closer than that cannot be decided)."""
    x = [float("-inf") if l != l else float(l) for l in logits]
    best = max(x)
    if best == float("-inf"):
        return -1, float("-inf"), 1.0
    ids = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if temperature == 0:
        return ids[0], 0.0, 1.0
    if top_k > 0:
        ids = ids[:top_k]

    def weight(l):
        return 1.0 if l == best else math.exp((l - best) / temperature)
    w = [weight(x[i]) for i in ids]
    margin = 1.0
    if top_p < 1:
        limit, run, n = top_p * math.fsum(w), 0.0, 0
        while n < len(w) and (n == 0 or run < limit):
            run += w[n]
            n += 1
            margin = min(margin, abs(run - limit)) if n < len(w) else margin
        ids, w = ids[:n], w[:n]
    kept = [(i, v) for i, v in zip(ids, w) if v >= min_p or i == ids[0]]
    # weights of 1 are exact and always kept
    margin = min([margin] + [abs(v - min_p) for v in w if min_p > 0 and v < 1])
    kept.sort()
    total = math.fsum(v for _, v in kept)
    run, target = 0.0, u * total
    for i, v in kept:
        run += v
        if v > 0:
            margin = min(margin, abs(run - target))
            last = (i, v)
        if run > target and v > 0:
            return i, math.log(v / total), margin
    return last[0], math.log(last[1] / total), margin
