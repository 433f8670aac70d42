"""CPU restatement, in 64 bits, of the block-scaled FP8 linear, of expert routing and
of the experts' products (test infrastructure; no reference counterpart)."""
import math

import torch

E4M3, F32, F64 = torch.float8_e4m3fn, torch.float32, torch.float64
BLOCK = 128


def expand(scale, n, k):
    """Block scales as one value per weight, 64 bits."""
    return scale.double().repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def dequant(codes, scale):
    return codes.double() * expand(scale, *codes.shape[-2:])


def quant_weight(w):
    """Codes and block scales (32-bit quotients) of a bf16 weight (n, k)."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pad = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    amax = pad.reshape(nb, BLOCK, kb, BLOCK).abs().amax((1, 3)).clamp(min=1e-12)
    scale = amax / torch.full_like(amax, 448)
    return (w.float() / expand(scale, n, k).float()).clamp(-448, 448).to(E4M3), scale


def quant_rows(x):
    """Codes (m, 128 kb) and scales (kb, m) of bf16 rows, 32-bit quotients."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    g = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).reshape(m, kb, BLOCK)
    amax = g.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    scale = amax / torch.full_like(amax, 448)
    codes = (g / scale).clamp(-448, 448).to(E4M3)
    return codes.reshape(m, kb * BLOCK), scale[..., 0].T.contiguous()


def rows_values(codes, scale, k):
    """The values that quantised rows stand for, (m, k) 64 bits."""
    return (codes.double().reshape(codes.shape[0], -1, BLOCK) * scale.T.double()[..., None]).reshape(codes.shape)[:, :k]


def sum_error(a, w):
    """Bound on the matrix instruction's error in a . w^T (values, 64 bits): it aligns
    each block of 32 products to the largest and keeps 13 bits or more, an error of at
    most 2^-14 of the largest for each of the 32."""
    m, k = a.shape
    kb = -(-k // 32)
    a = torch.nn.functional.pad(a.abs(), (0, kb * 32 - k)).reshape(m, kb, 32)
    w = torch.nn.functional.pad(w.abs(), (0, kb * 32 - k)).reshape(w.shape[0], kb, 32)
    out = torch.zeros(m, w.shape[0], dtype=F64)
    for b in range(kb):
        for r in range(0, m, 16):
            out[r:r + 16] += (a[r:r + 16, None, b] * w[None, :, b]).amax(-1)
    return out * 32 * 2.0 ** -14


def linear(x, codes, scale):
    """(y, bound on the kernel's distance from it): one bf16 rounding and ``sum_error``."""
    q, s = quant_rows(x)
    a, w = rows_values(q, s, x.shape[1]), dequant(codes, scale)
    y, e = a @ w.T, sum_error(a, w)
    return y, 2.0 ** -8 * (y.abs() + e) + e


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """Row by row with Python sorting."""
    t, e = logits.shape
    top_groups = groups if top_groups is None else top_groups
    weights, ids = torch.zeros(t, top_k, dtype=F64), torch.full((t, top_k), -1, dtype=torch.int32)
    for r in range(t):
        l = [float(v) for v in logits[r].double()]
        b = [0.0] * e if bias is None else [float(v) for v in bias.double()]
        if any(math.isnan(v) for v in l + b) or (score == "softmax" and math.inf in l):
            weights[r], ids[r] = math.nan, torch.arange(top_k, dtype=torch.int32)
            continue
        on = [j for j in range(e) if l[j] != -math.inf]
        if score == "softmax":
            top = max((l[j] for j in on), default=0.0)
            z = math.fsum(math.exp(l[j] - top) for j in on)
            p = {j: math.exp(l[j] - top) / z for j in on}
        else:
            p = {j: 1 / (1 + math.exp(-l[j])) if l[j] > -700 else 0.0 for j in on}
        # without a bias by logit: scores rise with it, and those that round to the same number keep their order
        c = {j: l[j] if bias is None else p[j] + b[j] for j in on}
        if groups > 1:
            per, best = e // groups, []
            for g in range(groups):
                s = sorted((c[j] for j in on if j // per == g and c[j] != -math.inf), reverse=True)
                best.append((s[0] + (s[1] if bias is not None and len(s) > 1 else 0.0)) if s else -math.inf)
            keep = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
            c = {j: v for j, v in c.items() if j // per in keep}
        chosen = sorted((j for j in c if c[j] != -math.inf), key=lambda j: (-c[j], j))[:top_k]
        total = sum(p[j] for j in chosen)
        for n, j in enumerate(chosen):
            ids[r, n] = j
            weights[r, n] = (p[j] / total if total > 0 else 0.0) * scale if renormalize else p[j] * scale
    return weights, ids


def experts(x, weights, ids, gate_up, gate_up_scale, down, down_scale):
    """y (t, h), 64 bits, the SwiGLU's values unrounded, and a bound on the kernel's distance."""
    t, h = x.shape
    q, s = quant_rows(x)
    a = rows_values(q, s, h)
    y, err = torch.zeros(t, h, dtype=F64), torch.zeros(t, h, dtype=F64)
    for e in range(gate_up.shape[0]):
        tok, slot = (ids == e).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        wg, wu = (dequant(gate_up[e, p], gate_up_scale[e, p]) for p in (0, 1))
        g, u = a[tok] @ wg.T, a[tok] @ wu.T
        eg, eu = sum_error(a[tok], wg), sum_error(a[tok], wu)
        sg = g * torch.sigmoid(g)
        mid = sg * u
        # |silu'| <= 1.1; one bf16 rounding; 2^-20: the 32-bit exp, quotient and products
        em = 1.1 * eg * u.abs() + (sg.abs() + 1.1 * eg) * eu + (2.0 ** -8 + 2.0 ** -20) * mid.abs()
        em = em * (1 + 2.0 ** -7)
        wd = dequant(down[e], down_scale[e])
        w = weights[tok, slot].double()[:, None]
        y.index_put_((tok,), w * (mid @ wd.T), accumulate=True)
        # fp32 sums of i products: one rounding each
        err.index_put_((tok,), w.abs() * ((em + (mid.shape[1] + 8) * 2.0 ** -24 * (mid.abs() + em)) @ wd.abs().T),
                       accumulate=True)
    return y, 2.0 ** -8 * (y.abs() + err) + err
