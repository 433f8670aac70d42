"""CPU restatement, in 64 bits, of the paged cache, its attention and token scores
(test infrastructure; no reference counterpart). A cache is a dict of CPU tensors: k, v
(pages, heads, page_size, d) and, for e4m3 codes, k_scale, v_scale bytes."""
import math

import torch

E4M3, F64 = torch.float8_e4m3fn, torch.float64


def exponent(x):
    """e of rows (..., d): the smallest integer in [-100, 120] with amax <= 448 2^e, over the
    finite values."""
    a = x.double().abs()
    amax = torch.where(a < math.inf, a, torch.zeros_like(a)).amax(-1)
    e = torch.full(amax.shape, -100, dtype=torch.int64)
    for _ in range(220):
        e += (amax > 448 * torch.exp2(e.double())).long()
    return e


def codes(x):
    """e4m3 codes (..., d) and scale bytes of bf16 rows."""
    e = exponent(x)
    y = x.double() * torch.exp2(-e.double())[..., None]
    most = torch.where(e == 120, 240.0, 448.0).double()[..., None]           # 256 2^120 is no bf16 value any more
    y = torch.where(y.abs() < math.inf, torch.minimum(torch.maximum(y, -most), most), torch.full_like(y, math.nan))
    return y.float().to(E4M3), (e + 127).to(torch.uint8)


def values(c, name):
    """What the pages hold, 64 bits."""
    x = c[name].double()
    return x if c.get(name + "_scale") is None else x * torch.exp2(c[name + "_scale"].double() - 127)[..., None]


def places(table, lengths, starts, t, page_size, pages):
    """(sequence, position, page, slot) of each of t rows; page -1 where the row has no place,
    sequence -1 where it has none."""
    batch, width = table.shape
    starts = list(range(batch + 1)) if starts is None else starts.tolist()
    out = [(-1, -1, -1, 0)] * t
    for b in range(batch):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            pos = int(lengths[b]) - n + i
            page = int(table[b, pos // page_size]) if 0 <= pos < width * page_size else -1
            out[starts[b] + i] = (b, pos, page if 0 <= page < pages else -1, pos % page_size)
    return out


def write(c, k, v, table, lengths, starts=None):
    """Writes into c, in place."""
    pages, _, ps, _ = c["k"].shape
    rows = {"k": k, "v": v}
    held = {name: codes(x) if c["k"].dtype == E4M3 else (x, None) for name, x in rows.items()}
    for r, (_, _, page, slot) in enumerate(places(table, lengths, starts, k.shape[0], ps, pages)):
        if page >= 0:
            for name, (x, s) in held.items():
                c[name].view(torch.uint8 if s is not None else x.dtype)[page, :, slot] = \
                    x[r].view(torch.uint8) if s is not None else x[r]
                if s is not None:
                    c[name + "_scale"][page, :, slot] = s[r]


def read(c, table, lengths, starts, t):
    """(k, v), 64 bits."""
    pages, heads, ps, d = c["k"].shape
    out = []
    for name in ("k", "v"):
        x = values(c, name)
        y = torch.zeros(t, heads, d, dtype=F64)
        for r, (_, _, page, slot) in enumerate(places(table, lengths, starts, t, ps, pages)):
            if page >= 0:
                y[r] = x[page, :, slot]
        out.append(y)
    return out


def attend(c, q, table, lengths, starts=None, scale=None):
    """(o, a, most): the attention's rows (t, heads, d), the sums of p |v| that a relative error of
    the weights moves them by, and the largest sum of |q| |k| scale of a row, for error bounds."""
    pages, hk, ps, d = c["k"].shape
    t, hq, _ = q.shape
    scale = d ** -0.5 if scale is None else scale
    k, v = values(c, "k"), values(c, "v")
    o, a = torch.zeros(t, hq, d, dtype=F64), torch.zeros(t, hq, d, dtype=F64)
    most = 0.0
    rows = places(table, lengths, starts, t, ps, pages)
    for b in {r[0] for r in rows if r[0] >= 0 and r[1] >= 0}:
        mine = [i for i, r in enumerate(rows) if r[0] == b and r[1] >= 0]
        pos = torch.tensor([rows[i][1] for i in mine])
        keys = torch.arange(min(int(pos.max()) + 1, table.shape[1] * ps))
        page = table[b].long()[keys // ps]
        there = (page >= 0) & (page < pages)
        keys, page = keys[there], page[there]
        if not keys.numel():
            continue
        seen = keys <= pos[:, None]
        for h in range(hq):
            kk, vv, qq = k[page, h // (hq // hk), keys % ps], v[page, h // (hq // hk), keys % ps], q[mine, h].double()
            s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            p = torch.where(seen.any(1, keepdim=True), torch.softmax(s, 1), torch.zeros(1, dtype=F64))
            odd = (vv.abs() < math.inf).logical_not().any(1)
            fine = torch.where(odd[:, None], torch.zeros(1, dtype=F64), vv)
            out, size = p @ fine, p @ fine.abs()
            for j in odd.nonzero().flatten().tolist():      # unseen, such a value does not count
                add = torch.where(seen[:, j, None], p[:, j, None] * vv[j], torch.zeros(1, dtype=F64))
                out, size = out + add, size + add.abs()
            o[mine, h], a[mine, h] = out, size
            bound = torch.where(seen, qq.abs() @ kk.abs().T, torch.zeros(1, dtype=F64)).nan_to_num(0, posinf=0)
            most = max(most, float(bound.max()) * scale)
    return o, a, most


def log_softmax(x):
    """(log p, log sum e^(x - max)) of 64-bit rows, both exact to 64 bits where little is left beside
    the maximum."""
    m, at = x.max(1, keepdim=True)
    rest = (x - m).exp().scatter(1, at, 0.0).sum(1, keepdim=True).log1p()
    return x - m - rest, rest[:, 0]


def token_scores(logits, tokens, top=0):
    x = logits.double()
    t, v = x.shape
    odd = (x.isnan() | (x == math.inf)).any(1)
    none = (x == -math.inf).all(1)
    lp, _ = log_softmax(torch.where(odd[:, None] | none[:, None], torch.zeros_like(x), x))
    lp[none], lp[odd] = -math.inf, math.nan
    tok = tokens.reshape(t, -1)
    inside = (tok >= 0) & (tok < v)
    logprobs = torch.where(inside, lp.gather(1, tok.clamp(0, v - 1)), torch.zeros(1, dtype=F64))
    entropy = -torch.where(lp == -math.inf, torch.zeros_like(lp), lp.exp() * lp).sum(1)
    # falling values, NaN above them, the lowest index first among equals (both sorts keep the order of equals)
    ids = torch.where(x.isnan(), torch.full_like(x, math.inf), x).sort(dim=1, descending=True, stable=True).indices
    ids = ids.gather(1, x.gather(1, ids).isnan().int().sort(dim=1, descending=True, stable=True).indices)[:, :top]
    return logprobs.reshape(tokens.shape), entropy, lp.gather(1, ids), ids.to(torch.int32)
