"""Performance cases of the block-scaled FP8 linear and of the mixture-of-experts
operators: what a serving program has each of them do, from the single token of
a decode step to a long prompt.

Three operators, each reached through the package's public entry points:

* ``linear``: ``linear.BlockFP8Linear``, e4m3 weights with one fp32 scale for
  every 128 x 128 block, activations quantised per row and 128 channels;
* ``route``: ``moe.route``, the experts of each token and their weights from the
  router's logits;
* ``experts``: ``moe.Experts``, the chosen experts' gate/up products (on quantised rows,
  as ``linear``), SwiGLU, down products (on the SwiGLU's unquantised values) and their
  weighted sum, all on block-scaled FP8 weights.

``listed`` holds the standing cases, ``draw`` makes more of the same ranges.
``run`` computes a case in its plain form (elementary torch operations in 32 bits)
or, where ``own`` is true, through the package; ``exact`` gives the operator's
definition in 64 bits.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
DEVICE = "cuda"
BLOCK = 128


def listed():
    return [
        # one row through the 8B o projection: a decode step's linear, the smallest call
        dict(name="linear_8b_o_row", kind="linear", m=1, n=4096, k=4096),
        # seven rows (a small ragged decode batch) through the 4B gate/up: weight-bound
        dict(name="linear_4b_gateup_7", kind="linear", m=7, n=19456, k=2560),
        # the benchmark's 576-token prompt through the 8B qkv
        dict(name="linear_8b_qkv_576", kind="linear", m=576, n=6144, k=4096),
        # the vision MLP's real width (4304 = 33 blocks and 80 channels), an odd number of rows
        dict(name="linear_ragged_333", kind="linear", m=333, n=1152, k=4304),
        # the 32B down projection over a long prompt: the largest product
        dict(name="linear_32b_down_4096", kind="linear", m=4096, n=5120, k=25600),
        # one token's choice among 128 experts, softmax scores renormalised over the eight chosen
        dict(name="route_softmax_row", kind="route", t=1, experts=128, top_k=8, score="softmax", bias=False, groups=1,
             top_groups=1, renormalize=True, scale=1.0, dtype="bf16", masked=False),
        # the 576-token prompt: sigmoid scores, a bias for balance, four of eight groups
        dict(name="route_sigmoid_groups_576", kind="route", t=576, experts=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, renormalize=True, scale=2.5, dtype="f32", masked=False),
        # a long ragged batch with padding rows and switched-off experts (logits of -inf)
        dict(name="route_softmax_16387", kind="route", t=16387, experts=160, top_k=6, score="softmax", bias=False,
             groups=5, top_groups=2, renormalize=False, scale=1.0, dtype="bf16", masked=True),
        # one decode token on eight of 128 experts: weight-bound, the latency case
        dict(name="experts_row", kind="experts", t=1, experts=128, top_k=8, h=2048, i=768, padded=False),
        # a decode batch of 48 tokens: nearly every expert is read, for a few rows each
        dict(name="experts_batch_48", kind="experts", t=48, experts=64, top_k=4, h=2560, i=1024, padded=False),
        # a ragged prompt with padding rows (no expert), widths that end inside a block
        dict(name="experts_ragged_577", kind="experts", t=577, experts=60, top_k=5, h=2120, i=1000, padded=True),
        # a long prompt on 128 experts: 256 rows per expert
        dict(name="experts_4096", kind="experts", t=4096, experts=128, top_k=8, h=2048, i=768, padded=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "route", "experts", "experts"])
    if kind == "linear":
        return dict(kind=kind, m=_log_int(rng, 1, 4096), n=_log_int(rng, 64, 16384), k=_log_int(rng, 64, 8192))
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log_int(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        score = rng.choice(["softmax", "sigmoid"])
        return dict(kind=kind, t=_log_int(rng, 1, 16384), experts=groups * per,
                    top_k=rng.randint(1, min(8, top_groups * per)), score=score, bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, renormalize=rng.random() < 0.5,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "f32"]), masked=rng.random() < 0.3)
    experts = _log_int(rng, 4, 128)
    return dict(kind=kind, t=_log_int(rng, 1, 4096), experts=experts, top_k=rng.randint(1, min(8, experts)),
                h=8 * _log_int(rng, 16, 320), i=8 * _log_int(rng, 8, 96), padded=rng.random() < 0.3)


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-n // BLOCK) * -(-k // BLOCK)
        return dict(bytes=2 * m * k + n * k + 4 * blocks + 2 * m * n, flops=2 * m * n * k)
    if case["kind"] == "route":
        t, e = case["t"], case["experts"]
        return dict(bytes=t * e * (2 if case["dtype"] == "bf16" else 4) + 8 * t * case["top_k"] + 4 * e * case["bias"],
                    flops=4 * t * e)
    t, e, top_k, h, i = (case[x] for x in ("t", "experts", "top_k", "h", "i"))
    real = t - _padding(case)
    read = e * (1 - (1 - top_k / e) ** real)                # experts that some token chose, on average
    return dict(bytes=int(read * 3 * h * i) + 4 * t * h + 8 * t * top_k, flops=6 * real * top_k * h * i)


# ---------------------------------------------------------------- inputs

def _gen(seed, part=0):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 1009 + part)
    return g


def _activations(g, m, k):
    # normalised activations with some channels much larger than the rest, as after an RMSNorm
    gain = 1 + 4 * (torch.rand(k, generator=g, device=DEVICE) < 0.01)
    return (torch.randn((m, k), generator=g, device=DEVICE) * gain).to(BF16)


def _weight(g, *shape):
    """e4m3 codes and block scales of random-init weights (the layout of block-scaled
    checkpoints: value = code * scale of its 128 x 128 block), rows and columns in
    the last two dimensions."""
    w = torch.randn(shape, generator=g, device=DEVICE) * 0.02
    n, k = shape[-2:]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pad = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    scale = pad.unflatten(-1, (kb, BLOCK)).unflatten(-3, (nb, BLOCK)).abs().amax((-3, -1)).clamp(min=1e-12) / 448
    return (w / _expand(scale, n, k)).clamp(-448, 448).to(E4M3), scale


def _expand(scale, n, k):
    """Block scales as one value per weight."""
    return scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _padding(case):
    """Padding rows at the end of the batch."""
    return case["t"] // 20 + 1 if case.get("padded") and case["t"] > 1 else 0


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "linear":
        codes, scale = _weight(g, case["n"], case["k"])
        return dict(codes=codes, scale=scale, x=_activations(g, case["m"], case["k"]))
    if case["kind"] == "route":
        t, e = case["t"], case["experts"]
        logits = 1.5 * torch.randn((t, e), generator=g, device=DEVICE)
        bias = 0.05 * torch.randn(e, generator=g, device=DEVICE) if case["bias"] else None
        if case["masked"]:
            logits[:, torch.rand(e, generator=g, device=DEVICE) < 0.1] = -math.inf
            logits[t - t // 20:] = -math.inf                          # padding rows choose no expert
        return dict(logits=logits.to(BF16) if case["dtype"] == "bf16" else logits, bias=bias)
    t, e, top_k, h, i = (case[x] for x in ("t", "experts", "top_k", "h", "i"))
    gate_up = torch.empty((e, 2, i, h), device=DEVICE, dtype=E4M3)
    down = torch.empty((e, h, i), device=DEVICE, dtype=E4M3)
    gate_up_scale, down_scale = [], []
    for j in range(e):
        gate_up[j], s = _weight(g, 2, i, h)
        gate_up_scale.append(s)
        down[j], s = _weight(g, h, i)
        down_scale.append(s)
    # experts of uneven popularity, weights renormalised over the chosen ones
    logits = torch.randn((t, e), generator=g, device=DEVICE) + 0.5 * torch.randn(e, generator=g, device=DEVICE)
    top, ids = logits.topk(top_k)
    weights, ids = top.softmax(-1), ids.to(torch.int32)
    real = t - _padding(case)
    ids[real:], weights[real:] = -1, 0
    return dict(gate_up=gate_up, gate_up_scale=torch.stack(gate_up_scale), down=down,
                down_scale=torch.stack(down_scale), x=_activations(g, t, h), weights=weights, ids=ids)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["kind"] == "linear":
        from fastforward_amd.linear import BlockFP8Linear
        state["op"] = BlockFP8Linear.from_codes(state["codes"], state["scale"])
    if own and case["kind"] == "experts":
        from fastforward_amd.moe import Experts
        state["op"] = Experts.from_codes(state["gate_up"], state["gate_up_scale"], state["down"], state["down_scale"])
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if case["kind"] == "linear":
        return state["op"](state["x"]) if own else _plain_linear(state["x"], state["codes"], state["scale"]).to(BF16)
    if case["kind"] == "route":
        if own:
            from fastforward_amd import moe
            weights, ids = moe.route(state["logits"], case["top_k"], score=case["score"], bias=state["bias"],
                                     groups=case["groups"], top_groups=case["top_groups"],
                                     renormalize=case["renormalize"], scale=case["scale"])
        else:
            weights, ids = _plain_route(state["logits"], state["bias"], case)
        return dict(weights=weights, ids=ids)
    if own:
        return state["op"](state["x"], state["weights"], state["ids"])
    return _plain_experts(state)


def _plain_quantise(x):
    """The values that x (32 bits) keeps in e4m3 with a scale for each row and 128 channels."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    groups = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).reshape(m, kb, BLOCK)
    amax = groups.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    scale = amax / torch.full_like(amax, 448)          # a quotient: by a Python number torch multiplies by 1 / 448
    return ((groups / scale).clamp(-448, 448).to(E4M3).float() * scale).reshape(m, kb * BLOCK)[:, :k]


def _plain_linear(x, codes, scale):
    w = codes.float() * _expand(scale, *codes.shape)
    return _plain_quantise(x.float()) @ w.T


def _plain_route(logits, bias, case):
    # scores in 64 bits: experts whose scores lie next to each other change places in 32
    t, e = logits.shape
    k, groups = case["top_k"], case["groups"]
    l = logits.double()
    off = l == -math.inf
    if case["score"] == "softmax":
        top = l.amax(-1, keepdim=True)
        p = (l - top.clamp(min=-1e300)).exp()
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        p = 1 / (1 + (-l).exp())
    c = (p if bias is None else p + bias.double()).masked_fill(off, -math.inf)
    if groups > 1:
        per = c.reshape(t, groups, e // groups).sort(dim=-1, descending=True, stable=True).values
        best = per[..., 0]
        if bias is not None and e > groups:
            best = best + torch.where(per[..., 1] == -math.inf, torch.zeros_like(best), per[..., 1])
        chosen = best.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros((t, groups), device=l.device, dtype=torch.bool).scatter_(1, chosen, True)
        c = c.masked_fill(~keep.repeat_interleave(e // groups, -1), -math.inf)
    c, ids = c.sort(dim=-1, descending=True, stable=True)
    c, ids = c[:, :k], ids[:, :k]
    none = c == -math.inf                                      # fewer than k experts left
    weights = p.gather(-1, ids).masked_fill(none, 0)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-300)
    return (weights * case["scale"]).float(), ids.masked_fill(none, -1).to(torch.int32)


def _plain_experts(state):
    x, weights, ids = state["x"], state["weights"], state["ids"]
    t, h = x.shape
    top_k = ids.shape[1]
    flat = ids.reshape(-1).long()
    order = flat.sort(stable=True).indices
    counts = (flat[:, None] == torch.arange(-1, state["gate_up"].shape[0], device=x.device)).sum(0).tolist()
    xq = _plain_quantise(x.float())
    y = torch.zeros((t * top_k, h), device=x.device, dtype=F32)
    start = counts[0]
    for j, n in enumerate(counts[1:]):
        if not n:
            continue
        pairs = order[start:start + n]
        start += n
        rows = xq[pairs // top_k]
        wgu, sgu, i = state["gate_up"][j], state["gate_up_scale"][j], state["gate_up"].shape[2]
        gate = rows @ (wgu[0].float() * _expand(sgu[0], i, h)).T
        up = rows @ (wgu[1].float() * _expand(sgu[1], i, h)).T
        mid = gate / (1 + (-gate).exp()) * up
        y[pairs] = mid @ (state["down"][j].float() * _expand(state["down_scale"][j], h, i)).T
    return (y.reshape(t, top_k, h) * weights[..., None]).sum(1).to(BF16)


# ---------------------------------------------------------------- the definition in 64 bits

def _e4m3(v):
    """Nearest e4m3 value (3 mantissa bits, steps of 2^-9 below 2^-6, largest 448), ties to even."""
    exponent = torch.frexp(v.abs()).exponent.double() - 1
    step = torch.exp2(exponent.clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_quantise(x):
    """Quantisation of x: scale = amax / 448 and code = e4m3(x / scale), scale and quotient
    32-bit numbers by definition (the quotient of two bf16 numbers often lies next to a
    border between two codes, and on it in 32 bits)."""
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], BLOCK):
        part = x[:, a:a + BLOCK]
        amax = part.abs().amax(1, keepdim=True).clamp(min=1e-12)
        s = (amax / torch.full_like(amax, 448)).to(F32).double()
        out[:, a:a + BLOCK] = _e4m3((part / s).to(F32).double()) * s
    return out


def _exact_weight(codes, scale):
    w = codes.double()
    for a in range(0, w.shape[0], BLOCK):
        for b in range(0, w.shape[1], BLOCK):
            w[a:a + BLOCK, b:b + BLOCK] *= scale[a // BLOCK, b // BLOCK].double()
    return w


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "linear":
        x = _exact_quantise(s["x"].double())
        step = max(BLOCK, (1 << 27) // case["k"] // BLOCK * BLOCK)
        return torch.cat([x @ _exact_weight(s["codes"][a:a + step], s["scale"][a // BLOCK:(a + step) // BLOCK]).T
                          for a in range(0, case["n"], step)], 1)
    if case["kind"] == "route":
        return _exact_route(s["logits"].double().cpu(), None if s["bias"] is None else s["bias"].double().cpu(), case)
    x = _exact_quantise(s["x"].double())
    y = torch.zeros((case["t"], case["h"]), device=DEVICE, dtype=F64)
    for j in range(case["experts"]):
        token, slot = (s["ids"] == j).nonzero(as_tuple=True)
        if token.numel():
            gate, up = (x[token] @ _exact_weight(s["gate_up"][j, p], s["gate_up_scale"][j, p]).T for p in (0, 1))
            mid = gate * torch.sigmoid(gate) * up
            part = mid @ _exact_weight(s["down"][j], s["down_scale"][j]).T
            y[token] += s["weights"][token, slot].double()[:, None] * part
    return y


def _exact_route(l, bias, case):
    t, e = l.shape
    groups, k = case["groups"], case["top_k"]
    p = torch.softmax(l, -1).nan_to_num(0) if case["score"] == "softmax" else torch.sigmoid(l)
    choice = p.clone() if bias is None else p + bias
    choice[l == -math.inf] = -math.inf
    if groups > 1:
        per = e // groups
        best = torch.full((t, groups), -math.inf, dtype=F64)
        for j in range(groups):
            top = choice[:, j * per:(j + 1) * per].topk(2 if bias is not None and per > 1 else 1).values
            rest = top[:, 1:].clone()
            rest[rest == -math.inf] = 0
            best[:, j] = top[:, 0] + rest.sum(-1)
        for _ in range(groups - case["top_groups"]):                  # drop the worst, the last of equal ones
            worst = groups - 1 - best.flip(-1).argmin(-1)
            best[torch.arange(t), worst] = math.inf
            for j in range(groups):
                choice[worst == j, j * per:(j + 1) * per] = -math.inf
    ids = torch.full((t, k), -1, dtype=torch.int32)
    weights = torch.zeros((t, k), dtype=F64)
    rows = torch.arange(t)
    for j in range(k):
        best = choice.argmax(-1)
        left = choice[rows, best] > -math.inf
        first = (choice == choice[rows, best][:, None]).int().argmax(-1)
        ids[left, j] = first[left].int()
        weights[left, j] = p[rows, first][left]
        choice[rows, first] = -math.inf
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-300)
    return dict(weights=(weights * case["scale"]).to(DEVICE), ids=ids.to(DEVICE))
