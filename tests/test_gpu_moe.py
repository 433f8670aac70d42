"""Expert routing and the experts' products on the GPU against the 64-bit oracle:
choices exact, weights to the fp32 rounding, products within the oracle's bound; one
token to many, ragged sizes, masked rows, repeated experts, ids that are none,
strides, streams, graphs; a router, the routing and the experts run together; refusals
on the CPU."""
import ctypes
import math

import pytest
import torch

from oracle import moe as M

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"
gpu_test = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------- routing

def _check_route(logits, top_k, **kw):
    from fastforward_amd import moe
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}
    w, ids = moe.route(logits.to(DEV), top_k, **dev)
    want_w, want_ids = M.route(logits, top_k, **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_ids), (tuple(logits.shape), top_k, kw)
    w = w.cpu().double()
    assert torch.equal(w.isnan(), want_w.isnan())
    # one rounding to fp32 (2^-24 of the value), 64-bit work before it
    assert ((w - want_w).abs().nan_to_num(0) <= (2.0 ** -24 + 1e-12) * want_w.abs().nan_to_num(0) + 1e-45).all()


@gpu_test
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 128, 8), (3, 5, 5), (7, 60, 6), (33, 64, 1), (65, 65, 4),
                                   (130, 160, 6), (64, 256, 8), (9, 512, 16), (5, 1000, 64), (2, 1024, 10),
                                   (1025, 60, 4), (1030, 128, 8), (1024, 150, 6), (1027, 256, 16), (1026, 9, 3)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(gpu, t, e, k, score):
    for dtype in (BF16, torch.float32):
        l = (torch.randn(t, e, generator=_g(t + e)) * 2).to(dtype)     # bf16 logits tie often
        _check_route(l, k, score=score)
        _check_route(l, k, score=score, renormalize=False, scale=2.5)
        _check_route(l, k, score=score, bias=torch.randn(e, generator=_g(e)) * 0.1)


@gpu_test
@pytest.mark.parametrize("t,e,k,groups,top", [(40, 256, 8, 8, 4), (9, 160, 6, 5, 1), (33, 64, 8, 64, 8), (5, 12, 4, 2, 2),
                                              (21, 96, 3, 3, 2), (4, 1024, 32, 32, 3),
                                                  (1029, 160, 6, 5, 2), (1024, 256, 8, 16, 3)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(gpu, t, e, k, groups, top, score):
    l = torch.randn(t, e, generator=_g(e + groups))
    for logits in (l, l.to(BF16), (l * 2).round() / 2):                  # the last: whole groups tie
        for bias in (None, torch.randn(e, generator=_g(2)) * 0.05):
            _check_route(logits, k, score=score, groups=groups, top_groups=top, bias=bias, scale=1.5)


@gpu_test
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_special_rows(gpu, score):
    """Switched-off experts, rows without any, ties everywhere, extreme and NaN logits."""
    inf, low = math.inf, torch.finfo(torch.float32).min
    l = torch.randn(14, 40, generator=_g(4))
    l[0] = -inf
    l[1, :38] = -inf                       # fewer left than top_k
    l[2] = 0                               # all equal
    l[3] = low                             # the type's lowest value is a logit like any other
    l[4, 7] = math.nan
    l[5, 9] = inf
    l[6] = torch.linspace(-1000, 1000, 40)
    l[7], l[7, 3] = low, 1.0
    l[8, ::2] = -inf
    l[9, 5:] = -inf
    l[10, :20] = -inf                      # a group switched off
    l[11] = torch.finfo(torch.float32).max
    for kw in (dict(), dict(renormalize=False), dict(groups=4, top_groups=2),
               dict(bias=torch.randn(40, generator=_g(5)) * 0.1, groups=4, top_groups=3)):
        _check_route(l, 6, score=score, **kw)
        _check_route(l.repeat(74, 1), 6, score=score, **kw)     # many rows: 16 lanes each
    bias = torch.zeros(40)
    bias[3], bias[4], bias[5] = -inf, inf, 1e30
    _check_route(l, 6, score=score, bias=bias)
    bias[8] = math.nan
    _check_route(l, 6, score=score, bias=bias)


@gpu_test
def test_route_strides_graph_stream(gpu):
    from fastforward_amd import moe
    base = torch.randn(37, 100, generator=_g(6)).to(DEV)
    for l in (base[:, :48], base[::3, 5:53], base[:, ::2], base[:1, :48].expand(9, 48), base[:0, :48]):
        for a, b in zip(moe.route(l, 4), moe.route(l.contiguous(), 4)):
            assert torch.equal(a, b) and a.shape == (l.shape[0], 4)
    static = base[:, :64].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = moe.route(static, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, moe.route(static, 4)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe.route(static, 4)
    for seed in (1, 2, 3):
        static.copy_(torch.randn(37, 64, generator=_g(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, moe.route(static, 4)))


@gpu_test
@pytest.mark.parametrize("scale", [2.446, 2.827, 1 / 3])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_scale_between_fp32_numbers(gpu, scale, renormalize):
    """A scale that fp32 does not hold: the weights have one rounding all the same."""
    l = torch.randn(200, 64, generator=_g(8)) * 2
    for bias in (None, torch.randn(64, generator=_g(9)) * 0.1):
        _check_route(l, 8, score="sigmoid", scale=scale, renormalize=renormalize, bias=bias)


# ---------------------------------------------------------------- experts

def _weights(e, h, i, seed=0):
    gu = (torch.randn(e, 2, i, h, generator=_g(seed)) * 60).clamp(-448, 448).to(E4M3)
    dn = (torch.randn(e, h, i, generator=_g(seed + 1)) * 60).clamp(-448, 448).to(E4M3)
    bi, bh = -(-i // 128), -(-h // 128)
    gs = torch.rand(e, 2, bi, bh, generator=_g(seed + 2)) * 1e-3 + 1e-4
    ds = torch.rand(e, bh, bi, generator=_g(seed + 3)) * 1e-3 + 1e-4
    return gu, gs, dn, ds


def _experts(w):
    from fastforward_amd.moe import Experts
    return Experts.from_codes(*(v.to(DEV) for v in w))


def _tokens(t, k, e, h, seed=0):
    x = torch.randn(t, h, generator=_g(seed)).to(BF16)
    ids = torch.rand(t, max(e, k), generator=_g(seed + 1)).argsort(1)[:, :k].remainder(e).to(torch.int32)
    w = torch.rand(t, k, generator=_g(seed + 2)) + 0.05
    return x, (w / w.sum(1, keepdim=True)), ids


def _check(y, x, w, ids, codes):
    want, bound = M.experts(x, w, ids, *codes)
    excess = ((y.cpu().double() - want).abs() - bound).max()
    assert float(excess) <= 0, f"beyond the bound by {float(excess)}"
    n = want.norm()
    # bf16 roundings of the SwiGLU's values and of the result, 2^-8 / sqrt(3) each at most
    assert float((y.cpu().double() - want).norm()) <= 4e-3 * float(n) + 1e-30


# (tokens, top_k, experts, h, i): single tokens, both sides of the pair limit, one row
# to many per expert, sizes of one, ends inside a block
EXPERT_CASES = [(1, 1, 1, 1, 1), (1, 8, 16, 256, 128), (1, 3, 7, 130, 70), (2, 2, 3, 300, 257), (8, 8, 16, 128, 96),
                (13, 5, 9, 264, 136), (40, 2, 64, 72, 40), (66, 1, 4, 129, 128), (100, 3, 5, 256, 64), (90, 4, 2, 64, 300),
                (257, 2, 3, 136, 72)]


@gpu_test
@pytest.mark.parametrize("t,k,e,h,i", EXPERT_CASES)
def test_experts(gpu, t, k, e, h, i):
    codes = _weights(e, h, i)
    x, w, ids = _tokens(t, k, e, h)
    y = _experts(codes)(x.to(DEV), w.to(DEV), ids.to(DEV))
    assert y.shape == (t, h) and y.dtype == BF16
    _check(y, x, w, ids, codes)


@gpu_test
@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("t,k,e,h,i", EXPERT_CASES)
def test_every_path(gpu, t, k, e, h, i, tile):
    """Pair by pair, 32- and 64-row tiles, at sizes that another would be chosen for."""
    from fastforward_amd import moe
    from fastforward_amd._lib import call
    codes = _weights(e, h, i)
    x, w, ids = _tokens(t, k, e, h)
    op = _experts(codes)
    call("ff_set_tuning", 13, tile)
    moe.experts_workspace.cache_clear()
    try:
        y = op(x.to(DEV), w.to(DEV), ids.to(DEV))
    finally:
        call("ff_set_tuning", 13, 0)
        moe.experts_workspace.cache_clear()
    _check(y, x, w, ids, codes)


def _check_rounded_twice(y, x, w, ids, codes):
    """Within the oracle's bound and, by norm, two bf16 roundings of at most 2^-8 each."""
    want, bound = M.experts(x, w, ids, *codes)
    y = y.cpu().double()
    assert ((y - want).abs() <= bound).all()
    assert float((y - want).norm()) <= 2.0 ** -7 * float(want.norm())


@gpu_test
@pytest.mark.parametrize("tile", [2, 3])
@pytest.mark.parametrize("h,i", [(8264, 40), (40, 8264)])
def test_more_block_scales_than_lanes(gpu, h, i, tile):
    """Both row tiles past the first scales that a wave loads, of gate and up (h) and in the down
    products (i)."""
    from fastforward_amd import moe
    from fastforward_amd._lib import call
    from tests.test_gpu_block_fp8 import late_scales
    codes = list(_weights(2, h, i))
    codes[1], codes[3] = late_scales(codes[1].shape, 8), late_scales(codes[3].shape, 9)
    x, w, ids = _tokens(40, 1, 2, h)
    op = _experts(codes)
    call("ff_set_tuning", 13, tile)
    moe.experts_workspace.cache_clear()
    try:
        y = op(x.to(DEV), w.to(DEV), ids.to(DEV))
    finally:
        call("ff_set_tuning", 13, 0)
        moe.experts_workspace.cache_clear()
    _check_rounded_twice(y, x, w, ids, codes)


@gpu_test
@pytest.mark.parametrize("t", [1, 3])
def test_rows_longer_than_a_workgroup_keeps(gpu, t):
    """Few pairs of a row whose codes do not fit in the pair kernel's LDS take the row tiles."""
    codes = _weights(3, 49160, 16)
    x, w, ids = _tokens(t, 2, 3, 49160)
    _check_rounded_twice(_experts(codes)(x.to(DEV), w.to(DEV), ids.to(DEV)), x, w, ids, codes)


@gpu_test
@pytest.mark.parametrize("t,k,e,h,i", [(1, 8, 128, 2048, 768), (48, 4, 64, 2560, 1024), (300, 5, 12, 2120, 1000),
                                       (1024, 8, 16, 2048, 768)])
def test_experts_at_model_sizes(gpu, t, k, e, h, i):
    """Relative RMS against a plain fp32 evaluation on the GPU of the same definition."""
    codes = [v.to(DEV) for v in _weights(e, h, i)]
    x, w, ids = (v.to(DEV) for v in _tokens(t, k, e, h))
    y = _experts(codes)(x, w, ids).float()
    q, s = M.quant_rows(x)
    a = M.rows_values(q, s, h).float()
    want = torch.zeros(t, h, device=DEV)
    for j in range(e):
        tok, slot = (ids == j).nonzero(as_tuple=True)
        if tok.numel():
            g, u = (a[tok] @ M.dequant(codes[0][j, p], codes[1][j, p]).float().T for p in (0, 1))
            part = torch.nn.functional.silu(g) * u @ M.dequant(codes[2][j], codes[3][j]).float().T
            want.index_put_((tok,), w[tok, slot][:, None] * part, accumulate=True)
    assert float((y - want).norm() / want.norm()) <= 4e-3


@gpu_test
@pytest.mark.parametrize("t", [1, 6, 150])
def test_experts_ids(gpu, t):
    """Ids that are no expert add nothing, whatever their weight; rows without experts are
    zero; an expert may come twice; all tokens may share one."""
    e, k, h, i = 6, 3, 144, 80
    codes = _weights(e, h, i)
    op = _experts(codes)
    x, w, ids = _tokens(t, k, e, h)
    ids[0, 1] = ids[0, 0]
    ids[-1, 2] = -1
    ids[t // 2, 0] = e
    ids[t // 3, 1] = 2 ** 31 - 1
    w[-1, 2] = math.nan
    y = op(x.to(DEV), w.to(DEV), ids.to(DEV))
    _check(y, x, w.nan_to_num(0), ids, codes)
    none = torch.full_like(ids, -1)
    assert (op(x.to(DEV), w.to(DEV), none.to(DEV)) == 0).all()
    one = torch.full_like(ids, 4)
    _check(op(x.to(DEV), w.nan_to_num(0).to(DEV), one.to(DEV)), x, w.nan_to_num(0), one, codes)
    assert op(x[:0].to(DEV), w[:0].to(DEV), ids[:0].to(DEV)).shape == (0, h)


@gpu_test
@pytest.mark.parametrize("t", [2, 150])
def test_experts_rows_stand_alone(gpu, t):
    """A NaN or an infinity stays in its token; strided rows give the bits of a copy; two
    calls the same bits."""
    e, k, h, i = 5, 2, 200, 130
    codes = _weights(e, h, i)
    op = _experts(codes)
    x, w, ids = _tokens(t, k, e, h)
    w, ids = w.to(DEV), ids.to(DEV)
    y = op(x.to(DEV), w, ids)
    assert torch.equal(op(x.to(DEV), w, ids), y)
    for bad in (math.nan, math.inf):
        xb = x.clone()
        xb[1, 150] = bad
        yb = op(xb.to(DEV), w, ids)
        assert yb[1].isnan().all() and torch.equal(yb[:1], y[:1]) and torch.equal(yb[2:], y[2:])
    base = torch.zeros(t + 1, 2 * h + 5, dtype=BF16, device=DEV)
    for view in (base[:t, 1:h + 1], base[:t, 8:h + 8], base[:t, :2 * h:2]):
        view.copy_(x)
        assert torch.equal(op(view, w, ids), y)


@gpu_test
@pytest.mark.parametrize("t", [1, 9, 120])
def test_experts_graph_and_stream(gpu, t):
    e, k, h, i = 8, 4, 256, 128
    op = _experts(_weights(e, h, i))
    x, w, ids = (v.to(DEV) for v in _tokens(t, k, e, h))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = op(x, w, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, op(x, w, ids))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(x, w, ids)
    for seed in (20, 30, 40):
        for static, new in zip((x, w, ids), _tokens(t, k, e, h, seed)):
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, op(x, w, ids))


@gpu_test
def test_experts_offsets_past_32_bits(gpu):
    """Down products of more than 2^32 bytes: equal tokens give equal rows."""
    rows, times, k, e, h, i = 1050, 64, 8, 16, 2048, 128
    op = _experts(_weights(e, h, i))
    x, w, ids = (v.to(DEV) for v in _tokens(rows, k, e, h))
    y = op(x.repeat(times, 1), w.repeat(times, 1), ids.repeat(times, 1)).view(times, rows, h)
    assert torch.equal(y[0], op(x, w, ids)) and (y == y[:1]).all()      # 64-row tiles both times


@gpu_test
def test_experts_two_streams(gpu):
    """Calls that overlap on two streams share nothing."""
    k, e, h, i = 4, 8, 256, 128
    op = _experts(_weights(e, h, i))
    args = [[v.to(DEV) for v in _tokens(t, k, e, h, t)] for t in (20, 130)]
    want = [op(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(op(*args[j]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for ys, v in zip(got, want) for y in ys)


@gpu_test
def test_path_and_workspace_agree(gpu):
    """The path is chosen once a call, so a knob set from another thread meanwhile moves the
    next call: every result is one path's or the other's."""
    import threading
    from fastforward_amd._lib import call, entry, stream
    t, k, e, h, i = 4, 2, 6, 136, 200
    op = _experts(_weights(e, h, i))
    x, w, ids = (v.to(DEV) for v in _tokens(t, k, e, h))
    need = ctypes.c_int64(0)

    def run(y, ws):
        entry("ff_moe_experts")(x.data_ptr(), h, w.data_ptr(), ids.data_ptr(), op.gate_up._packed.data_ptr(),
                                op.gate_up_scale.data_ptr(), op.down._packed.data_ptr(), op.down_scale.data_ptr(),
                                y.data_ptr(), h, t, k, e, h, i, ws.data_ptr(), ws.numel(), stream())

    stop, want, sizes = threading.Event(), [], []

    def flip():
        while not stop.is_set():
            call("ff_set_tuning", 13, 1)
            call("ff_set_tuning", 13, 2)
    thread = threading.Thread(target=flip)
    try:
        for tile in (1, 2):
            call("ff_set_tuning", 13, tile)
            call("ff_moe_experts_workspace", t, k, e, h, i, ctypes.byref(need))
            sizes.append(need.value)
            ws, y = torch.empty(need.value, dtype=torch.uint8, device=DEV), torch.empty(t, h, dtype=BF16, device=DEV)
            run(y, ws)
            want.append(y)
        assert sizes[0] < sizes[1]
        ws, ys = torch.empty(sizes[1], dtype=torch.uint8, device=DEV), torch.empty(300, t, h, dtype=BF16, device=DEV)
        thread.start()
        for y in ys:
            run(y, ws)
    finally:
        stop.set()
        if thread.ident is not None:
            thread.join()
        call("ff_set_tuning", 13, 0)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[0]) or torch.equal(y, want[1]) for y in ys)


@gpu_test
def test_moe_strides(gpu):
    """The whole MLP, its router's product included, on rows of any stride and alignment."""
    from fastforward_amd.moe import MoE, Router
    h, i, e = 128, 72, 8
    op = MoE(Router((torch.randn(e, h, generator=_g(1)) * 0.1).to(BF16).to(DEV)), _experts(_weights(e, h, i)), 3)
    base = torch.randn(2 * h + 9, 2 * h + 3, generator=_g(2)).to(BF16).to(DEV)
    for x in (base[:9, 1:h + 1], base[:9, 8:h + 8], base[:9, :2 * h:2], base[:1, :h].expand(9, h), base[:h, :6].T,
              base[:h, :1].T, base[:h, :1].contiguous().T, base[None, :4, 3:h + 3], base[0, 5:h + 5], base[:0, :h]):
        flat = x.reshape(-1, h)
        copy = torch.empty(flat.shape, dtype=BF16, device=DEV).copy_(flat)
        assert torch.equal(op.router(flat), op.router(copy))
        assert torch.equal(op(x), op(copy).reshape(x.shape))


@gpu_test
def test_experts_from_bf16(gpu):
    from fastforward_amd.moe import Experts
    e, h, i = 3, 136, 200
    gu = (torch.randn(e, 2, i, h, generator=_g(1)) * 0.02).to(BF16)
    dn = (torch.randn(e, h, i, generator=_g(2)) * 0.02).to(BF16)
    op = Experts(gu.to(DEV), dn.to(DEV))
    for j in range(e):
        for w, codes, scale in ((gu[j, 0], op.gate_up.rowmajor()[j, 0], op.gate_up_scale[j, 0]),
                                (gu[j, 1], op.gate_up.rowmajor()[j, 1], op.gate_up_scale[j, 1]),
                                (dn[j], op.down.rowmajor()[j], op.down_scale[j])):
            want, want_s = M.quant_weight(w)
            assert torch.equal(scale.cpu(), want_s)
            assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))


# ---------------------------------------------------------------- refusals

def test_route_refusals():
    from fastforward_amd import moe
    l = torch.zeros(2, 8)
    for args, kw in (((l, 0), {}), ((l, 9), {}), ((l[0], 2), {}), ((l.double(), 2), {}), ((l, 2), dict(score="relu")),
                     ((l, 2), dict(groups=3)), ((l, 2), dict(groups=4, top_groups=5)),
                     ((l, 5), dict(groups=4, top_groups=2)), ((l, 2), {}), ((torch.zeros(2, 2000), 2), {})):
        with pytest.raises(AssertionError):           # the last but one: not on the GPU
            moe.route(*args, **kw)


def test_refusals_c():
    from fastforward_amd import _lib
    _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def route(logits=p, f32=1, t=2, e=8, k=2, groups=1, top=1):
        _lib.call("ff_moe_route", logits, f32, e, None, p, p, t, e, k, 0, groups, top, 1, 1.0, None)

    for kw in (dict(k=9), dict(k=0), dict(e=1025), dict(groups=3), dict(groups=4, top=0), dict(groups=8, top=1),
               dict(t=-1), dict(e=200, k=65)):
        with pytest.raises(RuntimeError, match="bad sizes"):
            route(**kw)
    with pytest.raises(RuntimeError, match="null"):
        route(logits=None)
    with pytest.raises(RuntimeError, match="alignment"):
        route(logits=p + 2)
    route(logits=None, t=0)

    def experts(x=p, gu=p, t=1, k=2, e=4, h=8, i=8, ldy=8, ws=p, nbytes=4096):
        _lib.call("ff_moe_experts", x, h, p, p, gu, p, p, p, p, ldy, t, k, e, h, i, ws, nbytes, None)

    for kw in (dict(k=0), dict(e=0), dict(e=1025), dict(h=0, ldy=8), dict(i=0), dict(t=-1), dict(t=1 << 24),
               dict(t=1 << 21, h=2048, ldy=2048), dict(h=1 << 16, i=1 << 15, ldy=1 << 16), dict(t=1 << 20, k=1000)):
        with pytest.raises(RuntimeError, match="bad sizes"):
            experts(**kw)
    for kw, message in ((dict(ldy=7), "strides"), (dict(x=None), "null"), (dict(x=p + 1), "alignment"),
                        (dict(gu=p + 4), "alignment"), (dict(nbytes=100), "workspace"), (dict(ws=None), "workspace"),
                        (dict(ws=p + 16), "workspace")):
        with pytest.raises(RuntimeError, match=message):
            experts(**kw)
    experts(x=None, t=0, ws=None, nbytes=0)
    need = ctypes.c_int64(-1)
    with pytest.raises(RuntimeError, match="bad sizes"):
        _lib.call("ff_moe_experts_workspace", 1, 1, 2000, 8, 8, ctypes.byref(need))
    _lib.call("ff_moe_experts_workspace", 1, 8, 128, 2048, 768, ctypes.byref(need))
    assert need.value == 8 * 768 * 2
