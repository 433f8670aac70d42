"""Token scores on the GPU against the 64-bit oracle: one row to many, split rows, ties,
switched-off tokens, rows of nothing, NaN and infinities, near-certain tokens, strides,
streams, graphs; refusals on the CPU."""
import ctypes
import math

import pytest
import torch

from oracle import serving as S

BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
gpu_test = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _check(logits, tokens, top, times=1):
    """With ``times``, the rows that many times over in the call."""
    from fastforward_amd.scores import token_scores
    got = token_scores(logits.to(DEV).repeat(times, 1), tokens.to(DEV).repeat(times, *[1] * (tokens.dim() - 1)), top=top)
    if times > 1:
        for x in got[:4 if top else 2]:
            assert torch.equal(x.view(torch.int32).reshape(times, -1), x.view(torch.int32).reshape(times, -1)[:1].expand(times, -1))
    got = type(got)(*(x if x is None else x[:logits.shape[0]] for x in got))
    logprobs, entropy, top_logprobs, top_ids = S.token_scores(logits, tokens, top)
    assert got.logprobs.shape == tokens.shape and got.entropy.shape == (logits.shape[0],)
    # log p = (x - m) - log1p(r): the difference's rounding 2^-24 of it; r is a sum of at most v / 512
    # terms a lane, then of few, each off by at most 2^-23 |d| + 2^-22 of itself with |d| <= 30 where it
    # counts, 2^-17 in all, and so is log1p(r) at most; two roundings at the end
    v = logits.shape[1]
    rel = 2.0 ** -17 + (v / 512 + 20) * 2.0 ** -24
    x = logits.double()
    x[(x.isnan() | (x == math.inf)).any(1) | (x == -math.inf).all(1)] = 0     # rows of exact scores
    lse = S.log_softmax(x)[1]

    def near(a, want, tol):
        a = a.cpu().double()
        # the difference of the type's lowest and largest values, 6.8e38, is past fp32's 3.4e38: -inf there
        want = torch.where(want.abs() > 2.0 ** 128, want.sign() * math.inf, want)
        assert torch.equal(a.isnan(), want.isnan()) and torch.equal(a.isinf(), want.isinf())
        off = torch.where(want.abs() < math.inf, (a - want).abs() - tol, torch.zeros_like(want))
        assert float(off.max() if off.numel() else 0) <= 1e-37, float(off.max())
    near(got.logprobs, logprobs, 2.0 ** -22 * logprobs.abs() + (rel * lse).reshape(-1, *[1] * (tokens.dim() - 1)))
    # entropy = log1p(r) - t / (1 + r): both of one sign, t's terms off as r's
    near(got.entropy, entropy, 2 * rel * entropy.abs() + 2 * rel * lse)
    if top:
        assert torch.equal(got.top_ids.cpu(), top_ids)
        near(got.top_logprobs, top_logprobs, 2.0 ** -22 * top_logprobs.abs() + (rel * lse)[:, None])
    else:
        assert got.top_ids is None and got.top_logprobs is None


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,v,n,top", [(1, 1, 1, 1), (1, 7, 3, 7), (3, 100, 2, 64), (2, 511, 1, 0), (5, 4099, 4, 20),
                                       (1, 20011, 1, 5), (300, 65, 2, 3), (257, 200, 1, 33), (2, 40000, 8, 1), (2049, 70, 1, 9)])
def test_scores(gpu, dtype, t, v, n, top):
    l = (torch.randn(t, v, generator=_g(v)) * 3).to(dtype)           # bf16 logits tie often
    tokens = torch.randint(0, v, (t, n), generator=_g(n))
    tokens[0, 0] = l[0].argmax()
    _check(l, tokens, top)
    off = l.clone()
    off[:, torch.rand(v, generator=_g(1)) < 0.3] = -math.inf
    _check(off, tokens, min(top, v))
    _check(l, tokens[:, 0], top)


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("v", [60, 9001])
def test_scores_special_rows(gpu, dtype, v):
    """Rows of nothing, one token left, all equal, NaN, infinities, near-certain tokens, falling and rising
    rows (every logit enters the list of the likeliest), the type's lowest value, tokens that are none."""
    inf, low = math.inf, torch.finfo(dtype).min
    l = torch.randn(19, v, generator=_g(4)) * 2
    l[0] = -inf
    l[1], l[1, 37] = -inf, 3.0
    l[2] = 0
    l[3] = low
    l[4, 7] = math.nan
    l[5, 9] = inf
    l[6] = torch.linspace(-1000, 1000, v)
    l[7] = torch.linspace(100, -100, v)
    l[8], l[8, v - 1] = l[8] * 0.1, 30.0             # a near-certain token: log p of 1e-10
    l[9], l[9, 0] = -30.0, 0.0
    l[10] = torch.finfo(dtype).max
    l[11, ::2] = -inf
    l[12] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    l[13, 3], l[13, 5], l[13, 6], l[13, 8] = math.nan, -math.nan, inf, -inf
    l[14] = -inf
    l[14, 1::7] = low
    l[16, :v // 2] = low                             # whole waves of the lowest value, then others; the reverse
    l[17, v // 2:] = low
    l[18, :v // 2], l[18, v // 2:] = low, -low
    l = l.to(dtype)
    tokens = torch.tensor([0, 1, 37, v - 1, v, -1, -100, 7, 1 << 40]).repeat(19, 1)
    if v == 60:                                      # a row a wave
        l, tokens = l.repeat(108, 1), tokens.repeat(108, 1)
    for top in (0, 1, 20, min(v, 64)):
        _check(l, tokens, top)


@gpu_test
@pytest.mark.parametrize("top", [1, 8, 9, 20, 32, 33, 64])
def test_scores_lists_of_many_parts(gpu, top):
    """The likeliest tokens of rows in 64 parts: spread out, all in one part, in one wave of a part, one in
    each part, far apart, the same few values everywhere."""
    v = 140003
    l = torch.randn(8, v, generator=_g(9))
    l[1] = torch.linspace(4, -4, v)
    l[2] = torch.linspace(-4, 4, v)
    l[3, 70000:70300] += 9
    l[4, ::2189] += 9
    l[5] = -torch.arange(v) % 37 * 0.25
    for at in range(0, 80):
        l[6, 1024 * at] += 20 + 0.01 * at
    l[7, 100000:100064] += 9 + torch.randperm(64, generator=_g(1)) * 0.125
    for dtype in (F32, BF16):
        _check(l.to(dtype), torch.arange(8)[:, None], top)


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("v,times", [(26003, 13), (26000, 13), (4003, 103)])
def test_scores_long_rows(gpu, dtype, v, times):
    """Rows that one workgroup, or one wave, reads in many steps: the likeliest early, late, in one wave's share,
    equal ones and both zeros across waves, NaN and infinities late, rising and falling rows, nothing at first."""
    inf, low = math.inf, torch.finfo(dtype).min
    l = torch.randn(20, v, generator=_g(v)) * 2
    l[1] = torch.linspace(-30, 30, v)
    l[2] = torch.linspace(30, -30, v)
    l[3] = 0
    l[4] = torch.where(torch.arange(v) % 3 == 0, 0.0, -0.0)
    l[5] = -torch.arange(v) % 11 * 0.5
    l[6, v - 70:] += 20
    l[7, 512 * 3:512 * 3 + 64] += 12
    l[8, ::1024] = 9.0                                # a lane's vectors of a wave, all equal
    l[9, :v - 100] = -inf
    l[10, :v // 2] = low
    l[11, v - 2] = math.nan
    l[12, v - 300] = inf
    l[13] = -40.0
    l[13, v - 1] = 0.0
    l[14, v // 2:] = -inf
    l[15] = -inf
    l[16] = torch.where(torch.arange(v) % 2 == 0, -0.0, -1e-3)
    l[16, v // 3] = 0.0
    l[17, torch.arange(0, v, 97)] = 3.0 + torch.arange(0, v, 97) / v
    l[18] = l[18] * 1e37
    l[19] = torch.finfo(dtype).max
    l[19, ::5] = low
    l = l.to(dtype)
    tokens = torch.stack([torch.zeros(20, dtype=torch.int64), l.float().nan_to_num(0).argmax(1), torch.full((20,), v - 1)], 1)
    for top in (0, 1, 5, 20, 64):
        _check(l, tokens, top, times)


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_of_any_size(gpu, dtype):
    """Logits of every magnitude and offset, the largest of a wave's first ones and later ones of another size."""
    sizes = torch.tensor([10.0 ** i for i in range(-3, 38)])
    l = torch.randn(41, 3001, generator=_g(8)) * sizes[:, None]
    l = torch.cat([l, l[:30] + sizes[:30, None] * 4, l[:30] - sizes[:30, None] * 9, l.clone(), -l.abs()])
    l[101:142, 2500:] = torch.randn(41, 501, generator=_g(7)) * sizes.flip(0)[:, None]
    l = l.to(dtype)
    for times in (1, 15):                             # split rows, and a row a wave
        _check(l, torch.tensor([0, 1, 2600]).repeat(183, 1), 8, times)


@gpu_test
def test_scores_near_certain(gpu):
    """log p of a token that is all but certain, to 32-bit precision: -log1p of a small sum."""
    from fastforward_amd.scores import token_scores
    for gap in (5.0, 20.0, 40.0, 80.0):
        l = torch.full((2, 30000), -gap)
        l[0, 29999] = l[1, 17] = 0.0
        got = token_scores(l.to(DEV), torch.tensor([29999, 17], device=DEV), top=2)
        r = 29999 * math.exp(-gap)
        # r: 30000 equal terms in few fp32 sums, each term off by 2^-23 * gap log2 e + 2^-22
        rel = (59 + 20) * 2.0 ** -24 + gap * 1.45 * 2.0 ** -23 + 2.0 ** -21
        for x in got.logprobs.tolist():
            assert abs(x + math.log1p(r)) <= rel * math.log1p(r), (gap, x)
        h = math.log1p(r) + r * gap / (1 + r)
        for x in got.entropy.tolist():
            assert abs(x - h) <= 2 * rel * h
        assert got.top_ids.tolist() == [[29999, 0], [17, 0]]


@gpu_test
def test_scores_strides_streams_graph(gpu):
    from fastforward_amd.scores import token_scores
    base = torch.randn(40, 3001, generator=_g(2)).to(DEV)
    tok = torch.randint(0, 1500, (40, 6), generator=_g(3)).to(DEV)

    def same(a, b):
        assert all(x is y or torch.equal(x, y) for x, y in zip(a, b))
    for l in (base[:, :1500], base[:, 1:1502], base[::2, 5:1600], base[:, ::2], base[:1].expand(8, 3001),
              base.to(BF16)[:, 1:1502]):
        for t in (tok[:l.shape[0]], tok[:l.shape[0], ::2], tok.T.contiguous().T[:l.shape[0]], tok[:l.shape[0], 1]):
            same(token_scores(l, t, top=5), token_scores(l.contiguous(), t.contiguous(), top=5))
    l = base[:3].contiguous()
    want = token_scores(l, tok[:3], top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = token_scores(l, tok[:3], top=20)
    torch.cuda.current_stream().wait_stream(side)
    same(want, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_scores(l, tok[:3], top=20)
    for seed in range(4):
        l.copy_(torch.randn(3, 3001, generator=_g(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        same(got, token_scores(l, tok[:3], top=20))
    empty = token_scores(l[:0], tok[:0], top=3)
    assert empty.logprobs.shape == (0, 6) and empty.top_ids.shape == (0, 3)
    none = token_scores(l, tok[:3, :0], top=1)
    assert none.logprobs.shape == (3, 0) and torch.equal(none.entropy, token_scores(l, tok[:3]).entropy)


def test_refusals():
    from fastforward_amd.scores import token_scores
    l, tok = torch.zeros(2, 80), torch.zeros(2, 3, dtype=torch.int64)
    for args, kw in (((l[0], tok), {}), ((l.double(), tok), {}), ((l, tok.int()), {}), ((l, tok[:1]), {}),
                     ((l, tok[None]), {}), ((l, tok), dict(top=65)), ((l[:, :5], tok), dict(top=6)),
                     ((l, tok), dict(top=-1)), ((l[:, :0], tok), {}), ((l, tok), {})):
        with pytest.raises(AssertionError):           # the last: not on the GPU
            token_scores(*args, **kw)


def test_refusals_c():
    from fastforward_amd import _lib
    _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def scores(x=p, tok=p, tops=p, t=2, v=80, n=1, top=2, ws=p, nbytes=4096):
        _lib.call("ff_token_scores", x, 1, v, tok, 1, 1, p, p, tops, tops, t, v, n, top, ws, nbytes, None)

    for kw, message in ((dict(t=-1), "bad sizes"), (dict(v=0), "bad sizes"), (dict(top=65), "bad sizes"),
                        (dict(top=81, v=80), "bad sizes"), (dict(n=-1), "bad sizes"), (dict(x=None), "null"),
                        (dict(tok=None), "null"), (dict(tops=None), "null"), (dict(v=100000, nbytes=64), "workspace"),
                        (dict(v=100000, ws=None), "workspace")):
        with pytest.raises(RuntimeError, match=message):
            scores(**kw)
    scores(x=None, t=0)
    need = ctypes.c_int64(-1)
    _lib.call("ff_token_scores_workspace", 300, 100000, 20, ctypes.byref(need))
    assert need.value == 0                            # many rows are not split
