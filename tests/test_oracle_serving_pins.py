"""The 64-bit oracle of the paged cache, its attention and token scores against library
routines and closed forms (CPU)."""
import math

import pytest
import torch

from oracle import serving as S
from tests.numerics import e4m3_decode_np, e4m3_encode_np

BF16, E4M3, I32, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.int32, torch.float64


def _g(seed):
    return torch.Generator().manual_seed(seed)


def test_codes_are_the_nearest_under_the_smallest_power():
    x = torch.randn(300, 64, generator=_g(1)) * torch.exp2(torch.randint(-60, 60, (300, 1), generator=_g(2)).float())
    x[0], x[1, 3], x[2, 5] = 0, math.inf, math.nan
    x = x.to(BF16)
    e = S.exponent(x)
    amax = x.double().abs().nan_to_num(0, posinf=0).amax(1)
    assert e[0] == -100 and (amax <= 448 * torch.exp2(e.double())).all()
    assert (amax[1:] > 448 * torch.exp2(e[1:].double() - 1)).all()         # one less would not do
    codes, byte = S.codes(x)
    assert torch.equal(byte.long(), e + 127)
    y = (x.double() * torch.exp2(-e.double())[:, None]).float()
    odd = ~(x.float().abs() < math.inf)
    want = torch.from_numpy(e4m3_encode_np(y.masked_fill(odd, 0).numpy().reshape(-1)).reshape(300, 64))
    assert torch.equal(codes.view(torch.uint8)[~odd], want[~odd]) and codes.float()[odd].isnan().all()
    back = S.values({"k": codes, "k_scale": byte}, "k")
    lib = torch.from_numpy(e4m3_decode_np(codes.view(torch.uint8).numpy()).astype("float64")) * torch.exp2(e.double())[:, None]
    assert torch.equal(back[~odd], lib[~odd])
    assert torch.equal(back[~odd].to(BF16).double(), back[~odd])           # exact in bf16
    # half a step: 2^-4 of the value, 2^-10 of the scale below the normal range
    off = (back - x.double()).abs() - 2.0 ** -4 * x.double().abs() - 2.0 ** -10 * torch.exp2(e.double())[:, None]
    assert (off[~odd] <= 0).all()


def _filled(dtype, lengths, ps, hk, d):
    need = [-(-n // ps) for n in lengths]
    order = torch.randperm(sum(need), generator=_g(3)).to(I32)
    table = torch.full((len(lengths), max(need)), -1, dtype=I32)
    for i, n in enumerate(need):
        table[i, :n] = order[sum(need[:i]):sum(need[:i]) + n]
    c = {name: torch.zeros(sum(need), hk, ps, d, dtype=dtype) for name in ("k", "v")}
    if dtype == E4M3:
        c.update({name + "_scale": torch.zeros(sum(need), hk, ps, dtype=torch.uint8) for name in ("k", "v")})
    return c, table


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_cache_and_attention(dtype):
    """Whole sequences written and read back; the attention of their last rows is the library's on those."""
    lengths, new, hk, group, d = [20, 7, 33], [5, 7, 1], 2, 3, 64
    c, table = _filled(dtype, lengths, 16, hk, d)
    k, v = (torch.randn(60, hk, d, generator=_g(i)).to(BF16) for i in (4, 5))
    starts = torch.tensor([0, 20, 27, 60])
    S.write(c, k, v, table, torch.tensor(lengths), starts)
    kk, vv = S.read(c, table, torch.tensor(lengths), starts, 60)
    for x, y in ((k, kk), (v, vv)):
        if dtype == BF16:
            assert torch.equal(x.double(), y)
        else:
            codes, byte = S.codes(x)
            assert torch.equal(S.values({"k": codes, "k_scale": byte}, "k"), y)
    q = torch.randn(13, hk * group, d, generator=_g(6)).to(BF16)
    at = torch.tensor([0, 5, 12, 13])
    o, a, most = S.attend(c, q, table, torch.tensor(lengths), at)
    for b, (n, m) in enumerate(zip(lengths, new)):
        rows = slice(int(starts[b]), int(starts[b + 1]))
        mask = torch.arange(n) <= torch.arange(n - m, n)[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(
            q[at[b]:at[b + 1]].double().transpose(0, 1), kk[rows].transpose(0, 1).repeat_interleave(group, 0),
            vv[rows].transpose(0, 1).repeat_interleave(group, 0), attn_mask=mask).transpose(0, 1)
        # two evaluations in 64 bits, up to 33 terms and exponents of up to `most`
        assert ((o[at[b]:at[b + 1]] - want).abs() <= (4 * most + 100) * 2.0 ** -52 * a[at[b]:at[b + 1]]).all()
    assert (a >= o.abs() * (1 - 2.0 ** -40)).all()


def test_rows_without_a_place():
    c, table = _filled(BF16, [16, 16], 16, 1, 64)
    table[1, 0] = 9                                   # no such page
    k = torch.ones(4, 1, 64, dtype=BF16)
    S.write(c, k, k, table, torch.tensor([18, 2]), torch.tensor([0, 2, 4]))
    assert not c["k"].any()                           # positions 16, 17 are past the table, page 9 is none
    o, _, _ = S.attend(c, k, table, torch.tensor([18, 2]), torch.tensor([0, 2, 3]))
    assert torch.equal(o, torch.zeros(4, 1, 64, dtype=F64))


def test_token_scores():
    x = torch.randn(6, 200, generator=_g(7)) * 3
    x[1, 5] = 60.0
    x[2, ::2] = -math.inf
    x[3] = torch.randint(0, 5, (200,), generator=_g(8)).float()
    x[4] = -math.inf
    x[5, 3] = math.nan
    tokens = torch.tensor([[0, 5, -1], [5, 0, 200], [1, 0, 3], [0, 1, 2], [0, 1, -1], [0, 3, -1]])
    lp, h, top, ids = S.token_scores(x, tokens, 7)
    want = torch.log_softmax(x.double(), 1)
    for r in range(4):
        for i, t in enumerate(tokens[r].tolist()):
            assert lp[r, i] == 0 if not 0 <= t < 200 else torch.isclose(lp[r, i], want[r, t], rtol=1e-13, atol=1e-13)
        p = want[r].exp()
        assert torch.isclose(h[r], -(p * want[r].nan_to_num(0, neginf=0)).sum(), rtol=1e-12, atol=1e-14)
        order = sorted(range(200), key=lambda i: (-float(x[r, i]), i))[:7]
        assert ids[r].tolist() == order and torch.allclose(top[r], want[r, order], rtol=1e-13, atol=1e-13)
    assert torch.isclose(lp[1, 0], -(x[1].double() - 60).exp()[torch.arange(200) != 5].sum().log1p(), rtol=1e-12, atol=0)
    assert lp[4].tolist() == [-math.inf, -math.inf, 0] and h[4] == 0 and ids[4].tolist() == list(range(7))
    assert lp[5, :2].isnan().all() and h[5].isnan() and ids[5, 0] == 3
