"""The 64-bit oracle of the block-scaled FP8 and expert operators against library
routines and closed forms (CPU)."""
import math

import pytest
import torch

from oracle import moe as M
from tests.numerics import e4m3_decode_np, e4m3_encode_np

BF16 = torch.bfloat16


def _g(seed):
    return torch.Generator().manual_seed(seed)


def test_rows_codes_are_the_nearest():
    x = (torch.randn(5, 300, generator=_g(1)) * 3).to(BF16)
    q, s = M.quant_rows(x)
    pad = torch.nn.functional.pad(x.float(), (0, 84)).reshape(5, 3, 128)
    quotient = (pad / s.T[..., None]).clamp(-448, 448)
    assert (q.view(torch.uint8).numpy().reshape(-1) == e4m3_encode_np(quotient.numpy().reshape(-1))).all()
    assert torch.equal(s.T, pad.abs().amax(-1) / torch.full((5, 3), 448.0))
    back = M.rows_values(q, s, 300)
    want = e4m3_decode_np(q.view(torch.uint8).numpy()).reshape(5, 3, 128) * s.T.double().numpy()[..., None]
    assert (back.numpy() == want.reshape(5, 384)[:, :300]).all()
    # within half a step (2^-4 of the value, 2^-10 of the scale below the normal range)
    assert ((back - x.double()).abs() <= 2.0 ** -4 * x.double().abs() +
            2.0 ** -10 * s.T.double().repeat_interleave(128, 1)[:, :300]).all()


def test_weight_blocks():
    w = (torch.randn(200, 300, generator=_g(2)) * 0.02).to(BF16)
    q, s = M.quant_weight(w)
    assert s.shape == (2, 3)
    for a in range(2):
        for b in range(3):
            block = w[128 * a:128 * a + 128, 128 * b:128 * b + 128].float()
            assert s[a, b] == block.abs().max() / torch.tensor(448.0)
    assert (M.dequant(q, s) - w.double()).abs().max() <= 2.0 ** -4 * w.double().abs().max()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_is_topk_of_the_scores(score):
    l = torch.randn(40, 24, generator=_g(3))
    w, ids = M.route(l, 4, score=score, renormalize=False)
    p = torch.softmax(l.double(), -1) if score == "softmax" else torch.sigmoid(l.double())
    top = p.topk(4)
    assert torch.equal(ids.long(), top.indices) and torch.allclose(w, top.values, rtol=1e-14, atol=0)


def test_route_masks_ties_groups():
    inf = math.inf
    l = torch.tensor([[1.0, 1.0, 1.0, 0.0], [-inf, 2.0, -inf, -inf], [-inf] * 4, [math.nan, 0.0, 0.0, 0.0]])
    w, ids = M.route(l, 2)
    assert ids.tolist() == [[0, 1], [1, -1], [-1, -1], [0, 1]]
    assert w[0].tolist() == [0.5, 0.5] and w[1].tolist() == [1.0, 0.0] and w[2].tolist() == [0.0, 0.0]
    assert w[3].isnan().all()
    # group 1 holds the best expert, group 0 the two best together
    l = torch.tensor([[2.0, 1.9, -9.0, 2.1]])
    assert M.route(l, 1, groups=2, top_groups=1)[1].tolist() == [[3]]
    assert M.route(l, 1, bias=torch.zeros(4), groups=2, top_groups=1)[1].tolist() == [[0]]


def test_experts_is_a_swiglu_mlp():
    e, t, h, i = 3, 4, 40, 24
    codes = [torch.randn(s, generator=_g(4)).to(M.E4M3) for s in ((e, 2, i, h), (e, h, i))]
    scales = [torch.rand(s, generator=_g(5)) for s in ((e, 2, 1, 1), (e, 1, 1))]
    x = torch.randn(t, h, generator=_g(6)).to(BF16)
    ids = torch.tensor([[0, 2], [1, 1], [-1, 0], [-1, 7]], dtype=torch.int32)
    w = torch.rand(t, 2, generator=_g(7))
    y, bound = M.experts(x, w, ids, codes[0], scales[0], codes[1], scales[1])
    a = M.rows_values(*M.quant_rows(x), h)
    for r in range(t):
        want = torch.zeros(h, dtype=torch.float64)
        for j in range(2):
            k = int(ids[r, j])
            if 0 <= k < e:
                g, u = (codes[0][k, p].double() * float(scales[0][k, p, 0, 0]) @ a[r] for p in (0, 1))
                want += float(w[r, j]) * (codes[1][k].double() * float(scales[1][k, 0, 0])
                                          @ (torch.nn.functional.silu(g) * u))
        assert torch.allclose(y[r], want, rtol=1e-12, atol=1e-12)
    assert (y[3] == 0).all() and (bound[3] == 0).all()
