"""Mixture-of-experts MLP on gfx950 kernels: routing and the experts' products.

No reference counterpart (its models have one MLP per layer): the MLP of a decoder
layer whose gate/up and down projections are chosen per token. ``route`` picks each
token's experts from the router's logits, ``Experts`` holds block-scaled FP8 weights
(``linear.BlockFP8Linear``'s format) and computes the chosen experts' weighted sum,
``MoE`` is the whole MLP that the step runs where a layer has one.

Like the other ops: shape, dtype and device violations raise AssertionError before
any launch, outputs are fresh tensors, inputs are never written, launches go to the
current stream and can be captured (no host sync, no device-dependent grid).
"""
import ctypes
import functools

import torch

from ._lib import call, entry, ptr, stream
from .linear import BF16, _blocks, check_block_codes, check_here, pack_blocks

F32, I32 = torch.float32, torch.int32
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 64, 64


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """Experts of each token: (weights (T, top_k) fp32, ids (T, top_k) int32) from router
    logits (T, E), bf16 or fp32.

    p = softmax over the experts or, ``score="sigmoid"``, 1 / (1 + exp(-logit)). The
    ``top_k`` experts with the largest p + ``bias`` (E, fp32; for balance, not part of
    the weights) are chosen, in falling order, the lowest index first among equals.
    With ``groups`` > 1 (runs of E / groups experts) only experts of the ``top_groups``
    best groups are; a group's score is its best expert's, with a bias the sum of its
    two best. weights = p of the chosen, divided by their sum with ``renormalize``,
    times ``scale``.

    A logit of -inf switches its expert off; where fewer than ``top_k`` are left, the
    rest have id -1 and weight 0. A row with a NaN (or +inf under softmax) has NaN
    weights. Scores and weights are 64-bit until the weights' one rounding; without a bias
    experts are compared by their logits (scores rise with them), with one by score +
    bias in 64 bits."""
    assert logits.dim() == 2 and logits.dtype in (BF16, F32) and score in ("softmax", "sigmoid")
    t, e = logits.shape
    top_groups = groups if top_groups is None else top_groups
    assert 0 < e <= MAX_EXPERTS and 0 < top_k <= min(e, MAX_TOP_K), (e, top_k)
    assert 0 < groups <= MAX_GROUPS and e % groups == 0 and 0 < top_groups <= groups, (e, groups, top_groups)
    assert top_groups * (e // groups) >= top_k, "fewer experts in the kept groups than top_k"
    check_here(logits)
    if bias is not None:
        assert bias.shape == (e,) and bias.dtype == F32 and bias.is_contiguous()
        check_here(bias)
    if logits.stride(-1) != 1 and e > 1:
        logits = logits.contiguous()
    weights = logits.new_empty((t, top_k), dtype=F32)
    ids = logits.new_empty((t, top_k), dtype=I32)
    entry("ff_moe_route")(logits.data_ptr(), logits.dtype == F32, logits.stride(0), 0 if bias is None else bias.data_ptr(),
                          weights.data_ptr(), ids.data_ptr(), t, e, top_k, score == "sigmoid", groups, top_groups,
                          bool(renormalize), scale, stream())
    return weights, ids


@functools.lru_cache(maxsize=1024)
def experts_workspace(t, top_k, experts, h, i):
    """Bytes of workspace ff_moe_experts needs."""
    need = ctypes.c_int64(0)
    call("ff_moe_experts_workspace", t, top_k, experts, h, i, ctypes.byref(need))
    return need.value


class Experts:
    """The experts' MLPs in block-scaled FP8: y[t] = bf16(sum_j w[t, j] D_e (silu(G_e x)
    * (U_e x))), e = ids[t, j]. x is quantised per row and 128 channels, sums are fp32. The
    SwiGLU's values are rounded to bf16 (as large a rounding as the output's) and not
    quantised, unlike the rows of a dense layer's ``BlockFP8Linear``.

    ``Experts(gate_up, down)`` quantises bf16 weights, gate_up (E, 2, I, H) with the
    gate first and down (E, H, I); ``Experts.from_codes`` takes e4m3 codes of those
    shapes with their block scales (E, 2, ceil(I / 128), ceil(H / 128)) and (E,
    ceil(H / 128), ceil(I / 128))."""

    def __init__(self, gate_up, down):
        assert gate_up.dim() == 4 and down.dim() == 3 and gate_up.dtype == down.dtype == BF16
        check_here(gate_up, down)

        def quantise(w):
            flat = w.detach().reshape(-1, *w.shape[-2:])
            codes = torch.empty(flat.shape, device=w.device, dtype=torch.float8_e4m3fn)
            n, k = flat.shape[1:]
            scales = torch.empty((flat.shape[0], _blocks(n), _blocks(k)), device=w.device, dtype=F32)
            for j in range(flat.shape[0]):
                wj = flat[j].contiguous()
                call("ff_quant_weight_fp8_block", ptr(wj), ptr(codes[j]), ptr(scales[j]), n, k, stream())
            return codes.reshape(w.shape), scales.reshape(*w.shape[:-2], *scales.shape[1:])
        self._take(*quantise(gate_up), *quantise(down))

    @classmethod
    def from_codes(cls, gate_up, gate_up_scales, down, down_scales):
        op = cls.__new__(cls)
        op._take(gate_up, gate_up_scales, down, down_scales)
        return op

    def _take(self, gate_up, gate_up_scales, down, down_scales):
        check_block_codes(gate_up, gate_up_scales, 4)
        check_block_codes(down, down_scales, 3)
        check_here(gate_up, down)
        e, two, i, h = gate_up.shape
        assert two == 2 and down.shape == (e, h, i) and 0 < e <= MAX_EXPERTS, (gate_up.shape, down.shape)
        self.experts, self.hidden, self.inter = e, h, i
        self.gate_up = pack_blocks(gate_up.contiguous(), 128)
        self.down = pack_blocks(down.contiguous())
        self.gate_up_scale = gate_up_scales.float().contiguous()
        self.down_scale = down_scales.float().contiguous()

    def __call__(self, x, weights, ids):
        """x (T, H) bf16, weights (T, top_k) fp32, ids (T, top_k) int32 -> (T, H) bf16. An id
        outside [0, E) is no expert and adds nothing (a row without one is 0); an expert
        may come twice."""
        assert x.dim() == 2 and x.dtype == BF16 and x.shape[1] == self.hidden, (x.shape, x.dtype)
        t, h = x.shape
        assert weights.shape == ids.shape and ids.dim() == 2 and ids.shape[0] == t and ids.shape[1] > 0
        assert weights.dtype == F32 and ids.dtype == I32 and weights.is_contiguous() and ids.is_contiguous()
        check_here(x, weights, ids, self.down_scale)
        if x.stride(-1) != 1 and h > 1:
            x = x.contiguous()
        top_k = ids.shape[1]
        y = x.new_empty((t, h))
        need = experts_workspace(t, top_k, self.experts, h, self.inter)
        ws = x.new_empty((need,), dtype=torch.uint8)
        entry("ff_moe_experts")(x.data_ptr(), x.stride(0), weights.data_ptr(), ids.data_ptr(),
                                self.gate_up._packed.data_ptr(), self.gate_up_scale.data_ptr(),
                                self.down._packed.data_ptr(), self.down_scale.data_ptr(), y.data_ptr(), h, t, top_k,
                                self.experts, h, self.inter, ws.data_ptr(), need, stream())
        return y


class Router:
    """The router's linear: logits (T, E) bf16 = bf16(x . weight^T) from a bf16 weight (E, H),
    E % 4 == 0 and H % 64 == 0."""

    def __init__(self, weight):
        assert weight.dim() == 2 and weight.dtype == BF16 and weight.shape[0] % 4 == weight.shape[1] % 64 == 0
        check_here(weight)
        self.weight = weight.contiguous()
        self.zero = torch.zeros(weight.shape[0], device=weight.device, dtype=BF16)     # ff_gemm_bf16 takes a bias

    def __call__(self, x):
        assert x.dim() == 2 and x.dtype == BF16 and x.shape[1] == self.weight.shape[1]
        check_here(x, self.weight)
        m, k = x.shape
        n = self.weight.shape[0]
        lda = k if m == 1 else x.stride(0)
        if x.stride(1) != 1 or lda < k or lda % 8 or x.data_ptr() % 16:     # what ff_gemm_bf16 reads in place
            x, lda = x.clone(memory_format=torch.contiguous_format), k
        y = x.new_empty((m, n))
        if m:
            call("ff_gemm_bf16", ptr(x), lda, ptr(self.weight), ptr(self.zero), ptr(y), n, None, 0, m, n, k, 0,
                 stream())
        return y


class MoE:
    """A layer's mixture-of-experts MLP: ``router`` (a callable to logits (T, E), e.g.
    ``Router``), ``experts`` and the arguments of ``route``. ``moe(x)``: x (..., H) bf16 ->
    (..., H) bf16."""

    def __init__(self, router, experts, top_k, **routing):
        self.router, self.experts, self.top_k, self.routing = router, experts, top_k, routing

    def __call__(self, x):
        flat = x.reshape(-1, x.shape[-1])
        weights, ids = route(self.router(flat), self.top_k, **self.routing)
        return self.experts(flat, weights, ids).reshape(x.shape)


__all__ = ["route", "Experts", "Router", "MoE"]
