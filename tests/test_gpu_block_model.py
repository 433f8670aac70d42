"""Block-scaled FP8 and mixture-of-experts layers where the framework runs them: the step
(eager against the 64-bit oracle, graph replays against eager), block-scaled
checkpoints, the request API's linear format."""
import json
import os

import pytest
import torch

from oracle import moe as M

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"


def _request(cfg, tokens=70):
    from fastforward_amd.synthetic import make_request
    return make_request(cfg, tokens, 4, 6, seed=3)


@pytest.mark.gpu
def test_moe_step(gpu):
    """Every layer's MLP (router, routing, experts) against the oracle, teacher-forced on the
    step's own normalised activations; the tail's single row; graph replays = eager steps."""
    from fastforward_amd import ops
    from fastforward_amd.linear import Linear
    from fastforward_amd.runtime import LMConfig, Runtime
    from fastforward_amd.synthetic import make_model
    cfg = LMConfig("moe", 3, 512, 4, 2, 128, 136, 1000, experts=12, top_k=3)
    w = make_model(cfg, mode="fp8_block", seed=5, norm_jitter=0.2, n_options=4)
    assert Runtime.path_for(w) == "generic" and w.layers[0].gateup is None
    ids, pos, pick = _request(cfg)
    rt = Runtime(cfg, w, 70)
    rt.set_inputs(ids, pos, pick)
    trace = []
    eager = rt.step(trace=trace).clone()
    h = rt._prologue()[None]
    for j, lw in enumerate(w.layers[:-1]):
        x = ops.fast_norm(h, lw.input_norm)
        attn = rt._attention_generic(lw, x, rt.cos[None], rt.sin[None])
        residual, post = ops.add_rms(h, Linear.apply(attn, lw.o), None, lw.post_norm)
        moe, p = lw.moe, post[0]
        logits = moe.router(p)
        exact = p.cpu().double() @ moe.router.weight.cpu().double().T
        # one bf16 rounding and fp32 sums of 512 products
        assert ((logits.cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 1e-4).all()
        weights, chosen = M.route(logits.cpu(), 3)
        want, bound = M.experts(p.cpu(), weights, chosen, moe.experts.gate_up.cpu(), moe.experts.gate_up_scale.cpu(),
                                moe.experts.down.cpu(), moe.experts.down_scale.cpu())
        assert ((moe(p).cpu().double() - want).abs() <= bound + 1e-9).all(), f"layer {j}"
        h = residual + moe(post)
        assert torch.equal(h[0], trace[j])
    rt.capture()
    for k in range(3):
        ids2 = (ids * (k + 3) + k) % cfg.vocab
        rt.set_inputs(ids2, pos, pick - k)
        z = rt.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(z, rt.step())
    rt.set_inputs(ids, pos, pick)
    assert torch.equal(rt.replay(), eager)


@pytest.mark.gpu
def test_block_step(gpu):
    """The step with block-scaled linears: every linear of every full layer within the oracle's
    bound on the step's own activations, and graph replays = eager."""
    from fastforward_amd import ops
    from fastforward_amd.linear import BlockFP8Linear, Linear
    from fastforward_amd.runtime import LMConfig, Runtime
    from fastforward_amd.synthetic import make_model
    cfg = LMConfig("block", 3, 512, 4, 2, 128, 1024, 1000)
    ids, pos, pick = _request(cfg)
    w = make_model(cfg, mode="fp8_block", seed=5, norm_jitter=0.2, n_options=4)
    rt = Runtime(cfg, w, 70)
    assert rt.path == "generic" and all(isinstance(op, BlockFP8Linear) for op in w.layers[0].linears)
    rt.set_inputs(ids, pos, pick)
    trace = []
    eager = rt.step(trace=trace).clone()

    def check(op, x):
        y = Linear.apply(x, op)
        want, bound = M.linear(x[0].cpu(), op.weight.cpu(), op.scale.cpu())
        assert ((y[0].cpu().double() - want).abs() <= bound).all()
        return y

    h = rt._prologue()[None]
    for j, lw in enumerate(w.layers[:-1]):
        x = ops.fast_norm(h, lw.input_norm)
        check(lw.qkv, x)
        attn = rt._attention_generic(lw, x, rt.cos[None], rt.sin[None])
        residual, post = ops.add_rms(h, check(lw.o, attn), None, lw.post_norm)
        g, u = check(lw.gateup, post).chunk(2, -1)
        h = residual + check(lw.down, ops.swiglu(g, u))
        assert torch.equal(h[0], trace[j])
    for _ in range(3):
        assert torch.equal(rt.replay(), eager)
        torch.cuda.synchronize()


class Observe:
    """An op that keeps what it was given and what it returned."""

    def __init__(self, op, seen, name):
        self.op, self.seen, self.name = op, seen, name

    def __getattr__(self, name):
        return getattr(self.op, name)

    def __call__(self, x):
        y = self.op(x)
        self.seen[self.name] = (x.clone(), y.clone())
        return y


def _check_moe(moe, x, y, top_k, what):
    x, y = x.reshape(-1, x.shape[-1]), y.reshape(-1, y.shape[-1])
    weights, chosen = M.route(moe.router(x).cpu(), top_k)
    e = moe.experts
    want, bound = M.experts(x.cpu(), weights, chosen, e.gate_up.cpu(), e.gate_up_scale.cpu(), e.down.cpu(),
                            e.down_scale.cpu())
    assert ((y.cpu().double() - want).abs() <= bound + 1e-9).all(), what


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [0, 12])
@pytest.mark.parametrize("pick", [69, 31])
def test_last_layer_row(gpu, experts, pick):
    """The last layer runs one row: every op of it, dense and with experts, is given what the
    residual stream before it and the op before it make, and the logits are the readout of
    its result."""
    from oracle import ops as O
    from fastforward_amd import ops
    from fastforward_amd.runtime import LMConfig, Runtime
    from fastforward_amd.synthetic import make_model
    from tests.helpers import assert_bf16_close
    cfg = LMConfig("tail", 2, 512, 4, 2, 128, 136 if experts else 1024, 1000, experts=experts,
                   top_k=3 if experts else 0)
    w = make_model(cfg, mode="fp8_block", seed=6, norm_jitter=0.2, n_options=4)
    ids, pos, _ = _request(cfg)
    rt = Runtime(cfg, w, 70)
    rt.set_inputs(ids, pos, pick)
    eager = rt.step().clone()
    lw, seen, trace = w.layers[-1], {}, []
    plain = {name: op for name, op in vars(lw).items() if name in ("qkv", "o", "gateup", "down", "moe") and op}
    try:
        for name, op in plain.items():
            setattr(lw, name, Observe(op, seen, name))
        logits = rt.step(trace=trace).clone()
    finally:
        for name, op in plain.items():
            setattr(lw, name, op)
    assert torch.equal(logits, eager)

    def linear(name):
        x, y = seen[name]
        op = plain[name]
        want, bound = M.linear(x.reshape(-1, x.shape[-1]).cpu(), op.weight.cpu(), op.scale.cpu())
        assert ((y.reshape(want.shape).cpu().double() - want).abs() <= bound).all(), name

    h = trace[-1][None]
    x = ops.fast_norm(h, lw.input_norm)
    assert torch.equal(seen["qkv"][0], x)
    linear("qkv")
    # the attention of every row: the same row twice, each within a rounding of its weights and of its result
    attn = rt._attention_generic(lw, x, rt.cos[None], rt.sin[None])[0, pick].double()
    assert float((seen["o"][0].reshape(-1).double() - attn).norm() / attn.norm()) <= 2.0 ** -6
    linear("o")
    residual, post = ops.add_rms(h[:, pick:pick + 1].contiguous(), seen["o"][1].reshape(1, 1, -1), None, lw.post_norm)
    if experts:
        x, mlp = seen["moe"]
        _check_moe(plain["moe"], x, mlp, 3, "experts")
    else:
        x, gate_up = seen["gateup"]
        linear("gateup")
        mid, mlp = seen["down"]
        assert torch.equal(mid.reshape(-1), ops.swiglu(*gate_up.chunk(2, -1)).reshape(-1))
        linear("down")
    assert torch.equal(x.reshape(-1), post.reshape(-1))
    last = (residual.reshape(1, -1) + mlp.reshape(1, -1)).cpu()
    z = O.lm_readout(last, w.norm.weight.cpu(), cfg.eps, w.head.cpu())[0]
    assert_bf16_close(logits.cpu().to(BF16), z.to(BF16), 1, 0.25, "logits")


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["fp8", "fp8_static", "w4a16", "int4"])
def test_experts_beside_other_linears(gpu, mode):
    """The experts' format does not depend on the linears'."""
    from fastforward_amd.runtime import LMConfig, Runtime
    from fastforward_amd.synthetic import make_model
    cfg = LMConfig("modes", 3, 512, 4, 2, 128, 136, 1000, experts=12, top_k=3)
    w = make_model(cfg, mode=mode, seed=5, norm_jitter=0.2, n_options=4)
    rt = Runtime(cfg, w, 70)
    assert rt.path == "generic"
    rt.set_inputs(*_request(cfg))
    seen, moes = {}, [lw.moe for lw in w.layers]
    for j, lw in enumerate(w.layers):
        lw.moe = Observe(lw.moe, seen, j)
    eager = rt.step().clone()
    for lw, moe in zip(w.layers, moes):
        lw.moe = moe
    assert eager.isfinite().all()
    for j, moe in enumerate(moes):
        assert seen[j][0].numel() == 512 * (1 if j == 2 else 70)
        _check_moe(moe, *seen[j], 3, f"layer {j}")
    for _ in range(3):
        assert torch.equal(rt.replay(), eager)
        torch.cuda.synchronize()


def _save_block_checkpoint(tmp_path):
    """The tiny transformers checkpoint with its LM linears block-scaled FP8."""
    from safetensors import safe_open
    from safetensors.torch import save_file
    from tests.test_checkpoint import _tiny_hf
    _, path = _tiny_hf(tmp_path, seed=3)
    fn = os.path.join(path, "model.safetensors")
    with safe_open(fn, "pt") as f:
        tensors = {k: f.get_tensor(k) for k in f.keys()}
    for name in list(tensors):
        if ".language_model.layers." in name and name.endswith("_proj.weight"):
            tensors[name], tensors[name + "_scale_inv"] = M.quant_weight(tensors[name])
    save_file(tensors, fn)
    return path, tensors


def test_block_checkpoint_tensors(tmp_path):
    from fastforward_amd.checkpoint import Tensors
    path, tensors = _save_block_checkpoint(tmp_path)
    ts = Tensors(path)
    name = "model.language_model.layers.0.mlp.down_proj.weight"
    codes, scales = ts.blocks(name, "cpu")
    assert torch.equal(codes.view(torch.uint8), tensors[name].view(torch.uint8))
    want = (codes.float() * M.expand(scales, *codes.shape).float()).to(BF16)
    assert torch.equal(ts.get(name, "cpu"), want)
    assert ts.blocks("model.language_model.norm.weight", "cpu") is None
    from safetensors.torch import save_file
    tensors[name + "_scale_inv"] = tensors[name + "_scale_inv"][:1].contiguous()
    save_file(tensors, os.path.join(path, "model.safetensors"))
    with pytest.raises(ValueError, match="scales"):
        Tensors(path).get(name, "cpu")


def test_expert_checkpoint_is_refused(tmp_path):
    """By name, and before any tensor is read."""
    from safetensors.torch import save_file
    from fastforward_amd.checkpoint import Tensors, load_lm
    from fastforward_amd.runtime import LMConfig
    q = "model.language_model.layers."
    save_file({q + "0.mlp.gate_proj.weight": torch.zeros(8, 4), q + "1.mlp.gate.weight": torch.zeros(2, 4),
               q + "1.mlp.experts.down_proj": torch.zeros(2, 8, 4)}, os.path.join(tmp_path, "model.safetensors"))
    cfg = LMConfig("experts", 2, 4, 1, 1, 128, 8, 10)
    for ts in (None, Tensors(str(tmp_path))):
        with pytest.raises(ValueError, match="layer 1 .* mixture of experts"):
            load_lm(str(tmp_path), cfg, [0, 1], mode="fp8_block", device="cpu", tensors=ts)


@pytest.mark.gpu
def test_tensors_reach_the_gpu_in_bf16(gpu, tmp_path):
    """A tensor of another type is converted on its way: the GPU holds its bf16 copy only."""
    from safetensors.torch import save_file
    from fastforward_amd.checkpoint import Tensors
    w = torch.randn(2048, 1024, generator=torch.Generator().manual_seed(4))
    save_file({"w": w}, os.path.join(tmp_path, "model.safetensors"))
    ts = Tensors(str(tmp_path))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ts.get("w", DEV)
    assert torch.cuda.max_memory_allocated() - before <= 2 * w.numel() + 512
    assert torch.equal(got.cpu(), w.to(BF16))


@pytest.mark.gpu
def test_block_checkpoint_loads(gpu, tmp_path):
    """fp8_block takes the checkpoint's codes and scales as they are, fp8 the dequantised weight."""
    from fastforward_amd.checkpoint import load_pretrained
    from fastforward_amd.linear import BlockFP8Linear, FP8Linear
    path, tensors = _save_block_checkpoint(tmp_path)
    p = "model.language_model.layers.1."
    names = [p + f"self_attn.{x}_proj.weight" for x in "qkv"]
    codes = torch.cat([tensors[n].view(torch.uint8) for n in names])
    scales = torch.cat([tensors[n + "_scale_inv"] for n in names])
    _, lw, _, _, _ = load_pretrained(path, option_ids=list(range(8)), mode="fp8_block")
    op = lw.layers[1].qkv
    assert isinstance(op, BlockFP8Linear)
    assert torch.equal(op.weight.cpu().view(torch.uint8), codes) and torch.equal(op.scale.cpu(), scales)
    _, lw, _, _, _ = load_pretrained(path, option_ids=list(range(8)), mode="fp8")
    want = FP8Linear(M.dequant(codes.view(E4M3), scales).float().to(BF16).to(DEV))
    assert torch.equal(lw.layers[1].qkv.weight.view(torch.uint8), want.weight.view(torch.uint8))


@pytest.mark.gpu
def test_block_bundle(gpu, tmp_path):
    """A bundle's linear: fp8_block serves token requests."""
    from fastforward_amd import runtime
    from fastforward_amd.api import Accelerator
    from fastforward_amd.runtime import LMConfig
    runtime.PRESETS["tiny-block"] = LMConfig("tiny-block", 2, 256, 2, 1, 128, 512, 1000)
    try:
        p = tmp_path / "bundle.json"
        p.write_text(json.dumps(dict(schema_version=1, task="visual_choice", architecture="qwen3_vl_lm",
                                     preset="tiny-block", linear="fp8_block", seed=1, tokens=64, image_grid=[4, 4],
                                     prefix_tokens=4)))
        acc = Accelerator(str(p))
        r = acc.predict_tokens(list(range(5, 45)), ["a", "b", "c"])
        assert len(r["logits"]) == 3 and r["answer"]["text"] in ("a", "b", "c")
    finally:
        del runtime.PRESETS["tiny-block"]
