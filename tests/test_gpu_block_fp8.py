"""The block-scaled FP8 linear on the GPU: codes, scales and packing bit for bit,
products within the bound that the 64-bit oracle derives (one bf16 rounding, the
matrix instruction's alignment error), strides, sizes from one, special values,
streams and graphs; refusals on the CPU."""
import ctypes

import pytest
import torch

from oracle import moe as M

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"
gpu_test = pytest.mark.gpu

# (m, n, k): one row to several row tiles, sizes of one, ends inside a block, a
# fragment, a vector; more k steps than waves and fewer
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 300, 700), (2, 16, 130), (3, 129, 1025), (4, 512, 4096), (5, 100, 257), (5, 64, 4096), (9, 8200, 130), (16, 80, 1024),
          (7, 2560, 640), (16, 48, 384), (17, 33, 129), (31, 200, 1152), (33, 257, 512), (64, 80, 2049), (65, 384, 300),
          (100, 1152, 431), (129, 640, 896), (333, 136, 264)]


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _case(m, n, k, seed=0):
    x = torch.randn(m, k, generator=_g(seed))
    x[torch.rand(m, k, generator=_g(seed + 1)) < 0.01] *= 20
    codes = (torch.randn(n, k, generator=_g(seed + 2)) * 60).clamp(-448, 448).to(E4M3)
    scale = torch.rand(-(-n // 128), -(-k // 128), generator=_g(seed + 3)) * 1e-3 + 1e-5
    return x.to(BF16), codes, scale


def _op(codes, scale):
    from fastforward_amd.linear import BlockFP8Linear
    return BlockFP8Linear.from_codes(codes.to(DEV), scale.to(DEV))


def _check(y, x, codes, scale):
    want, bound = M.linear(x, codes, scale)
    excess = ((y.cpu().double() - want).abs() - bound).max()
    assert float(excess) <= 0, f"{tuple(x.shape)} x {tuple(codes.shape)}: beyond the bound by {float(excess)}"


@gpu_test
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(gpu, m, n, k):
    x, codes, scale = _case(m, n, k)
    op = _op(codes, scale)
    y = op(x.to(DEV))
    assert y.shape == (m, n) and y.dtype == BF16
    _check(y, x, codes, scale)
    q, s = op.quantize(x.to(DEV))
    want_q, want_s = M.quant_rows(x)
    assert torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s.cpu(), want_s)
    assert m <= 16 or torch.equal(op.gemm(q, s), y)    # up to 16 rows: may be one launch, other sums' order
    assert torch.equal(op.weight.cpu().view(torch.uint8), codes.view(torch.uint8))


@gpu_test
@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_every_kernel(gpu, m, n, k, tile):
    """Each kernel of the product at sizes that another would be chosen for."""
    from fastforward_amd._lib import call
    x, codes, scale = _case(m, n, k)
    op = _op(codes, scale)
    q, s = op.quantize(x.to(DEV))
    call("ff_set_tuning", 12, tile)
    try:
        y = op.gemm(q, s)
    finally:
        call("ff_set_tuning", 12, 0)
    _check(y, x, codes, scale)


@gpu_test
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (7, 19456, 2560), (48, 2048, 6144), (176, 6144, 4096),
                                   (576, 4096, 2048), (500, 5120, 8200), (1024, 2560, 9728), (700, 1152, 4304)])
def test_linear_at_model_sizes(gpu, m, n, k):
    """Relative RMS against float64 on the GPU: one bf16 rounding is at most 2^-8 / sqrt(3)
    = 2.3e-3; the sums' error adds less than a tenth of that."""
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(m, k, generator=g, device=DEV).to(BF16)
    codes = (torch.randn(n, k, generator=g, device=DEV) * 60).clamp(-448, 448).to(E4M3)
    scale = torch.rand(-(-n // 128), -(-k // 128), generator=g, device=DEV) * 1e-3 + 1e-5
    from fastforward_amd.linear import BlockFP8Linear
    op = BlockFP8Linear.from_codes(codes, scale)
    q, s = op.quantize(x)
    want = M.rows_values(q, s, k) @ M.dequant(codes, scale).T
    y = op(x).double()
    assert float((y - want).norm() / want.norm()) <= 2.5e-3
    # and no element apart: 2^-8 of the value and 1/64 of the row's RMS (sum_error's bound at these sizes)
    assert bool(((y - want).abs() <= 2.0 ** -8 * want.abs() + want.square().mean(1, keepdim=True).sqrt() / 64).all())


# A wave of the tile kernels holds the block scales of 63 or 64 k steps at once, of its k group where
# there are two: these k blocks come after them.
LATE_BLOCKS = (63, 64, 128, 129)


def late_scales(shape, seed):
    """Block scales over a factor of 256, those of LATE_BLOCKS 16 times larger: a scale taken
    from another block shows in the whole sum."""
    s = torch.exp2(torch.randint(-8, 1, shape, generator=_g(seed)).float()) * 1e-3
    for b in LATE_BLOCKS:
        s[..., b:b + 1] *= 16
    return s


@gpu_test
@pytest.mark.parametrize("k", [8264, 16584])
def test_more_block_scales_than_lanes(gpu, k):
    """Every kernel past the first scales that its waves load. Beside the oracle's bound (for
    every 32 products 2^-9 of the largest) there are 130 fp32 additions, each off by 2^-24
    of at most 32 times the same sum: 2^-12 of it, an eighth more."""
    from fastforward_amd._lib import call
    m, n = 33, 136
    x, codes, scale = _case(m, n, k)
    scale = late_scales(scale.shape, 7)
    op = _op(codes, scale)
    q, s = op.quantize(x.to(DEV))
    want, bound = M.linear(x, codes, scale)
    for tile in range(6):
        call("ff_set_tuning", 12, tile)
        try:
            y = op.gemm(q, s).cpu().double()
        finally:
            call("ff_set_tuning", 12, 0)
        assert ((y - want).abs() <= 1.125 * bound).all(), f"tile {tile}"


@gpu_test
def test_weight_quantisation(gpu):
    from fastforward_amd.linear import BlockFP8Linear
    for n, k in ((1, 1), (128, 128), (200, 300), (257, 129)):
        w = (torch.randn(n, k, generator=_g(n)) * 0.02).to(BF16)
        op = BlockFP8Linear(w.to(DEV))
        codes, scale = M.quant_weight(w)
        assert torch.equal(op.scale.cpu(), scale)
        assert torch.equal(op.weight.cpu().view(torch.uint8), codes.view(torch.uint8))


@gpu_test
@pytest.mark.parametrize("m", [1, 4, 5, 40])
def test_strides_and_shapes(gpu, m):
    """Rows at odd strides and offsets, broadcast rows, transposed views, leading
    dimensions: the bits of a contiguous copy."""
    k, n = 130, 70
    _, codes, scale = _case(m, n, k)
    op = _op(codes, scale)
    base = torch.randn(m + 2, 2 * k + 3, generator=_g(9)).to(BF16).to(DEV)
    for x in (base[:m, :k], base[1:m + 1, 3:3 + k], base[:m, 8:8 + k], base[:m, ::2][:, :k], base[:1, :k].expand(m, k),
              torch.randn(k, m, generator=_g(10)).to(BF16).to(DEV).T):
        before = x.clone()
        y = op(x)
        assert torch.equal(y, op(x.contiguous())) and torch.equal(x, before)
    _check(op(base[1:m + 1, 3:3 + k]), base[1:m + 1, 3:3 + k].cpu(), codes, scale)
    x3 = base[:m, :k].reshape(1, m, k)
    assert op(x3).shape == (1, m, n) and torch.equal(op(x3)[0], op(base[:m, :k]))
    assert op(base[0, :k]).shape == (n,)
    assert op(base[:0, :k]).shape == (0, n)


@gpu_test
@pytest.mark.parametrize("m", [1, 5, 80])
def test_special_values(gpu, m):
    """Zero rows give zeros; a NaN or an infinity stays in its row; the smallest and the
    largest magnitudes quantise against their own group."""
    n, k = 40, 384
    x, codes, scale = _case(m, n, k)
    x[0] = 0
    y = _op(codes, scale)(x.to(DEV)).cpu()
    assert (y[0] == 0).all()
    _check(y, x, codes, scale)
    for bad in (float("nan"), float("inf"), -float("inf")):
        xb = x.clone()
        xb[-1, 200] = bad
        yb = _op(codes, scale)(xb.to(DEV)).cpu()
        assert yb[-1].isnan().all() and torch.equal(yb[:-1], y[:-1])
    x[-1, :128], x[-1, 128:256] = 3e38, 1e-30
    yb = _op(codes, torch.full_like(scale, 1e-4))(x.to(DEV))
    q, s = M.quant_rows(x)
    assert torch.equal(_op(codes, scale).quantize(x.to(DEV))[0].cpu().view(torch.uint8), q.view(torch.uint8))
    assert torch.equal(yb[:-1].isnan(), torch.zeros_like(yb[:-1]).bool())


@gpu_test
def test_quantise_special_values(gpu):
    """Beside an infinity x / scale is 0 and its own code NaN; a NaN keeps its code and
    leaves the others to the largest number."""
    inf, nan = float("inf"), float("nan")
    x, codes, scale = _case(8, 16, 300)
    x[1, 7], x[2, 128:256], x[3, 299], x[4, 0], x[4, 1] = inf, -inf, -inf, inf, -inf
    x[5, 3], x[6, 128:256], x[7, 298] = nan, nan, nan
    q, s = _op(codes, scale).quantize(x.to(DEV))
    q = q.cpu()
    none = torch.nn.functional.pad(~x.isfinite(), (0, 84))
    want_q, want_s = M.quant_rows(x.masked_fill(x.isnan(), 0))
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.float().isnan(), none)
    assert torch.equal(q.view(torch.uint8)[~none], want_q.view(torch.uint8)[~none])


@gpu_test
@pytest.mark.parametrize("m", [1, 6, 96])
def test_graph_and_stream(gpu, m):
    """Captured once, replayed on new inputs with eager calls between; on a side stream."""
    x, codes, scale = _case(m, 192, 640)
    op = _op(codes, scale)
    static = x.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = op(static)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, op(static))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(static)
    for seed in (11, 12, 13):
        xi = torch.randn(m, 640, generator=_g(seed)).to(BF16).to(DEV)
        static.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, op(xi))


@gpu_test
def test_offsets_past_32_bits(gpu):
    """More than 2^32 codes of activations: equal rows of x give equal rows of y."""
    from fastforward_amd.linear import BlockFP8Linear
    rows, times, n, k = 1024, 64, 128, 65792
    g = torch.Generator(device=DEV).manual_seed(0)
    op = BlockFP8Linear((torch.randn(n, k, generator=g, device=DEV) * 0.02).to(BF16))
    base = torch.randn(rows, k, generator=g, device=DEV).to(BF16)
    y = op(base.repeat(times, 1)).view(times, rows, n)
    assert (y == y[:1]).all()
    want = op(base).float()     # another tile's order of sums: two bf16 roundings apart at most
    assert float((y[0].float() - want).norm() / want.norm()) <= 2 ** -7


@gpu_test
def test_two_streams(gpu):
    """Calls that overlap on two streams share nothing."""
    from fastforward_amd.linear import BlockFP8Linear
    g = torch.Generator(device=DEV).manual_seed(1)
    op = BlockFP8Linear((torch.randn(512, 1024, generator=g, device=DEV) * 0.02).to(BF16))
    xs = [torch.randn(m, 1024, generator=g, device=DEV).to(BF16) for m in (40, 300)]
    want = [op(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(op(xs[j]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_refusals_python():
    """Checked before any launch: no GPU is touched."""
    from fastforward_amd.linear import BlockFP8Linear
    codes = torch.zeros(4, 4).to(E4M3)
    for c, s in ((codes, torch.ones(1, 1)), (codes.float(), torch.ones(1, 1)), (codes[0], torch.ones(1, 1))):
        with pytest.raises(AssertionError):
            BlockFP8Linear.from_codes(c, s)
    with pytest.raises(AssertionError):
        BlockFP8Linear(torch.zeros(4, 4, dtype=BF16))


def test_refusals_c():
    from fastforward_amd import _lib
    _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    need = ctypes.c_int64(-1)
    bad = [("ff_linear_fp8_block", (p, 8, p, p, p, 8, 1, 0, 8, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 7, 1, 8, 8, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 1 << 20, 1, 1 << 20, 1 << 20, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 1 << 23, 1, 1 << 23, 64, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 8, 17, 8, 1 << 24, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 8, 1 << 24, 8, 128 * 64, None, 0, None), "bad sizes"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 8, 17, 8, 8, None, 0, None), "workspace"),
           ("ff_linear_fp8_block", (p, 8, p, p, p, 8, 17, 8, 8, p, 16, None), "workspace"),
           ("ff_linear_fp8_block", (None, 8, p, p, p, 8, 1, 8, 8, None, 0, None), "null"),
           ("ff_linear_fp8_block", (p + 1, 8, p, p, p, 8, 1, 8, 8, None, 0, None), "alignment"),
           ("ff_gemm_fp8_block", (p, p, p + 8, p, p, 8, 1, 8, 8, None), "alignment"),
           ("ff_gemm_fp8_block", (p, None, p, p, p, 8, 1, 8, 8, None), "null"),
           ("ff_quant_rows_fp8_block", (p, 8, p, p, -1, 8, None), "bad sizes"),
           ("ff_quant_weight_fp8_block", (p, p, p, 0, 8, None), "bad sizes"),
           ("ff_pack_weight_fp8_block", (p, p, 1, 17, 8, 16, None), "bad sizes"),
           ("ff_pack_weight_fp8_block", (p, p, 1, 8, 8, 24, None), "bad sizes"),
           ("ff_unpack_weight_fp8_block", (p, None, 1, 8, 8, 16, None), "null")]
    for name, args, message in bad:
        with pytest.raises(RuntimeError, match=message):
            _lib.call(name, *args)
    for m, n, k, want in ((1, 4096, 4096, 0), (4, 8192, 4096, 0), (4, 8193, 4096, 1), (4, 16, 4097, 1), (16, 16, 1024, 0),
                          (17, 16, 128, 1), (0, 16, 128, 0)):
        _lib.call("ff_linear_fp8_block_workspace", m, n, k, ctypes.byref(need))
        assert (need.value > 0) == bool(want), (m, n, k, need.value)
    _lib.call("ff_linear_fp8_block", None, 8, None, None, None, 8, 0, 8, 8, None, 0, None)   # no rows: nothing to do
