"""The paged cache and its attention on the GPU against the 64-bit oracle: pages anywhere,
ragged batches, rows without a place, one token to chunks, groups of any size, masked
garbage, strides, streams, graphs; refusals on the CPU."""
import ctypes
import math

import pytest
import torch

from oracle import serving as S

BF16, E4M3, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
DEV = "cuda"
gpu_test = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _rows(seed, *shape, gain=1.0):
    return (torch.randn(*shape, generator=_g(seed)) * gain).to(BF16)


class Case:
    """A cache filled at random on both sides, sequences on pages anywhere."""

    def __init__(self, lengths, new, hk=2, d=128, ps=16, dtype=BF16, seed=0, spare=2, width=None, fill=True):
        from fastforward_amd.cache import PagedCache
        self.lengths = torch.tensor(lengths, dtype=I32)
        need = [max(0, -(-n // ps)) for n in lengths]
        self.width = max(1, *need) if width is None else width
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=_g(seed)).to(I32)
        self.table = torch.full((len(lengths), self.width), -1, dtype=I32)
        at = 0
        for i, n in enumerate(need):
            n = min(n, self.width)
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = None if new is None else torch.tensor([0] + list(new)).cumsum(0).to(I32)
        self.t = len(lengths) if new is None else sum(new)
        self.hk, self.d, self.ps, self.dtype = hk, d, ps, dtype
        self.dev = PagedCache(pages, ps, hk, d, dtype)
        self.cpu = {}
        for i, name in enumerate(("k", "v")):
            x = _rows(seed + 11 + i, pages, hk, ps, d) if fill else torch.zeros(pages, hk, ps, d, dtype=BF16)
            if dtype == BF16:
                self.cpu[name] = x
            else:
                self.cpu[name], self.cpu[name + "_scale"] = S.codes(x)
            self.upload(name)

    def upload(self, name):
        getattr(self.dev, name).copy_(self.cpu[name])
        if self.dtype == E4M3:
            getattr(self.dev, name + "_scale").copy_(self.cpu[name + "_scale"])

    def args(self, starts=True):
        return [x if x is None else x.to(DEV) for x in (self.table, self.lengths, self.starts)[:3 if starts else 2]]

    def check_attend(self, q, scale=None):
        y = self.dev.attend(q.to(DEV), *self.args(), scale=scale)
        o, a, most = S.attend(self.cpu, q, self.table, self.lengths, self.starts, scale)
        assert y.shape == q.shape and y.dtype == BF16
        return close(y, o, a, most, self.d)


def close(y, o, a, most, d):
    """The output's rounding 2^-8 |o|; the weights' 2^-8 of sum p |v|; and the fp32 work before: scores
    off by (d + 8) 2^-24 of the largest sum of |q k| scale on both sides of the maximum, their difference
    and its product with log2 e by 2^-23 of it each, 2^-22 for the exponential and 2^-18 for the sums."""
    y = y.cpu().double()
    assert torch.equal(y.isnan(), o.isnan())
    e = 2.0 ** -8 + 2 * ((d + 8) * 2.0 ** -24 + 2.0 ** -22) * most + 2.0 ** -22 + 2.0 ** -18
    off = ((y - o).abs() - 2.0 ** -8 * o.abs() - e * a).nan_to_num(0)
    assert float(off.max()) <= 1e-30, float(off.max())
    return y, o


# ---------------------------------------------------------------- write, read

@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("hk,d,ps,lengths,new", [
    (8, 128, 64, [1], None), (2, 64, 16, [5, 1, 33, 16, 17], None), (3, 128, 32, [40, 7], [33, 7]),
    (1, 64, 256, [300, 0, 12], [299, 0, 11]), (5, 128, 16, [70] * 70, [1] * 70), (2, 64, 4096, [4100], [3]),
    (2, 128, 16, [20, 50, 3], [20, 41, 3])])
def test_write_read(gpu, dtype, hk, d, ps, lengths, new):
    c = Case(lengths, new, hk, d, ps, dtype, seed=sum(lengths))
    k, v = _rows(1, c.t, hk, d, gain=3), _rows(2, c.t, hk, d, gain=0.01)
    c.dev.write(k.to(DEV), v.to(DEV), *c.args())
    S.write(c.cpu, k, v, c.table, c.lengths, c.starts)
    for name, want in c.cpu.items():                      # every byte, those of rows not written too
        assert torch.equal(getattr(c.dev, name).cpu().view(torch.uint8), want.view(torch.uint8)), name
    total = sum(lengths)
    starts = torch.tensor([0] + lengths).cumsum(0).to(I32)
    got = c.dev.read(*c.args(False), starts.to(DEV), rows=total + 3)       # and three rows of no sequence
    for x, want in zip(got, S.read(c.cpu, c.table, c.lengths, starts, total + 3)):
        assert x.dtype == BF16 and torch.equal(x.cpu().double(), want)
    got = c.dev.read(*c.args(), rows=None if new is None else c.t)
    if dtype == BF16:
        assert torch.equal(got[0].cpu(), k) and torch.equal(got[1].cpu(), v)


@gpu_test
@pytest.mark.parametrize("d", [64, 128])
def test_write_codes(gpu, d):
    """Every exponent, borders between scales, zeros, subnormals, infinities and NaN."""
    x = torch.zeros(260, 1, d)
    for i in range(250):
        x[i, 0] = torch.randn(d, generator=_g(i)).clamp(-1, 1) * 2.0 ** (i - 126)
        x[i, 0, i % d] = 1.75 * 2.0 ** (i - 126) * (1 if i % 2 else 1 + 2.0 ** -7)
    x[251, 0, 3], x[252, 0, 5], x[253, 0, 7] = math.inf, -math.inf, math.nan
    x[251, 0, 9], x[252, 0, 9], x[253, 0, 9] = 3.3, 1e-3, -77.0
    x[254] = 1e-45
    x[255] = 3.38e38
    x[256, 0] = torch.linspace(-448, 448, d)
    x[257], x[258] = math.nan, -0.0
    x = x.to(BF16)
    c = Case([260], [260], 1, d, 64, E4M3)
    c.dev.write(x.to(DEV), x.to(DEV), *c.args())
    S.write(c.cpu, x, x, c.table, c.lengths, c.starts)
    assert torch.equal(c.dev.k_scale.cpu(), c.cpu["k_scale"]) and torch.equal(c.dev.v_scale.cpu(), c.cpu["v_scale"])
    for name in ("k", "v"):
        got, want = getattr(c.dev, name).cpu().float(), c.cpu[name].float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    k, _ = c.dev.read(*c.args(), rows=260)
    k, y = k.cpu().double(), x.double()
    fine = y.abs() < math.inf
    unit = torch.exp2(S.exponent(x).double())[..., None]
    assert torch.equal(k.isnan(), ~fine)
    # half a step: 2^-4 of the value, and 2^-10 of the scale below e4m3's normal range
    assert ((k - y).abs() <= torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * unit.expand_as(y)))[fine].all()


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_rows_without_a_place(gpu, tile, dtype):
    """Lengths under the rows' count, past the table, of nothing; page ids of none; rows behind the
    last sequence; starts and lengths that are nonsense."""
    c = Case([10, 5, 100, 40, 0], [6, 9, 60, 40, 2], 2, 64, 16, dtype, width=4, spare=7)
    c.table[3, 1], c.table[3, 2] = c.dev.pages, -5
    t = c.t + 9
    k, v, q = _rows(3, t, 2, 64), _rows(4, t, 2, 64), _rows(5, t, 6, 64)
    c.dev.write(k.to(DEV), v.to(DEV), *c.args())
    S.write(c.cpu, k, v, c.table, c.lengths, c.starts)
    for name, want in c.cpu.items():
        assert torch.equal(getattr(c.dev, name).cpu().view(torch.uint8), want.view(torch.uint8)), name
    for x, want in zip(c.dev.read(*c.args(), rows=t), S.read(c.cpu, c.table, c.lengths, c.starts, t)):
        assert torch.equal(x.cpu().double(), want)
    y, o = c.check_attend(q)
    assert not o[6:10].any() and not o[c.t:].any() and o[:6].any()
    # nonsense stays inside the buffers
    for starts in ([0, 50, 20, 90, 117, 117], [5, 6, -3, 1 << 30, 2, 126], [-(1 << 31)] * 6, [(1 << 31) - 1] * 6):
        for lengths in (c.lengths.tolist(), [-(1 << 31), (1 << 31) - 1, -1, 1 << 20, 3]):
            args = (c.table.to(DEV), torch.tensor(lengths, dtype=I32, device=DEV), torch.tensor(starts, dtype=I32, device=DEV))
            c.dev.write(k.to(DEV), v.to(DEV), *args)
            c.dev.read(*args, rows=t)
            c.dev.attend(q.to(DEV), *args)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- attention

@pytest.fixture(params=[0, 1, 2, 3])
def tile(request):
    """The library's own choice of tiles, then each of them for every call."""
    from fastforward_amd import _lib
    _lib.call("ff_set_tuning", 14, request.param)
    yield request.param
    _lib.call("ff_set_tuning", 14, 0)


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("hk,group,d,ps,lengths,new", [
    (1, 1, 128, 16, [1], None), (8, 4, 128, 64, [577], None), (2, 5, 64, 16, [63, 64, 65, 1, 200], None),
    (2, 16, 128, 32, [129, 128], None), (1, 17, 64, 16, [90], None), (2, 3, 128, 16, [31, 90, 4], [31, 1, 4]),
    (2, 4, 64, 64, [150, 300], [150, 61]), (1, 7, 128, 256, [333], [57]), (4, 1, 128, 32, [70, 0, 66], [70, 0, 3]),
    (2, 2, 128, 16, [257, 40, 1], [129, 40, 1]), (1, 4, 64, 16, [40] * 67, [2] * 67)])
def test_attend(gpu, tile, dtype, hk, group, d, ps, lengths, new):
    c = Case(lengths, new, hk, d, ps, dtype, seed=len(lengths) + d)
    c.check_attend(_rows(6, c.t, hk * group, d, gain=1.5))


@gpu_test
@pytest.mark.parametrize("batch,most,hk,dtype,d", [
    (63, 1, 1, BF16, 64), (64, 1, 1, E4M3, 64), (65, 3, 2, BF16, 64), (256, 1, 1, BF16, 64), (300, 1, 2, E4M3, 128),
    (700, 1, 1, BF16, 64), (260, 2, 1, E4M3, 64), (257, 1, 8, BF16, 64)])
def test_attend_many_sequences(gpu, batch, most, hk, dtype, d):
    """More sequences than a wave's lanes, short ones, none, and one that is far past the others."""
    lengths = torch.randint(0, 60, (batch,), generator=_g(batch))
    lengths[batch // 3] = 1500
    lengths[batch - 1] = 130
    new = None if most == 1 else torch.randint(0, most + 1, (batch,), generator=_g(3)).minimum(lengths).tolist()
    c = Case(lengths.tolist(), new, hk, d, 16, dtype, seed=batch)
    k, v = _rows(8, c.t, hk, d), _rows(9, c.t, hk, d)
    c.dev.write(k.to(DEV), v.to(DEV), *c.args())
    S.write(c.cpu, k, v, c.table, c.lengths, c.starts)
    for name, want in c.cpu.items():
        assert torch.equal(getattr(c.dev, name).cpu().view(torch.uint8), want.view(torch.uint8)), name
    c.check_attend(_rows(7, c.t, 2 * hk, d))
    if batch == 300:                                  # starts that say anything: other rows, but no fault
        for seed in range(3):
            odd = torch.randint(-5, 400, (batch + 1,), generator=_g(seed)).to(I32)
            q = _rows(7, c.t, 2 * hk, d).to(DEV)
            assert c.dev.attend(q, c.table.to(DEV), c.lengths.to(DEV), odd.to(DEV)).shape == q.shape
        torch.cuda.synchronize()
    if most == 1:                                     # the same rows by starts
        c.starts = torch.arange(batch + 1, dtype=I32)
        c.check_attend(_rows(7, c.t, 2 * hk, d))
        for x, y in zip(c.dev.read(*c.args(), rows=c.t + 5), c.dev.read(*c.args(False))):
            assert torch.equal(x[:c.t], y) and not x[c.t:].any()


@gpu_test
@pytest.mark.parametrize("ragged", [False, True])
def test_attend_many_sequences_graph(gpu, ragged):
    """The list of many sequences is written anew on every replay."""
    batch = 100
    lengths = [30 + i for i in range(batch)]
    lengths[40] = 5000
    c = Case(lengths, [2] * batch if ragged else None, 1, 64, 16)
    q, args = _rows(3, c.t, 4, 64).to(DEV), c.args()
    c.dev.attend(q, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.dev.attend(q, *args)
    for seed in range(4):
        now = [int(n) for n in torch.randint(2, 140, (batch,), generator=_g(seed)).minimum(c.lengths)]
        now[40] = (5000, 700, 0, 4999)[seed]
        args[1].copy_(torch.tensor(now, dtype=I32))
        q.copy_(_rows(seed, c.t, 4, 64))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, c.dev.attend(q, *args))
        close(got, *S.attend(c.cpu, q.cpu(), c.table, torch.tensor(now), c.starts), 64)


@gpu_test
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (E4M3, 128), (E4M3, 64)])
@pytest.mark.parametrize("n,heads", [(1, 4), (5, 4), (70, 2), (200, 4)])
def test_attend_every_key_counts(gpu, tile, dtype, d, n, heads):
    """Long sequences: each row looks for one key, far ahead of the others, all over the range it sees,
    borders of blocks, pages and splits among them; and all the others share the rest evenly."""
    length = 5000
    c = Case([length], [n], 1, d, 64, dtype, seed=3)
    first = length - n
    rows = n * heads
    spots = [0, 1, 63, 64, 127, 128, 255, 256, 511, 512, 1023, 1024, 2047, 2048, 4095, 4096]
    aim = torch.tensor([spots[i] if i < len(spots) and rows > 20 else
                        min(first + i // heads, (i * 7919 + 13) % length if i % 3 else first + i // heads)
                        for i in range(rows)]).reshape(n, heads)
    keys = S.values(c.cpu, "k")[c.table[0].long()[aim // 64], 0, aim % 64]        # (n, heads, d)
    c.check_attend((keys * 2).to(BF16))
    # q = 0: every visible key has the same weight, so a wrong count or a key too many shows in the mean
    for name in ("v",):
        x = torch.zeros_like(c.cpu[name].float())
        for j in range(d):
            x[..., j] = 1.0
        if dtype == BF16:
            c.cpu[name] = x.to(BF16)
        else:
            c.cpu[name], c.cpu[name + "_scale"] = S.codes(x.to(BF16))
        c.upload(name)
    y, o = c.check_attend(torch.zeros(n, heads, d, dtype=BF16))
    assert torch.equal(y, torch.ones_like(y))      # fp32 sums of equal terms up to 2^13 are exact


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_attend_counts(gpu, tile, dtype):
    """q = 0 and one-hot values by position: output j is the share of visible positions p with
    p % d == j, so that each position's being there is seen."""
    for d, n, length in ((64, 1, 1500), (128, 1, 700), (64, 90, 1100), (128, 33, 300)):
        c = Case([length], [n], 1, d, 16, dtype, seed=4)
        x = torch.zeros(c.dev.pages, 1, 16, d)
        for p in range(length):
            x[int(c.table[0, p // 16]), 0, p % 16, p % d] = 1.0
        c.cpu["v"] = x.to(BF16)
        if dtype == E4M3:
            c.cpu["v"], c.cpu["v_scale"] = S.codes(c.cpu["v"])
        c.upload("v")
        y = c.dev.attend(torch.zeros(n, 3, d, dtype=BF16, device=DEV), *c.args()).cpu().double()
        for i in range(n):
            seen = length - n + i + 1
            want = torch.tensor([len(range(j, seen, d)) / seen for j in range(d)], dtype=torch.float64)
            # counts are exact in fp32: the quotient's two roundings and the output's
            assert ((y[i] - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want).all(), (d, n, length, i)


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_attend_garbage_behind_the_mask(gpu, tile, dtype):
    """NaN and infinities in slots past the length, in pages of no sequence and, for earlier rows, in
    later rows of the same chunk; scores that overflow the exponential's range."""
    for d, new in ((128, [1, 1]), (64, [20, 37]), (128, [70, 9]), (64, [130, 140])):
        c = Case([150, 141], new, 2, d, 16, dtype, seed=5)
        q = _rows(7, c.t, 4, d)
        used = torch.zeros(c.dev.pages, 16, dtype=torch.bool)
        for b in range(2):
            for p in range(int(c.lengths[b])):
                used[int(c.table[b, p // 16]), p % 16] = True
        for name in ("k", "v"):
            bad = torch.where(torch.arange(16) % 2 == 0, math.nan, math.inf)[None, None, :, None]
            if dtype == BF16:
                c.cpu[name] = torch.where(used[:, None, :, None], c.cpu[name], bad.to(BF16))
            else:
                c.cpu[name] = torch.where(used[:, None, :, None], c.cpu[name].view(torch.uint8),
                                          torch.full((1,), 0x7F, dtype=torch.uint8)).view(E4M3)
                c.cpu[name + "_scale"] = torch.where(used[:, None, :], c.cpu[name + "_scale"],
                                                     torch.full((1,), 255, dtype=torch.uint8))
            c.upload(name)
        o = c.check_attend(q)[1]
        assert not o.isnan().any()
        c.check_attend(q * 200)                     # scores of thousands
        c.check_attend(q, scale=1e-4)
        c.check_attend(q, scale=3.0)
        # the last token of sequence 0: rows before it do not see it, its own row does
        page, slot = int(c.table[0, 149 // 16]), 149 % 16
        if dtype == BF16:
            c.cpu["v"][page, 0, slot, 3], c.cpu["v"][page, 0, slot, 9] = math.nan, math.inf
            c.cpu["v"][page, 0, slot, 17] = -math.inf
        else:
            c.cpu["v"].view(torch.uint8)[page, 0, slot, 3] = 0x7F
        c.upload("v")
        y = c.dev.attend(q.to(DEV), *c.args()).cpu().double()
        o, a, most = S.attend(c.cpu, q, c.table, c.lengths, c.starts)
        assert torch.equal(y.isnan(), o.isnan()) and torch.equal(y.isinf(), o.isinf())
        assert torch.equal(y[o.isinf()], o[o.isinf()]) and o[new[0] - 1].isnan().any()
        fine = o.abs() < math.inf
        close(y[fine], o[fine], a[fine], most, d)
        c.cpu["k"].view(torch.uint8 if dtype == E4M3 else BF16)[page, 0, slot, 3] = 0x7F if dtype == E4M3 else math.nan
        c.upload("k")
        y = c.dev.attend(q.to(DEV), *c.args()).cpu()
        rows = y.reshape(c.t, 2, 2, d)
        assert rows[new[0] - 1, 0].isnan().all() and not rows[:new[0] - 1].isnan().any() and not rows[new[0]:].isnan().any()
        assert not rows[new[0] - 1, 1].isnan().any()


@gpu_test
def test_attend_strides_streams_graph(gpu):
    c = Case([130, 77, 20], [33, 1, 20], 2, 128, 32)
    args = c.args()
    base = _rows(8, 54, 9, 256).to(DEV)
    for q in (base[:, :4, :128], base[:, 1::2, 128:], base.as_strided((54, 4, 128), (2304, 256, 1), 3),
              base[:, :4, ::2], base[:1, :4, :128].expand(54, 4, 128)):
        assert torch.equal(c.dev.attend(q, *args), c.dev.attend(q.contiguous(), *args))
    for kv in (base[:, 2:4, :128], base.as_strided((54, 2, 128), (2304, 256, 1), 5), base[:, :2, ::2]):
        c.dev.write(kv, kv, *args)
        for x in c.dev.read(*args, rows=54):
            assert torch.equal(x, kv.contiguous())
    q = base[:, :4, :128].contiguous()
    y = c.dev.attend(q, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = c.dev.attend(q, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, again)
    kv = base[:, 2:4, :128].contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.dev.write(kv, kv, *args)
        out = c.dev.attend(q, *args)
        back = c.dev.read(*args, rows=54)
    for seed in range(4):                              # inputs, lengths and the split change between replays
        q.copy_(_rows(seed, 54, 4, 128))
        kv.copy_(_rows(seed + 9, 54, 2, 128))
        args[1].copy_(torch.tensor([130 - seed, 77 - 20 * seed, 20 + seed], dtype=I32))
        args[2].copy_(torch.tensor([0, 33 - seed, 34, 54 - seed], dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, *back)]
        c.dev.write(kv, kv, *args)
        for x, want in zip(got, (c.dev.attend(q, *args), *c.dev.read(*args, rows=54))):
            assert torch.equal(x, want)
    assert c.dev.attend(q[:0], *args).shape == (0, 4, 128)
    c.dev.write(kv[:0], kv[:0], *args)


@gpu_test
def test_shared_pages_and_chunks(gpu):
    """Two sequences on one prefix's pages, and a prompt written and attended to in chunks: the rows of the
    whole at once, within the bound of both."""
    for dtype in (BF16, E4M3):
        c = Case([200, 200], [0, 0], 2, 128, 32, dtype, fill=False, spare=20)
        c.table[1, :5] = c.table[0, :5]                # 160 shared positions
        k, v, q = _rows(1, 200, 2, 128), _rows(2, 200, 2, 128), _rows(3, 200, 8, 128)
        at = 0
        parts = []
        for n in (64, 1, 31, 64, 40):
            at += n
            last = at == 200
            lengths = torch.tensor([at, at if last else 0], dtype=I32, device=DEV)
            starts = torch.tensor([0, n, 2 * n if last else n], dtype=I32, device=DEV)
            rows = [torch.cat([x[at - n:at]] * (2 if last else 1)).to(DEV) for x in (k, v, q)]
            c.dev.write(*rows[:2], c.table.to(DEV), lengths, starts)
            parts.append(c.dev.attend(rows[2], c.table.to(DEV), lengths, starts))
        assert torch.equal(parts[-1][:40], parts[-1][40:])
        y = torch.cat([*parts[:-1], parts[-1][:40]])
        starts = torch.tensor([0, 200, 200], dtype=I32)
        S.write(c.cpu, k, v, c.table, torch.tensor([200, 0]), starts)
        close(y, *S.attend(c.cpu, q, c.table, torch.tensor([200, 0]), starts), 128)


@gpu_test
def test_far_pages(gpu):
    """Page offsets past 32 bits: 2^32 values and more lie before the pages in use."""
    from fastforward_amd.cache import PagedCache
    pages = (1 << 32) // (8 * 4096 * 64) + 3
    c = PagedCache(pages, 4096, 8, 64, E4M3)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=I32, device=DEV)
    lengths, starts = torch.tensor([4100], dtype=I32, device=DEV), torch.tensor([0, 4100], dtype=I32, device=DEV)
    k, v = _rows(1, 4100, 8, 64).to(DEV), _rows(2, 4100, 8, 64).to(DEV)
    c.write(k, v, table, lengths, starts)
    small = PagedCache(2, 4096, 8, 64, E4M3)
    near = torch.tensor([[1, 0]], dtype=I32, device=DEV)
    small.write(k, v, near, lengths, starts)
    for x, want in zip(c.read(table, lengths, starts, 4100), small.read(near, lengths, starts, 4100)):
        assert torch.equal(x, want)
    q = _rows(3, 150, 8, 64).to(DEV)
    for n in (1, 150):
        s = torch.tensor([0, n], dtype=I32, device=DEV)
        assert torch.equal(c.attend(q[:n], table, lengths, s), small.attend(q[:n], near, lengths, s))


# ---------------------------------------------------------------- refusals (CPU)

def _bare():
    """A cache object without a GPU, for calls that are refused before any launch."""
    from fastforward_amd.cache import PagedCache
    c = PagedCache.__new__(PagedCache)
    c.pages, c.page_size, c.kv_heads, c.head_dim, c.dtype = 4, 16, 2, 64, BF16
    c._hold(*(torch.zeros(4, 2, 16, 64, dtype=BF16) for _ in range(2)), None, None)
    return c


def test_refusals():
    from fastforward_amd.cache import PagedCache
    for args in ((0, 16, 2, 64), (4, 24, 2, 64), (4, 8, 2, 64), (4, 8192, 2, 64), (4, 16, 0, 64), (4, 16, 2, 96),
                 (4, 16, 2, 64, torch.float32), (4, 16, 2, 64, BF16, "cpu")):
        with pytest.raises(AssertionError):
            PagedCache(*args)
    c = _bare()
    table, lengths, starts = torch.zeros(3, 2, dtype=I32), torch.ones(3, dtype=I32), torch.zeros(4, dtype=I32)
    rows, q = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(3, 4, 64, dtype=BF16)
    bad = [(table.long(), lengths, starts), (table[0], lengths, starts), (table[:, :0], lengths, starts),
           (table.T.contiguous().T, lengths, starts), (table, lengths[:2], starts), (table, lengths.long(), starts),
           (table, lengths, starts[:3]), (table, lengths, starts.long()), (table[:2], lengths[:2], None),
           (torch.zeros(3, 1 << 27, dtype=I32, device="meta"), lengths, starts),
           (torch.zeros(3, (1 << 27) - 4095, dtype=I32, device="meta"), lengths, starts),
           (table, lengths, starts)]                                  # the last: not on the GPU
    for args in bad:
        for call in (lambda *a: c.write(rows, rows, *a), lambda *a: c.attend(q, *a), lambda *a: c.read(*a, rows=3)):
            with pytest.raises(AssertionError):
                call(*args)
    for k, v in ((rows, rows[:2]), (rows.float(), rows.float()), (rows[:, :1], rows[:, :1]), (rows[..., :32], rows[..., :32]),
                 (q, q)):
        with pytest.raises(AssertionError):
            c.write(k, v, table, lengths, starts)
    for bad_q in (q.float(), q[0], q[..., :32], q[:, :3], q[:, :0]):
        with pytest.raises(AssertionError):
            c.attend(bad_q, table, lengths, starts)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(AssertionError):
            c.attend(q, table, lengths, starts, scale=scale)
    with pytest.raises(AssertionError, match="rows is missing"):
        c.read(table, lengths, starts)


def test_refusals_c():
    from fastforward_amd import _lib
    _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def cache(k=p, ks=None, pages=4, ps=16, hk=2, d=64, fp8=0):
        return ctypes.byref(_lib.PagedCacheStruct(k, p, ks, ks, pages, ps, hk, d, fp8))

    def attend(q=p, hq=4, width=2, lengths=p, starts=p, batch=3, t=3, scale=1.0, y=p, ws=p, nbytes=1 << 30, **kw):
        _lib.call("ff_attention_paged", q, 256, 64, cache(**kw), hq, p, width, lengths, starts, batch, y, t, scale, ws,
                  nbytes, None)

    def write(k_rows=p, width=2, lengths=p, starts=p, batch=3, t=3, **kw):
        _lib.call("ff_cache_write", k_rows, 128, 64, p, 128, 64, cache(**kw), p, width, lengths, starts, batch, t, None)

    def read(k_rows=p, width=2, lengths=p, starts=p, batch=3, t=3, **kw):
        _lib.call("ff_cache_read", cache(**kw), p, width, lengths, starts, batch, k_rows, p, t, None)

    shared = ((dict(d=96), "head_dim"), (dict(ps=24), "page_size"), (dict(ps=8), "page_size"), (dict(ps=8192), "page_size"),
              (dict(hk=0), "bad sizes"), (dict(width=0), "bad sizes"), (dict(width=1 << 27), "bad sizes"),
              (dict(width=(1 << 27) - 4095), "bad sizes"),
              (dict(batch=0), "bad sizes"), (dict(t=-1), "bad sizes"), (dict(t=1 << 25), "bad sizes"),
              (dict(pages=0), "bad sizes"), (dict(pages=1 << 31), "bad sizes"), (dict(k=None), "null"),
              (dict(lengths=None), "null"), (dict(fp8=1), "null"), (dict(starts=None, t=2), "starts"),
              (dict(k=p + 8), "alignment"), (dict(ks=p + 4, fp8=1), "alignment"))
    for f in (attend, write, read):
        for kw, message in shared:
            with pytest.raises(RuntimeError, match=message):
                f(**kw)
    for kw, message in ((dict(hq=3), "bad sizes"), (dict(hq=0), "bad sizes"), (dict(t=1 << 24, width=1 << 20), "too large"),
                        (dict(q=None), "null"), (dict(y=None), "null"), (dict(scale=0.0), "scale"),
                        (dict(scale=math.nan), "scale"), (dict(y=p + 2), "alignment"),
                        (dict(width=100, nbytes=64), "workspace"), (dict(width=100, ws=None), "workspace")):
        with pytest.raises(RuntimeError, match=message):
            attend(**kw)
    for f in (write, read):
        with pytest.raises(RuntimeError, match="null|output"):
            f(k_rows=None)
    attend(q=None, t=0)
    write(k_rows=None, t=0)
    read(k_rows=None, t=0)
    need = ctypes.c_int64(-1)
    _lib.call("ff_attention_paged_workspace", cache(hk=8, d=128, ps=64), 32, 2, 1, 0, 1, ctypes.byref(need))
    assert need.value == 0                              # 128 positions are never split
