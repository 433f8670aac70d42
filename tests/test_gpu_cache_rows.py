"""Rows of the paged attention that are not ordinary: NaN and infinities in queries and in the keys
that a row sees, in calls that are split and calls that are not."""
import math

import pytest
import torch

from oracle import serving as S
from tests.test_gpu_cache import BF16, DEV, E4M3, Case, _rows, close, tile  # noqa: F401 (a fixture)

gpu_test = pytest.mark.gpu


@gpu_test
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("lengths,new,heads,width", [
    ([90], None, 4, None), ([1500], None, 4, None), ([90], None, 4, 300), ([1500], [40], 4, None),
    ([700, 1300], [300, 5], 8, 200), ([100] * 70, [2] * 70, 4, None)])
def test_odd_queries(gpu, tile, dtype, lengths, new, heads, width):  # noqa: F811
    """A NaN in a query makes its row NaN, and so do scores that are all -inf; rows that see nothing
    are zero, and the others are as they were. Rows joined by workgroups and by groups of lanes."""
    for d in (64, 128):
        c = Case(lengths, new, 2, d, 16, dtype, seed=d, width=width)
        c.cpu["k"][..., 5] = -1.0 if dtype == BF16 else torch.tensor(-1.0).to(E4M3)
        c.upload("k")
        if len(lengths) > 1:
            c.lengths[-1] = 1                             # the rows of its sequence before the last see nothing
        q = _rows(d, c.t, heads, d)
        q[0, 0, 7] = math.nan
        q[c.t // 2, heads - 1, 5] = math.inf              # -inf for every key
        q[c.t // 3, 1, 5] = math.inf
        y, o = c.check_attend(q)
        assert y[0, 0].isnan().all() and y[c.t // 3, 1].isnan().all()
        if lengths == [1500] and new is None:             # without any key
            c.lengths[0] = 0
            assert not c.dev.attend(q.to(DEV), *c.args()).any()


@gpu_test
@pytest.mark.parametrize("new", [None, [9], [200]])
def test_odd_ranges_of_keys(gpu, tile, new):  # noqa: F811
    """Long runs of keys that score -inf weigh nothing beside others; one NaN key that is seen is NaN,
    wherever it lies and whatever the others are."""
    for at in (0, 1000, 2499):
        c = Case([2500], new, 1, 128, 16, BF16, seed=at)
        keys = torch.arange(2500)
        page, slot = c.table[0].long()[keys // 16], keys % 16
        far = (keys - at).abs() > 40                       # all but a few score -inf
        c.cpu["k"][page[far], 0, slot[far], 3] = -math.inf
        c.upload("k")
        q = _rows(1, c.t, 4, 128).abs()
        y, o = c.check_attend(q)
        assert not o[-1].isnan().any()
        c.cpu["k"][page[at], 0, slot[at], 9] = math.nan
        c.upload("k")
        y = c.dev.attend(q.to(DEV), *c.args()).cpu()
        o, _, _ = S.attend(c.cpu, q, c.table, c.lengths, c.starts)
        assert torch.equal(y.isnan(), o.isnan()) and y[-1].isnan().all()


@gpu_test
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (E4M3, 128), (E4M3, 64)])
@pytest.mark.parametrize("length,n", [(128, 1), (128, 30), (2000, 3), (2000, 200)])
def test_large_values(gpu, tile, dtype, d, length, n):  # noqa: F811
    """Values whose size times the positions' number is below 2^127 never overflow: the first block's
    scores are 2^7.9 times below the others', the most that a reference may lag behind."""
    c = Case([length], [n], 1, d, 64, dtype, seed=length + d)
    for name in ("k", "v"):
        x = S.values(c.cpu, name)
        if name == "k":
            x[..., 0] = 1.0
            page = int(c.table[0, 0])
            x[page, :, :, 0] = 0.0
            x[..., 1:] *= 2.0 ** -10
        else:
            x = (x.sign() + (x == 0)) * 2.0 ** (119 if length == 128 else 115)
        x = x.to(BF16)
        if dtype == BF16:
            c.cpu[name] = x
        else:
            c.cpu[name], c.cpu[name + "_scale"] = S.codes(x)
        c.upload(name)
    q = _rows(2, n, 4, d) * 2.0 ** -10
    q[..., 0] = 7.875                                     # in base 2, by the scale
    y, o = c.check_attend(q.to(BF16), scale=math.log(2.0))
    assert (o.abs() < math.inf).all() and y.isfinite().all()


@gpu_test
def test_every_scale_byte(gpu):
    """read gives code * 2^(byte - 127) of all codes under all bytes, rounded to bf16 where that has fewer
    bits (below its normal range) or no such value; NaN under byte 255."""
    c = Case([4096], None, 1, 128, 16, E4M3, fill=False, spare=0)
    c.table[0] = torch.arange(256)
    byte = torch.arange(256, dtype=torch.uint8)
    c.cpu["k"] = byte.reshape(1, 1, 2, 128).repeat(256, 1, 8, 1).view(E4M3)
    c.cpu["v"] = c.cpu["k"].flip(2)
    for name in ("k", "v"):
        c.cpu[name + "_scale"] = byte[:, None, None].expand(256, 1, 16).contiguous()
        c.upload(name)
    starts = torch.tensor([0, 4096], dtype=torch.int32)
    got = c.dev.read(*c.args(False), starts.to(DEV), rows=4096)
    for x, want in zip(got, S.read(c.cpu, c.table, c.lengths, starts, 4096)):
        want[255 * 16:] = math.nan
        want = want.float().to(BF16)                       # exact in fp32: 2^-136 is a multiple of its smallest value
        assert torch.equal(x.cpu().isnan(), want.isnan()) and torch.equal(x.cpu().nan_to_num(0), want.nan_to_num(0))


@gpu_test
@pytest.mark.parametrize("n,length", [(20, 100), (3, 700), (150, 400)])
def test_scale_bytes(gpu, tile, n, length):  # noqa: F811
    """A row does not depend on the scale bytes of keys that it does not see, whatever they are; bytes that write
    never makes are read as they are."""
    for d in (64, 128):
        c = Case([length], [n], 1, d, 64, E4M3, seed=d)
        page, slot = int(c.table[0, (length - 1) // 64]), (length - 1) % 64
        q = _rows(3, n, 3, d)
        want = c.dev.attend(q.to(DEV), *c.args())
        for byte in (0, 1, 26, 248, 254, 255):
            c.dev.k_scale[page, 0, slot], c.dev.v_scale[page, 0, slot] = byte, byte
            assert torch.equal(c.dev.attend(q.to(DEV), *c.args())[:-1], want[:-1]), byte
        small = S.codes((torch.rand(c.cpu["v"].shape, generator=torch.Generator().manual_seed(1)) * 448).to(BF16))[0]
        small = (small.float() / 448).to(E4M3)
        for k_byte, v_byte in ((1, 1), (26, 26), (120, 248 - 5), (133, 90)):
            for name, x, byte in (("k", c.cpu["k"], k_byte), ("v", small, v_byte)):
                c.cpu[name], c.cpu[name + "_scale"] = x, torch.full_like(c.cpu[name + "_scale"], byte)
                c.upload(name)
            c.check_attend(q)
        c.cpu["k_scale"].fill_(120)
        c.cpu["v_scale"].fill_(254)                        # values up to 2^127, one position
        c.upload("k"), c.upload("v")
        c.starts = torch.tensor([0, 1], dtype=torch.int32)
        c.lengths[0], c.t = 1, 1
        c.check_attend(q[:1])


@gpu_test
def test_tile_choice_between_calls(gpu):
    """A tile choice that is set between two calls of the same sizes."""
    from fastforward_amd import _lib
    c = Case([600], [200], 2, 128, 64)
    q = _rows(1, 200, 8, 128)
    try:
        for choice in (0, 1, 2, 3, 1, 0):
            _lib.call("ff_set_tuning", 14, choice)
            c.check_attend(q)
    finally:
        _lib.call("ff_set_tuning", 14, 0)


def _part(c, q, y, sequences):
    """Compares the rows of some sequences with the oracle's."""
    starts = list(range(len(c.lengths) + 1)) if c.starts is None else c.starts.tolist()
    rows = [i for b in sequences for i in range(starts[b], starts[b + 1])]
    upto = torch.tensor([0] + [starts[b + 1] - starts[b] for b in sequences]).cumsum(0).to(torch.int32)
    o, a, most = S.attend(c.cpu, q[rows], c.table[sequences], c.lengths[sequences], upto)
    close(y[rows], o, a, most, c.d)


@gpu_test
@pytest.mark.parametrize("batch,hk,dtype", [(1023, 8, BF16), (1024, 8, E4M3), (1025, 8, BF16), (2100, 8, BF16), (4200, 2, E4M3)])
@pytest.mark.parametrize("ragged", [False, True])
def test_thousands_of_sequences(gpu, batch, hk, dtype, ragged):
    """The work list past one, two and four times its workgroup's threads; some sequences without rows or
    keys, two past 4096 positions."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 31, (batch,), generator=gen)
    lengths[1022], lengths[batch - 2] = 5000, 4100
    new = torch.randint(0, 4, (batch,), generator=gen).minimum(lengths).tolist() if ragged else None
    c = Case(lengths.tolist(), new, hk, 64, 16, dtype, seed=batch)
    k, v, q = _rows(1, c.t, hk, 64), _rows(2, c.t, hk, 64), _rows(3, c.t, 2 * hk, 64)
    c.dev.write(k.to(DEV), v.to(DEV), *c.args())
    S.write(c.cpu, k, v, c.table, c.lengths, c.starts)
    for name, want in c.cpu.items():
        assert torch.equal(getattr(c.dev, name).cpu().view(torch.uint8), want.view(torch.uint8)), name
    y = c.dev.attend(q.to(DEV), *c.args()).cpu()
    near = {0, 1, 63, 64, 511, 512, 1020, 1021, 1022, batch - 3, batch - 2, batch - 1}
    near |= set(range(1000, min(batch, 1060))) | set(range(2040, min(batch, 2056))) | set(range(4090, min(batch, 4102)))
    _part(c, q, y, sorted(near | set(range(0, batch, 37))))
    if not ragged:                                        # the same rows by starts
        c.starts = torch.arange(batch + 1, dtype=torch.int32)
        _part(c, q, c.dev.attend(q.to(DEV), *c.args()).cpu(), sorted(near))
