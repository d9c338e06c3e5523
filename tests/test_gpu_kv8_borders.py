"""Keys of an 8-bit cache that lie on the border of two codes: rows of one magnitude come out of the norm as plus or minus the weights, exactly, and go to the code whose last bit is zero."""
import pytest

from test_gpu_kv import _i32, _rotated, _starts, _table, _type
from test_gpu_kv8 import Cache8, _kept, _same
from test_gpu_parity import bam  # noqa: F401  (the module fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,page", [(128, 4096), (64, 4096), (256, 4096), (80, 4096), (112, 4096), (208, 8192)])
@pytest.mark.parametrize("rot,style", [(0, "half"), (32, "half"), (32, "pairs")])
def test_rows_of_one_magnitude(bam, dtype, dim, page, rot, style):
    """x = +-c in every place: mean x^2 is c^2, so x / sqrt(mean x^2) * w is +-w.  Weights of 1.0625, 1.1875, ..: five significant bits, half-way between numbers of four.  Turned by nothing, and by a half turn"""
    import torch
    gen = torch.Generator().manual_seed(3)
    n, dt = 256, _type(dtype)
    c = torch.arange(129, 129 + n).float().remainder(128).add(128).ldexp(torch.randint(-9, 2, (n,), generator=gen).float())[:, None, None]      # eight significant bits, both types have them
    x = (c * (torch.randint(0, 2, (n, 1, dim), generator=gen) * 2 - 1)).to(dt)
    assert torch.equal(x.float().abs(), c.expand(-1, -1, dim))
    w = ((17 + 2 * torch.randint(0, 8, (dim,), generator=gen)).float() / 16).to(dt)
    turn = 1.0 - 2.0 * torch.randint(0, 2, (n, rot // 2), generator=gen)
    with Cache8(bam, 2 + n // 16, 1, dim, dtype, page) as k:
        table = _table([n], k.t, k.n_blocks).cuda()
        at = (_i32([n]), table)
        k.kv.append(x.cuda(), x.cuda(), *at, starts=_starts([n]), k_norm=w.cuda(), eps=0.0, cos=turn.cuda() if rot else None, sin=torch.zeros_like(turn).cuda() if rot else None, rotary=style)
        got, _ = k.kv.read(n, *at, starts=_starts([n]))
        want = x.double().sign() * w.double()
        if rot:
            turns = torch.cat([turn, turn], 1) if style == "half" else turn.repeat_interleave(2, 1)
            want[:, 0, :rot] *= turns
        _same(got, _kept(want, dtype))
        assert not k.rig.c.aborted()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [128, 80])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -20])
def test_norms_of_what_is_not_finite_and_of_nothing(bam, dtype, dim, eps):
    """an infinity makes the others zero and itself NaN, NaN makes all NaN, rows of zeros are NaN without eps; the largest and the smallest numbers of the type"""
    import torch
    gen = torch.Generator().manual_seed(4)
    dt = _type(dtype)
    x = torch.randn(12, 1, dim, generator=gen).to(dt)
    x[0, 0, 7], x[1, 0, 0], x[2, 0, dim - 1], x[3] = float("inf"), float("-inf"), float("nan"), 0
    x[4, 0, 3] = x[4, 0, 9] = float("inf")
    x[5] = x[5].sign() * torch.finfo(dt).max
    x[6] = x[6].sign() * torch.finfo(dt).smallest_normal
    w = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dt)
    with Cache8(bam, 4, 1, dim, dtype) as k:
        table = _table([12], k.t, 4).cuda()
        at = (_i32([12]), table)
        k.kv.append(x.cuda(), x.cuda(), *at, starts=_starts([12]), k_norm=w.cuda(), eps=eps)
        got, _ = k.kv.read(12, *at, starts=_starts([12]))
        want = torch.stack([_rotated(x[i, 0], w, i, None, None, "half", eps)[0] for i in range(12)])
        _same(got[:, 0], _kept(want, dtype))


@pytest.mark.parametrize("dim,page", [(128, 4096), (256, 4096), (80, 4096), (16, 512)])
@pytest.mark.parametrize("dtype,top", [("bf16", 2.0 ** 127), ("bf16", 2.0 ** -112), ("f16", 2.0 ** 15), ("f16", 2.0 ** -14)])
@pytest.mark.parametrize("rot", [0, 16])
def test_weights_at_the_ends_of_the_range(bam, dtype, top, dim, page, rot):
    """normed keys past the type's largest number are kept as the largest that is, and weights near its ends do not lose or overflow on the way: rows of one magnitude, and with a few large numbers"""
    import torch
    gen = torch.Generator().manual_seed(dim)
    n, dt = 64, _type(dtype)
    x = torch.randn(n, 1, dim, generator=gen).sign()
    x[16:32] *= torch.exp2(torch.randint(-3, 4, (16, 1, dim), generator=gen).float())
    x[32:48] = torch.randn(16, 1, dim, generator=gen)
    x[48:, :, 1:] = 0                               # sqrt(dim) times the mean size, and nothing
    x = x.to(dt)
    w = ((1 + torch.randint(0, 127, (dim,), generator=gen) / 128) * top).to(dt)
    angle = torch.rand(n, rot // 2, generator=gen) * 6.28
    with Cache8(bam, 2 + n // 16, 1, dim, dtype, page) as k:
        table = _table([n], k.t, k.n_blocks).cuda()
        at = (_i32([n]), table)
        k.kv.append(x.cuda(), x.cuda(), *at, starts=_starts([n]), k_norm=w.cuda(), eps=0.0, cos=angle.cos().cuda() if rot else None, sin=angle.sin().cuda() if rot else None)
        got, _ = k.kv.read(n, *at, starts=_starts([n]))
        cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
        want = torch.stack([_rotated(x[i, 0], w, i, cos, sin, "half", 0.0)[0] for i in range(n)])
        assert bool(torch.isfinite(want).all())
        _same(got[:, 0], _kept(want, dtype))
