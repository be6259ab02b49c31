"""MX4 quantisation and back against the format's definition in 64 bits (tests/_mx4.py): every code and scale is equal."""
import numpy as np
import pytest

import _mx4
from _util import torch_mod

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import aotx_b200
    made = aotx_b200.Q8Context(0)
    yield made
    assert made.device_status() == 0
    made.close()


def dtype(name):
    torch = torch_mod()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def inputs(rows, k, name, seed):
    """Rows with blocks of every kind: plain, zero, on the borders between codes, huge, tiny, subnormal, negative zeros."""
    torch = torch_mod()
    rng = np.random.Generator(np.random.PCG64(seed))
    x = rng.standard_normal((rows, k // 32, 32))
    kind = rng.integers(0, 8, (rows, k // 32))
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.5]) * 2.0 ** -3
    at_borders = rng.choice(borders, (rows, k // 32, 32)) * rng.choice([-1.0, 1.0], (rows, k // 32, 32))
    at_borders[:, :, 0] = 7.0 * 2.0 ** -3
    x = np.where((kind == 1)[:, :, None], 0.0, x)
    x = np.where((kind == 2)[:, :, None], at_borders, x)
    x = np.where((kind == 3)[:, :, None], x * 2.0 ** 12, x)
    x = np.where((kind == 4)[:, :, None], x * 2.0 ** -16, x)
    x = np.where((kind == 5)[:, :, None], -0.0, x)
    if name != "f16":
        x = np.where((kind == 6)[:, :, None], x * 2.0 ** -128, x)     # subnormal floats
        x = np.where((kind == 7)[:, :, None], x * 2.0 ** 124, x)
    return torch.from_numpy(x.reshape(rows, k)).clamp(-3e38, 3e38).to(dtype(name))


def check(got, x64):
    codes, scales = _mx4.quantize(x64)
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 96), (17, 160), (65, 1024), (130, 2016)])
def test_quantize_and_back(ctx, rows, k, name):
    torch = torch_mod()
    x = inputs(rows, k, name, rows * k)
    q = ctx.mx4_quantize(x.cuda())
    check(q, x.double().numpy())
    want = _mx4.values(*(t.cpu().numpy() for t in (q.codes, q.scales)))
    for out in ("f32", "f16", "bf16"):
        got = ctx.mx4_dequant(q, dtype=dtype(out)).cpu()
        # one rounding of the float that the two stand for (two significant bits: a float holds it, or its half below 2^-127)
        assert torch.equal(got, torch.from_numpy(want).to(torch.float32).to(dtype(out)))
    if rows > 2:
        part = ctx.mx4_dequant(q, first_row=1, rows=rows - 2, dtype=torch.float32).cpu()
        assert torch.equal(part, torch.from_numpy(want[1:-1]).to(torch.float32))


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_not_a_number_and_infinity_take_their_block(ctx, name):
    torch = torch_mod()
    x = inputs(4, 256, name, 5)
    x[0, 3] = float("nan")
    x[1, 40] = float("inf")
    x[2, 200] = -float("inf")
    q = ctx.mx4_quantize(x.cuda())
    check(q, x.double().numpy())
    back = ctx.mx4_dequant(q, dtype=torch.float32).cpu()
    assert torch.isnan(back[0, :32]).all() and torch.isnan(back[1, 32:64]).all() and torch.isnan(back[2, 192:224]).all()
    assert int(torch.isnan(back).sum()) == 96


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("skip,extra", [(0, 24), (1, 3), (8, 8)])
def test_rows_that_lie_apart_and_off_a_boundary(ctx, name, skip, extra):
    torch = torch_mod()
    rows, k = 9, 320
    wide = torch.full((rows, skip + k + extra), float("nan"), dtype=dtype(name))
    wide[:, skip:skip + k] = inputs(rows, k, name, 7)
    view = wide.cuda()[:, skip:skip + k]
    check(ctx.mx4_quantize(view), wide[:, skip:skip + k].double().numpy())


def test_chosen_rows_and_a_live_number(ctx):
    import aotx_b200
    torch = torch_mod()
    x = inputs(6, 288, "f16", 9)
    chosen = [5, 0, 0, 6, 3, -1, 2, 2 ** 31 - 1]
    out = aotx_b200.Mx4Tensor.empty(len(chosen), 288, "cuda")
    for live in (None, 0, 3, 7, 100):
        out.codes.fill_(0xA5)
        out.scales.fill_(0x5A)
        word = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
        ctx.mx4_quantize(x.cuda(), rows=torch.tensor(chosen, dtype=torch.int32, device="cuda"), rows_dev=word, out=out)
        codes, scales = out.codes.cpu().numpy(), out.scales.cpu().numpy()
        for i, row in enumerate(chosen):
            if (live is None or i < live) and 0 <= row < 6:
                want = _mx4.quantize(x[row:row + 1].double().numpy())
                assert np.array_equal(codes[i:i + 1], want[0]) and np.array_equal(scales[:, i:i + 1], want[1])
            else:
                assert (codes[i] == 0xA5).all() and (scales[:, i] == 0x5A).all()


def test_no_rows(ctx):
    torch = torch_mod()
    q = ctx.mx4_quantize(torch.empty((0, 64), device="cuda"))
    assert q.rows == 0 and ctx.mx4_dequant(q).shape == (0, 64)
    some = ctx.mx4_quantize(torch.ones((2, 64), device="cuda"), rows=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert some.rows == 0
