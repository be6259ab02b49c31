"""MX4 products: the gated unit far from zero, offsets that are out of order, a caller's own workspace, no overlap of launches."""
import numpy as np
import pytest

import _mx4
from _util import GUARD, torch_mod
from test_gpu_y_mx4_product import dtype, random_codes, tensor

pytestmark = pytest.mark.gpu
SWIGLU = 2


@pytest.fixture(scope="module")
def ctx():
    import aotx_b200
    made = aotx_b200.Q8Context(0)
    yield made
    assert made.device_status() == 0
    made.close()


def row_of(k, value):
    """Codes whose values add up to `value`, a multiple of a half."""
    left, codes = abs(value), []
    for code in range(7, 0, -1):
        while left >= _mx4.GRID[code]:
            left -= _mx4.GRID[code]
            codes.append(code + (8 if value < 0 else 0))
    return codes + [0] * (k - len(codes))


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_gated_unit_against_the_size_of_its_result(ctx, m, out):
    """Gates that float sums hold exactly, each beside a power of two that brings silu(gate) * up near one, so that the result is held to
    its own size and not to the gate's.  What the unit may lose, in halves of a unit (2^-24): float results 8 (expf, sum, quotient and
    product, two each); 16 bits 9 + 2 |gate| (_mx4.gated_bound), all of it relative to the result, because the sigmoid moves by no
    more, relatively, than the exponential does; where one plus the exponential passes 2^126 its reciprocal is a subnormal
    float, off by half of 2^-149.  Below -88.73 the exponential of a float is infinite and the result is a zero, as g / (1 + expf(-g))
    in floats is."""
    torch = torch_mod()
    k = 64
    gates = [20, 5, 1, 0.5, 0, -0.5, -1, -3, -8, -10.5, -14, -20, -40, -60, -80, -86, -87, -87.5, -88, -88.5, -89, -100, -150]
    codes, power = [], []
    for g in gates:
        silu = abs(g) / (1 + np.exp(-g))
        power += [0, int(np.clip(-np.floor(np.log2(silu)), 0, 126)) if silu > 0 else 3]
        codes += [row_of(k, g), row_of(k, 1.0)]
    codes = np.array(codes, np.uint8)
    scales = np.zeros((1, len(codes), 4), np.uint8)
    scales[0, :, :2] = 127 + np.array(power)[:, None]
    w = tensor(codes[:, 0::2] | codes[:, 1::2] << 4, scales)
    got = ctx.mx4_linear(w, torch.ones((m, k), device="cuda"), y_dtype=dtype(out), epilogue=SWIGLU).double().cpu().numpy()
    assert (got == got[:1]).all()
    for g, p, y in zip(gates, power[1::2], got[0]):
        want = g / (1 + np.exp(-float(g))) * 2.0 ** p
        steps = 8 if out == "f32" else 9 + 2 * abs(g)
        error = abs(want) * steps * 2.0 ** -24 + (2.0 ** -150 * abs(g) * 2.0 ** p if g < -87 else 0.0)
        if g < -88.73:
            assert y == 0
        else:
            assert abs(y - want) <= error + (abs(want) + error) * _mx4.half_step(out), (g, y, want)


@pytest.mark.parametrize("n,k,rows", [(64, 64, 50), (2404, 352, 1500)])
def test_offsets_out_of_order(ctx, n, k, rows):
    """Entries past the rows count as the rows, a range that runs backwards is empty, and what no expert has stays as it was."""
    torch = torch_mod()
    experts = 4
    w, x = random_codes(experts * n, k, 1, -2, 2), random_codes(rows, k, 2, -2, 2)
    w64, x64 = _mx4.values(*w).reshape(experts, n, k), _mx4.values(*x)
    dw, dx = tensor(*w), tensor(*x)
    part = rows // 5
    for offsets in ([0, part, part, rows + 10, rows + 20], [2 * part, part, 3 * part, 4 * part, rows],
                    [rows + 1, rows + 2, rows + 3, rows + 4, rows + 5], [-5, 2 * part, 2 * part, 3 * part, 2 ** 31 - 1],
                    [4 * part, 3 * part, 2 * part, part, 0], [part, part + 1, part + 1, part + 3, -1]):
        edges = [o if 0 <= o < rows else rows for o in offsets]
        want = np.full((rows, n), GUARD)
        for e in range(experts):
            a, b = edges[e], edges[e + 1]
            if b > a:
                assert (want[a:b] == GUARD).all()        # no row has two experts
                want[a:b] = x64[a:b] @ w64[e].T
        y = torch.full((rows, n), GUARD, device="cuda")
        ctx.mx4_matmul_grouped(dw, experts, dx, torch.tensor(offsets, dtype=torch.int32, device="cuda"), y=y)
        assert np.array_equal(y.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("n,k,m", [(300, 416, 33), (4096, 2080, 64), (20000, 1056, 300)])
def test_a_workspace_of_the_callers(ctx, n, k, m):
    """The same result, nothing written behind its end; one that is too small or off its boundary is refused."""
    import aotx_b200
    torch = torch_mod()
    w = tensor(*random_codes(n, k, n, -9, -3))
    x = torch.randn((m, k), device="cuda").half()
    want = ctx.mx4_linear(w, x)
    size = ctx.lib.aotx_mx4_linear_workspace_bytes(ctx._address, n, k, m)
    assert size >= m * k // 2 + m * 4
    work = torch.full((size + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert torch.equal(ctx.mx4_linear(w, x, workspace=work[:size]), want)
        assert (work[size:] == 0xA5).all()
    # one for more rows serves fewer, of another type
    few = x[:m // 2].bfloat16()
    assert torch.equal(ctx.mx4_linear(w, few, workspace=work), ctx.mx4_linear(w, few))
    for wrong in (work[:size - 1], work[8:]):
        with pytest.raises(aotx_b200.Q8Error) as refused:
            ctx.mx4_linear(w, x, workspace=wrong)
        assert refused.value.code == 5


def test_without_overlap(ctx):
    """One launch after the other: the same results."""
    import aotx_b200
    torch = torch_mod()
    alone = aotx_b200.Q8Context(0)
    alone.set_overlap(False)
    for n, k, m in ((520, 544, 3), (4096, 1056, 16), (20000, 1056, 300), (40000, 2080, 40)):
        w = tensor(*random_codes(n, k, n, -9, -3))
        x = torch.randn((m, k), device="cuda").half()
        results = []
        for by in (alone, ctx):
            q = by.mx4_quantize(x)
            results.append((by.mx4_matmul(w, q), by.mx4_linear(w, x), by.mx4_linear(w, x, y_dtype=torch.float16, epilogue=SWIGLU),
                            by.mx4_dequant(q)))
        torch.cuda.synchronize()
        for one, other in zip(*results):
            assert torch.equal(one, other)
    assert alone.device_status() == 0
    alone.close()
