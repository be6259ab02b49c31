"""Products right behind the quantisation of their weights: what they read is what it wrote, whichever way the rows came, whatever
product it is, and whatever the context quantises in between on another stream or into a graph.  (A call repeats its results bit
for bit, so each is held to itself, once everything has ended.  tests/test_mx4_order_of_launches.py looks at the same on the CPU.)"""
import pytest

from _util import torch_mod

pytestmark = pytest.mark.gpu
N, K = 14336, 2048


@pytest.fixture(scope="module")
def ctx():
    import aotx_b200
    made = aotx_b200.Q8Context(0)
    yield made
    assert made.device_status() == 0
    made.close()


@pytest.mark.parametrize("between", ["nothing", "stream", "graph", "context"])
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("call", ["matmul", "linear"])
@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_weights_quantised_just_before(ctx, m, call, listed, between):
    import aotx_b200
    torch = torch_mod()
    made = aotx_b200.Q8Context(0) if between == "context" else None
    by = made or ctx
    x = torch.randn((m, K), device="cuda").half()
    q, other = by.mx4_quantize(x), by.mx4_quantize(x)
    w = ctx.mx4_quantize(torch.zeros((N, K), device="cuda"))
    order = torch.randperm(N, device="cuda").to(torch.int32) if listed else None
    y = torch.empty((m, N), device="cuda")
    side = torch.cuda.Stream()
    multiply = (lambda: by.mx4_matmul(w, q, y=y)) if call == "matmul" else (lambda: by.mx4_linear(w, x, y=y))
    multiply()
    for turn in range(4):
        w16 = torch.randn((N, K), device="cuda").half()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        torch.cuda._sleep(200000)            # so that all of it is enqueued before the first of it runs
        ctx.mx4_quantize(w16, rows=order, out=w)
        if between == "stream":
            with torch.cuda.stream(side):
                ctx.mx4_quantize(x, out=other)
        elif between == "graph":
            with torch.cuda.stream(side):
                graph.capture_begin(capture_error_mode="relaxed")
                ctx.mx4_quantize(x, out=other)
                graph.capture_end()
        multiply()
        torch.cuda.synchronize()
        first = y.clone()
        y.zero_()
        torch.cuda.synchronize()
        multiply()
        torch.cuda.synchronize()
        assert torch.equal(first, y)
    if made is not None:
        assert made.device_status() == 0
        made.close()
