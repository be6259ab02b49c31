"""The routed step on MX4 weights as one call: every type of x and of the result, values that binary16 does not hold, into a graph."""
import numpy as np
import pytest

import _mx4
from _util import torch_mod
from test_gpu_y_mx4_product import dtype, order_of, random_codes, tensor

pytestmark = pytest.mark.gpu
SWIGLU = 2


@pytest.fixture(scope="module")
def ctx():
    import aotx_b200
    made = aotx_b200.Q8Context(0)
    yield made
    assert made.device_status() == 0
    made.close()


def constant(rows, k, code, power):
    """Every value is that of `code` times 2^power."""
    codes = np.full((rows, k // 2), code * 17, np.uint8)
    scales = np.zeros((rows, (k + 127) // 128 * 4), np.uint8)
    scales[:, :k // 32] = 127 + power
    return tensor(codes, np.ascontiguousarray(scales.reshape(rows, -1, 4).transpose(1, 0, 2)))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_an_activation_that_binary16_does_not_hold(ctx, kind):
    """All exact: gate and up are 64 * 4 * 4 = 2^10, silu(2^10) = 2^10, the activation 2^20 (above 65504), 32 of them by 2^-10 make
    2^15, half of that twice."""
    torch = torch_mod()
    experts, hidden, ffn, tokens = 4, 64, 32, 5
    x = torch.full((tokens, hidden), 4.0, device="cuda", dtype=dtype(kind))
    prob = torch.full((tokens, experts), 0.5, device="cuda")
    ids = torch.tensor([[0, 3], [1, 2], [2, 0], [3, 1], [0, 1]], dtype=torch.int32, device="cuda")
    out = ctx.mx4_moe_ffn(constant(experts * 2 * ffn, hidden, 6, 0), constant(experts * hidden, ffn, 2, -10), experts, x, prob, ids)
    assert (out == 2.0 ** 15).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,used,experts,hidden,ffn", [(1, 2, 8, 256, 160), (77, 4, 20, 544, 96)])
def test_every_type(ctx, tokens, used, experts, hidden, ffn, kind):
    """Each step held to the step before it, as in test_routed_step; results in 16 bits are the float ones, rounded once."""
    torch = torch_mod()
    w_gate_up, w_down = random_codes(experts * 2 * ffn, hidden, 1, -9, -5), random_codes(experts * hidden, ffn, 2, -9, -5)
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, hidden), generator=gen).to(dtype(kind)).cuda()
    prob = torch.rand((tokens, experts), generator=gen).cuda()
    ids = torch.topk(torch.randn((tokens, experts), generator=gen), used, dim=1)[1].to(torch.int32).cuda()
    up, down = tensor(*w_gate_up), tensor(*w_down)
    out = ctx.mx4_moe_ffn(up, down, experts, x, prob, ids)
    assert out.dtype == torch.float32
    for name in ("f16", "bf16"):
        assert torch.equal(ctx.mx4_moe_ffn(up, down, experts, x, prob, ids, out_dtype=dtype(name)), out.to(dtype(name)))
    ids_host = ids.cpu().numpy()
    order, edges = order_of(ids_host, experts, tokens)
    _, token_of, offsets = ctx.moe_order(ids, experts)
    act = ctx.mx4_matmul_grouped(up, experts, ctx.mx4_quantize(x, rows=token_of), offsets, y_dtype=x.dtype, epilogue=SWIGLU)
    act_host = act.double().cpu().numpy()
    x64 = _mx4.values(*_mx4.quantize(x.double().cpu().numpy()[order // used]))
    act64 = _mx4.values(*_mx4.quantize(act_host))
    up64, down64 = _mx4.values(*w_gate_up), _mx4.values(*w_down)
    proj64, proj_error = np.zeros((tokens * used, hidden)), np.zeros((tokens * used, hidden))
    for e in range(experts):
        a, b = edges[e], edges[e + 1]
        w64 = up64[e * 2 * ffn:(e + 1) * 2 * ffn]
        y64, error = x64[a:b] @ w64.T, _mx4.sum_bound(w64, x64[a:b])
        assert _mx4.close(act_host[a:b], _mx4.gated(y64), _mx4.gated_bound(y64, error, kind), kind).all()
        w64 = down64[e * hidden:(e + 1) * hidden]
        proj64[order[a:b]] = act64[a:b] @ w64.T
        proj_error[order[a:b]] = _mx4.sum_bound(w64, act64[a:b])
    chosen = np.take_along_axis(prob.double().cpu().numpy(), ids_host.astype(np.int64), axis=1)[:, :, None]
    want, parts, error = ((v.reshape(tokens, used, hidden) * chosen).sum(axis=1) for v in (proj64, np.abs(proj64), proj_error))
    # each rank: a rounded product and a rounded sum
    assert (np.abs(out.double().cpu().numpy() - want) <= error + parts * (2 * used) * 2.0 ** -24).all()


def test_captured(ctx):
    torch = torch_mod()
    tokens, used, experts, hidden, ffn = 8, 4, 16, 512, 256
    up, down = tensor(*random_codes(experts * 2 * ffn, hidden, 1, -9, -5)), tensor(*random_codes(experts * hidden, ffn, 2, -9, -5))
    x = torch.randn((tokens, hidden), device="cuda").bfloat16()
    prob = torch.rand((tokens, experts), device="cuda")
    ids = torch.zeros((tokens, used), dtype=torch.int32, device="cuda")
    live = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    out = torch.empty((tokens, hidden), device="cuda")
    call = lambda to: ctx.mx4_moe_ffn(up, down, experts, x, prob, ids, tokens_dev=live, out=to)
    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for turn in range(4):
        x.copy_(torch.randn((tokens, hidden), device="cuda"))
        ids.copy_(torch.topk(torch.randn((tokens, experts), device="cuda"), used, dim=1)[1])
        live.fill_(tokens - turn)
        out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        again = torch.full_like(out, -7.0)
        call(again)
        assert torch.equal(out, again) and (out[tokens - turn:] == -7.0).all()
