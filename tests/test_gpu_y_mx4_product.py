"""Products of MX4 tensors against the sums in 64 bits (tests/_mx4.py), plain and grouped by expert."""
import numpy as np
import pytest

import _mx4
from _util import GUARD, torch_mod

pytestmark = pytest.mark.gpu
STORE, ADD, SWIGLU = 0, 1, 2


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


def tensor(codes, scales):
    import aotx_b200
    torch = torch_mod()
    return aotx_b200.Mx4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())


def random_codes(rows, k, seed, low, high):
    """Codes of every kind and scales 2^low .. 2^high."""
    rng = np.random.Generator(np.random.PCG64(seed))
    codes = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8)
    chunks = (k + 127) // 128
    flat = np.zeros((rows, chunks * 4), np.uint8)
    flat[:, :k // 32] = rng.integers(127 + low, 128 + high, (rows, k // 32))
    return codes, np.ascontiguousarray(flat.reshape(rows, chunks, 4).transpose(1, 0, 2))


# one block; one tile; tiles cut by every edge; a depth that ends inside a stage, inside a word of scales; clusters of every size;
# tiles cut between blocks
SHAPES = [(128, 64, 16), (16, 32, 1), (1, 32, 3), (130, 96, 5), (127, 256, 17), (300, 416, 33), (129, 1056, 100), (512, 512, 128),
          (260, 320, 129), (257, 288, 200), (200, 1024, 256), (140, 192, 257), (388, 544, 513), (64, 4096, 2), (2000, 2560, 300),
          (4100, 1312, 40), (2050, 1024, 20), (6144, 1024, 100), (4096, 2080, 256), (1030, 8192, 3), (8192, 512, 130),
          (9000, 608, 16), (40000, 800, 9), (40000, 288, 60), (30000, 1056, 128)]
# pairs of blocks: whole tiles, cut ones, edges of either operand
PAIRS = [(9472, 256, 258), (9500, 96, 290), (10001, 544, 300), (9472, 1312, 448), (4800, 800, 1000), (20000, 2080, 260)]


@pytest.mark.parametrize("n,k,m", PAIRS + SHAPES)
def test_exact_sums(ctx, n, k, m):
    """Scales 2^-2 .. 2^2: products are multiples of 2^-6, and where the magnitudes of a sum add up to less than 2^18 floats hold
    every partial sum: the result is the sum itself."""
    w, x = random_codes(n, k, n + k, -2, 2), random_codes(m, k, m + k + 1, -2, 2)
    want = _mx4.values(*x) @ _mx4.values(*w).T
    assert (np.abs(_mx4.values(*x)) @ np.abs(_mx4.values(*w)).T).max() < 2.0 ** 18
    torch = torch_mod()
    y = torch.full((m + 1, n), GUARD, device="cuda")
    got = ctx.mx4_matmul(tensor(*w), tensor(*x), y=y[:m]).cpu().numpy()
    assert np.array_equal(got, want.astype(np.float32))
    assert (y[m:] == GUARD).all()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(130, 96, 5), (300, 416, 33), (388, 544, 140), (256, 1024, 300), (1000, 512, 8),
                                   (9600, 352, 290)])
def test_types_and_epilogues(ctx, n, k, m, out):
    torch = torch_mod()
    w, x = random_codes(n, k, n, -9, -3), random_codes(m, k, m, -4, 3)
    w64, x64 = _mx4.values(*w), _mx4.values(*x)
    want, error = x64 @ w64.T, _mx4.sum_bound(w64, x64)
    dw, dx = tensor(*w), tensor(*x)
    got = ctx.mx4_matmul(dw, dx, y_dtype=dtype(out)).double().cpu().numpy()
    assert _mx4.close(got, want, error, out).all()
    got = ctx.mx4_matmul(dw, dx, y_dtype=dtype(out), epilogue=SWIGLU).double().cpu().numpy()
    assert got.shape == (m, n // 2)
    assert _mx4.close(got, _mx4.gated(want), _mx4.gated_bound(want, error, out), out).all()
    if out == "f32":
        before = torch.randn((m, n), device="cuda")
        y = before.clone()
        ctx.mx4_matmul(dw, dx, y=y, epilogue=ADD)
        plain = ctx.mx4_matmul(dw, dx)
        assert torch.equal(y, before + plain)


@pytest.mark.parametrize("n", [200, 9600])
@pytest.mark.parametrize("m,live", [(1, 0), (1, 1), (40, 17), (40, 99), (300, 0), (300, 5), (300, 256), (300, 290)])
def test_live_batch(ctx, n, m, live):
    torch = torch_mod()
    k = 320
    w, x = random_codes(n, k, 1, -2, 2), random_codes(m, k, 2, -2, 2)
    want = _mx4.values(*x) @ _mx4.values(*w).T
    y = torch.full((m, n), GUARD, device="cuda")
    word = torch.tensor([live], dtype=torch.int32, device="cuda")
    ctx.mx4_matmul(tensor(*w), tensor(*x), y=y, m_dev=word)
    got = y.cpu().numpy()
    rows = min(live, m)
    assert np.array_equal(got[:rows], want[:rows].astype(np.float32)) and (got[rows:] == GUARD).all()


def test_y_off_a_boundary_and_scale_nan(ctx):
    torch = torch_mod()
    n, k, m = 66, 128, 9
    w, x = random_codes(n, k, 1, -2, 2), random_codes(m, k, 2, -2, 2)
    x[1][0, 3, 2] = 255      # a block of row 3 is not a number, and with it the row
    want = _mx4.values(*x) @ _mx4.values(*w).T
    flat = torch.full((m * n + 3,), GUARD, device="cuda")
    for name in ("f32", "f16", "bf16"):
        flat = torch.full((m * n + 3,), GUARD, device="cuda", dtype=dtype(name))
        y = flat[1:1 + m * n].view(m, n)
        ctx.mx4_matmul(tensor(*w), tensor(*x), y=y)
        got = y.double().cpu().numpy()
        rows = np.arange(m) != 3
        assert np.isnan(got[3]).all()
        assert _mx4.close(got[rows], want[rows], 0.0, name).all()
        assert flat[0] == flat[m * n + 1] == flat[m * n + 2] == torch.tensor(GUARD, dtype=flat.dtype)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(130, 96, 1), (300, 416, 5), (200, 2080, 16), (4096, 512, 8), (140, 1056, 17), (200, 96, 33),
                                   (260, 320, 100), (130, 64, 300), (4000, 4128, 2), (19000, 1056, 3), (40000, 2080, 4),
                                   (40000, 288, 16), (20000, 1056, 3), (1000, 288, 16)])
def test_linear_is_quantisation_and_product(ctx, n, k, m, kind):
    """Against the sums of what mx4_quantize makes of the same rows."""
    torch = torch_mod()
    codes = random_codes(n, k, n, -9, -3)
    w, w64 = tensor(*codes), _mx4.values(*codes)
    gen = torch.Generator().manual_seed(m)
    x = torch.randn((m, k + 8), generator=gen)
    x[m // 2, :32] = 0
    x = x.to(dtype(kind)).cuda()
    for view in (x[:, :k].contiguous(), x[:, 8:], x[:, 1:k + 1]):
        q = ctx.mx4_quantize(view)
        x64 = _mx4.values(q.codes.cpu().numpy(), q.scales.cpu().numpy())
        want, error = x64 @ w64.T, _mx4.sum_bound(w64, x64)
        assert _mx4.close(ctx.mx4_linear(w, view).double().cpu().numpy(), want, error, "f32").all()
        for out in ("f16", "bf16"):
            got = ctx.mx4_linear(w, view, y_dtype=dtype(out), epilogue=SWIGLU).double().cpu().numpy()
            assert _mx4.close(got, _mx4.gated(want), _mx4.gated_bound(want, error, out), out).all()
        y = torch.ones((m, n), device="cuda")
        ctx.mx4_linear(w, view, y=y, epilogue=ADD)
        assert _mx4.close(y.double().cpu().numpy(), 1 + want, error + np.abs(want) * 2.0 ** -24, "f32").all()
        live = torch.tensor([m // 2], dtype=torch.int32, device="cuda")
        y = torch.full((m, n), GUARD, device="cuda")
        ctx.mx4_linear(w, view, y=y, m_dev=live)
        assert _mx4.close(y[:m // 2].double().cpu().numpy(), want[:m // 2], error[:m // 2], "f32").all()
        assert (y[m // 2:] == GUARD).all()


def test_linear_takes_not_a_number_into_its_row_only(ctx):
    torch = torch_mod()
    w = tensor(*random_codes(256, 512, 3, -9, -3))
    for m in (4, 40):
        x = torch.randn((m, 512), device="cuda").half()
        clean = ctx.mx4_linear(w, x)
        x[1, 100] = float("inf")
        y = ctx.mx4_linear(w, x)
        assert torch.isnan(y[1]).all()
        rows = torch.arange(m, device="cuda") != 1
        assert torch.equal(y[rows], clean[rows])


def order_of(ids, experts, live):
    flat = ids[:live].reshape(-1)
    lists = [np.nonzero(flat == e)[0] for e in range(experts)]
    return np.concatenate(lists), np.cumsum([0] + [len(part) for part in lists])


@pytest.mark.parametrize("tokens,used,experts", [(1, 1, 1), (1, 8, 128), (8, 8, 128), (7, 3, 5), (77, 4, 20), (512, 8, 128),
                                                 (300, 2, 256), (2048, 8, 64), (33, 1, 3), (5000, 7, 200)])
def test_order(ctx, tokens, used, experts):
    torch = torch_mod()
    rng = np.random.Generator(np.random.PCG64(tokens))
    ids = np.argsort(rng.standard_normal((tokens, experts)) + rng.standard_normal(experts), axis=1)[:, :used].astype(np.int32)
    strange = ids.copy()
    strange[rng.random(ids.shape) < 0.2] = -1
    strange[rng.random(ids.shape) < 0.1] = experts
    one = np.zeros_like(ids)
    for chosen in (ids, strange, one, np.full_like(ids, -1)):
        for live in (None, 0, tokens // 2, tokens, tokens + 9):
            word = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
            got = [t.cpu().numpy() for t in ctx.moe_order(torch.from_numpy(chosen).cuda(), experts, tokens_dev=word)]
            want, offsets = order_of(chosen, experts, tokens if live is None else min(live, tokens))
            assert np.array_equal(got[2], offsets)
            assert np.array_equal(got[0][:len(want)], want) and (got[0][len(want):] == -1).all()
            assert np.array_equal(got[1][:len(want)], want // used) and (got[1][len(want):] == -1).all()


@pytest.mark.parametrize("counts", [[5], [0, 3, 0, 0, 129, 1, 0], [0] * 7, [16] * 20, [0] * 255 + [40], [1] * 256, [600, 0, 2],
                                    [300, 20, 257, 31]])
@pytest.mark.parametrize("n,k", [(96, 160), (260, 512)])
def test_grouped(ctx, counts, n, k):
    grouped(ctx, counts, n, k)


@pytest.mark.parametrize("counts", [[300] * 8, [0, 1100, 1, 133, 0, 700, 165, 1]])
def test_grouped_by_pairs_of_blocks(ctx, counts):
    grouped(ctx, counts, 2404, 352)


def grouped(ctx, counts, n, k):
    """Every expert's rows by its own matrix; rows behind the last expert's stay as they are."""
    torch = torch_mod()
    experts, spare = len(counts), 3
    rows = sum(counts) + spare
    edges = np.cumsum([0] + counts)
    w, x = random_codes(experts * n, k, n, -2, 2), random_codes(rows, k, rows, -2, 2)
    w64, x64 = _mx4.values(*w), _mx4.values(*x)
    want = np.full((rows, n), GUARD)
    for e in range(experts):
        want[edges[e]:edges[e + 1]] = x64[edges[e]:edges[e + 1]] @ w64[e * n:e * n + n].T
    offsets = torch.from_numpy(edges.astype(np.int32)).cuda()
    dw, dx = tensor(*w), tensor(*x)
    y = torch.full((rows, n), GUARD, device="cuda")
    ctx.mx4_matmul_grouped(dw, experts, dx, offsets, y=y)
    assert np.array_equal(y.cpu().numpy(), want.astype(np.float32))
    # rows to places of their own, some outside y
    rng = np.random.Generator(np.random.PCG64(3))
    places = rng.permutation(rows + 4)[:rows].astype(np.int32)
    places[rng.random(rows) < 0.1] = -1
    scattered = np.full((rows, n), GUARD)
    for i in range(edges[-1]):
        if 0 <= places[i] < rows:
            scattered[places[i]] = want[i]
    y = torch.full((rows, n), GUARD, device="cuda")
    ctx.mx4_matmul_grouped(dw, experts, dx, offsets, y_rows=torch.from_numpy(places).cuda(), y=y)
    assert np.array_equal(y.cpu().numpy(), scattered.astype(np.float32))
    for out in ("f16", "bf16"):
        act = torch.full((rows, n // 2), GUARD, device="cuda", dtype=dtype(out))
        ctx.mx4_matmul_grouped(dw, experts, dx, offsets, y=act, epilogue=SWIGLU)
        got = act.double().cpu().numpy()
        assert (act[edges[-1]:] == torch.tensor(GUARD, dtype=act.dtype)).all()
        if edges[-1]:
            placed = want[:edges[-1]]
            bound = _mx4.gated_bound(placed, np.zeros_like(placed), out)
            assert _mx4.close(got[:edges[-1]], _mx4.gated(placed), bound, out).all()


def test_offsets_that_make_no_sense_reach_nothing_outside(ctx):
    torch = torch_mod()
    experts, n, k, rows = 4, 64, 64, 50
    w, x = tensor(*random_codes(experts * n, k, 1, -2, 2)), tensor(*random_codes(rows, k, 2, -2, 2))
    guard = torch.full((rows + 2, n), GUARD, device="cuda")
    for offsets in ([0, 10, 5, 60, 70], [-5, 20, 20, 30, 2 ** 31 - 1], [50, 40, 30, 20, 10], [60, 61, 62, 63, 64]):
        ctx.mx4_matmul_grouped(w, experts, x, torch.tensor(offsets, dtype=torch.int32, device="cuda"), y=guard[1:-1])
        torch.cuda.synchronize()
        assert (guard[0] == GUARD).all() and (guard[-1] == GUARD).all()


@pytest.mark.parametrize("tokens,used,experts,hidden,ffn", [(1, 2, 8, 256, 160), (8, 8, 128, 512, 256), (77, 4, 20, 544, 96),
                                                            (300, 2, 4, 256, 256)])
def test_routed_step(ctx, tokens, used, experts, hidden, ffn):
    """The calls of a routed layer as they are used together.  The activations between the two products are rounded to four bits, so
    the second product is held to what the first one gave: each step is checked on the step before it."""
    torch = torch_mod()
    w_gate_up = random_codes(experts * 2 * ffn, hidden, 1, -9, -5)
    w_down = random_codes(experts * hidden, ffn, 2, -9, -5)
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, hidden), generator=gen).half().cuda()
    router = torch.randn((experts, hidden), generator=gen).cuda()
    prob, ids = ctx.moe_route(x, router, used)
    out = ctx.mx4_moe_ffn(tensor(*w_gate_up), tensor(*w_down), experts, x, prob, ids)
    order, token_of, offsets = ctx.moe_order(ids, experts)
    feed = ctx.mx4_quantize(x, rows=token_of)
    act = ctx.mx4_matmul_grouped(tensor(*w_gate_up), experts, feed, offsets, y_dtype=torch.float16, epilogue=SWIGLU)
    ids_host, edges = ids.cpu().numpy(), offsets.cpu().numpy()
    want_order, want_edges = order_of(ids_host, experts, tokens)
    assert np.array_equal(order.cpu().numpy(), want_order) and np.array_equal(edges, want_edges)
    x64 = _mx4.values(*_mx4.quantize(x.cpu().double().numpy()[want_order // used]))
    gate_up64, down64 = _mx4.values(*w_gate_up), _mx4.values(*w_down)
    act64 = _mx4.values(*_mx4.quantize(act.cpu().double().numpy()))
    proj64, proj_error = np.zeros((tokens * used, hidden)), np.zeros((tokens * used, hidden))
    for e in range(experts):
        a, b = edges[e], edges[e + 1]
        w64 = gate_up64[e * 2 * ffn:(e + 1) * 2 * ffn]
        y64, error = x64[a:b] @ w64.T, _mx4.sum_bound(w64, x64[a:b])
        assert _mx4.close(act.cpu().double().numpy()[a:b], _mx4.gated(y64), _mx4.gated_bound(y64, error, "f16"), "f16").all()
        w64 = down64[e * hidden:(e + 1) * hidden]
        proj64[want_order[a:b]] = act64[a:b] @ w64.T
        proj_error[want_order[a:b]] = _mx4.sum_bound(w64, act64[a:b])
    chosen = np.take_along_axis(prob.cpu().double().numpy(), ids_host.astype(np.int64), axis=1)[:, :, None]
    want = (proj64.reshape(tokens, used, hidden) * chosen).sum(axis=1)
    parts = (np.abs(proj64).reshape(tokens, used, hidden) * chosen).sum(axis=1)
    error = (proj_error.reshape(tokens, used, hidden) * chosen).sum(axis=1)
    # each rank: a rounded product and a rounded sum
    assert (np.abs(out.cpu().double().numpy() - want) <= error + parts * (2 * used) * 2.0 ** -24).all()
    # selections that name no expert, and tokens past the live ones
    ids[0, 0] = experts + 3
    live = torch.tensor([max(tokens - 1, 1)], dtype=torch.int32, device="cuda")
    got = torch.full((tokens, hidden), GUARD, device="cuda")
    ctx.mx4_moe_ffn(tensor(*w_gate_up), tensor(*w_down), experts, x, prob, ids, tokens_dev=live, out=got)
    rows = int(live)
    assert torch.equal(got[1:rows], out[1:rows])
    assert (got[rows:] == GUARD).all()
    part = (proj64.reshape(tokens, used, hidden) * chosen)[0, 1:].sum(axis=0)
    assert (np.abs(got[0].cpu().double().numpy() - part) <= error[0] + parts[0] * (2 * used) * 2.0 ** -24).all()


def test_weights_quantised_just_before(ctx):
    """A product right behind the quantisation of its weights, and behind one of other rows, reads what they wrote."""
    torch = torch_mod()
    n, k = 4096, 2048
    for m in (3, 300):
        x = ctx.mx4_quantize(torch.randn((m, k), device="cuda"))
        out = ctx.mx4_quantize(torch.zeros((n, k), device="cuda"))
        for turn in range(8):
            w = torch.randn((n, k), device="cuda").half()
            ctx.mx4_quantize(w, out=out)
            if turn % 2:
                x = ctx.mx4_quantize(torch.randn((m, k), device="cuda"))
            y = ctx.mx4_matmul(out, x)
            torch.cuda.synchronize()
            assert torch.equal(ctx.mx4_matmul(out, x), y)


@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_captured_twice_and_on_another_stream(ctx, m):
    """Two graphs of the same calls, replayed in turn with new inputs, and the calls on a second stream."""
    torch = torch_mod()
    n, k = 520, 544
    w = tensor(*random_codes(n, k, 3, -9, -3))
    x = torch.randn((m, k), device="cuda").half()
    ys = [torch.empty((m, n), device="cuda") for _ in range(2)]
    ctx.mx4_linear(w, x, y=ys[0])
    torch.cuda.synchronize()
    graphs = []
    for y in ys:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.mx4_linear(w, x, y=y)
            ctx.mx4_linear(w, x, y=y, epilogue=ADD)
        graphs.append(graph)
    for turn in range(4):
        x.copy_(torch.randn((m, k), device="cuda").half())
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        once = ctx.mx4_linear(w, x)
        assert torch.equal(ys[turn % 2], once + once)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ctx.mx4_linear(w, x)
    side.synchronize()
    assert torch.equal(other, ctx.mx4_linear(w, x))


def test_two_contexts_at_once(ctx):
    """Products whose tiles are cut between blocks, on two contexts and two streams at the same time: blocks wait for blocks of
    their own launch while the other launch holds some of the SMs."""
    import aotx_b200
    torch = torch_mod()
    other = aotx_b200.Q8Context(0)
    shapes = ((40000, 1056, 8), (20000, 2080, 300), (38000, 544, 130))
    tensors = [(tensor(*random_codes(n, k, n, -9, -3)), tensor(*random_codes(m, k, m, -4, 3))) for n, k, m in shapes]
    want = [ctx.mx4_matmul(w, x) for w, x in tensors]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for turn in range(6):
        for context, stream in zip((ctx, other), streams):
            with torch.cuda.stream(stream):
                w, x = tensors[(turn + (context is other)) % 3]
                results.append(((turn + (context is other)) % 3, context.mx4_matmul(w, x)))
    torch.cuda.synchronize()
    for i, got in results:
        assert torch.equal(got, want[i])
    assert other.device_status() == 0
    other.close()


def test_tensors_past_four_gigabytes(ctx):
    """Addresses of codes, of values and of results that pass 32 bits: the last rows against a tensor of those rows alone."""
    import aotx_b200
    torch = torch_mod()
    n, k, m = 1100000, 8192, 3
    w = aotx_b200.Mx4Tensor.empty(n, k, "cuda")
    w.codes.random_(0, 256)
    w.scales.random_(120, 124)
    x = torch.randn((m, k), device="cuda").half()
    last = slice(n - 300, n)
    part = aotx_b200.Mx4Tensor(w.codes[last].contiguous(), w.scales[:, last].contiguous())
    q = ctx.mx4_quantize(x)
    w64 = _mx4.values(part.codes.cpu().numpy(), part.scales.cpu().numpy())
    x64 = _mx4.values(q.codes.cpu().numpy(), q.scales.cpu().numpy())
    want, error = x64 @ w64.T, _mx4.sum_bound(w64, x64)
    assert _mx4.close(ctx.mx4_matmul(w, q)[:, last].double().cpu().numpy(), want, error, "f32").all()
    assert _mx4.close(ctx.mx4_linear(w, x)[:, last].double().cpu().numpy(), want, error, "f32").all()
    rows = 600000
    values = ctx.mx4_dequant(w, first_row=n - rows, rows=rows)
    assert torch.equal(values[-300:].double().cpu(), torch.from_numpy(w64).half().double())
    back = ctx.mx4_quantize(values)
    assert torch.equal(ctx.mx4_dequant(back, first_row=rows - 300, rows=300), values[-300:])
    del w, values, back
    torch.cuda.empty_cache()
    # many rows of x: results past 4 GB
    w = tensor(*random_codes(70000, 64, 1, -2, 2))
    x = tensor(*random_codes(20000, 64, 2, -2, 2))
    y = ctx.mx4_matmul(w, x)
    rows64, cols64 = _mx4.values(x.codes[-5:].cpu().numpy(), x.scales[:, -5:].contiguous().cpu().numpy()), \
        _mx4.values(w.codes[-200:].cpu().numpy(), w.scales[:, -200:].contiguous().cpu().numpy())
    assert np.array_equal(y[-5:, -200:].cpu().numpy(), (rows64 @ cols64.T).astype(np.float32))


# clusters whose blocks share an SM; x in as many parts as there are SMs or clusters for; a tile a block, up to 256 wide; pairs of blocks
# for one part of x, whole and cut
DEALT = [(12288, 320, 16), (18432, 512, 1), (6100, 4128, 8), (2500, 8192, 20), (512, 640, 512), (2048, 1056, 250), (5120, 288, 200),
         (8192, 288, 512), (12160, 544, 250), (18432, 288, 256), (19456, 800, 96), (19001, 352, 65), (20000, 1312, 128),
         (10240, 1056, 400)]


@pytest.mark.parametrize("n,k,m", DEALT)
def test_exact_sums_however_the_tiles_are_dealt(ctx, n, k, m):
    test_exact_sums(ctx, n, k, m)


@pytest.mark.parametrize("n,k,m,live", [(2560, 8192, 2048, 100), (2560, 8192, 2048, 0), (2560, 8192, 2048, 1999), (2560, 8192, 1500, 100),
                                        (6144, 512, 200, 70), (6144, 512, 200, 200), (6144, 512, 200, 130)])
def test_fewer_tiles_than_the_launch_provides_for(ctx, n, k, m, live):
    """The device finds fewer tiles than the host dealt: several blocks share one, and more than one leaves its sums to the owner.
    (Exact, as in test_exact_sums.)"""
    torch = torch_mod()
    w, x = random_codes(n, k, n + k, -2, 2), random_codes(m, k, m + k + 1, -2, 2)
    want = _mx4.values(*x)[:live] @ _mx4.values(*w).T
    y = torch.full((m, n), GUARD, device="cuda")
    ctx.mx4_matmul(tensor(*w), tensor(*x), m_dev=torch.tensor([live], dtype=torch.int32, device="cuda"), y=y)
    assert np.array_equal(y[:live].cpu().numpy(), want.astype(np.float32))
    assert (y[live:] == GUARD).all()


@pytest.mark.parametrize("counts,n,k", [([3, 2], 128, 8192), ([1], 384, 8192), ([70] * 8, 2560, 544), ([0, 200, 96, 65, 1, 97, 0, 33], 2600, 1056)])
def test_grouped_however_the_tiles_are_dealt(ctx, counts, n, k):
    grouped(ctx, counts, n, k)


@pytest.mark.parametrize("n,k,m,live", [(20480, 4128, 70, None), (20000, 4128, 300, None), (40000, 4128, 9, None), (20480, 4128, 384, 100),
                                        (38500, 3232, 40, 33)])
def test_a_few_cut_tiles_before_whole_ones(ctx, n, k, m, live):
    """Deep tiles, a few more than every block has one of: these few are cut.  (Exact, as in test_exact_sums; the sums in 64 bits are
    formed on the device, from values that test_gpu_y_mx4_quantize.py checks.)"""
    torch = torch_mod()
    w, x = tensor(*random_codes(n, k, n + k, -2, 2)), tensor(*random_codes(m, k, m + k + 1, -2, 2))
    rows = m if live is None else live
    x64 = ctx.mx4_dequant(x, dtype=torch.float32).double()[:rows]
    w64 = ctx.mx4_dequant(w, dtype=torch.float32).double()
    assert (x64.abs() @ w64.abs().T).max() < 2.0 ** 18
    y = torch.full((m, n), GUARD, device="cuda")
    for _ in range(2):
        y.fill_(GUARD)
        ctx.mx4_matmul(w, x, y=y, m_dev=None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda"))
        assert torch.equal(y[:rows], (x64 @ w64.T).float())
        assert (y[rows:] == GUARD).all()


@pytest.mark.parametrize("tokens,used,experts", [(128, 8, 128), (129, 8, 256), (1, 1, 256), (1024, 1, 2), (1025, 1, 33)])
def test_order_at_the_border_of_its_two_forms(ctx, tokens, used, experts):
    test_order(ctx, tokens, used, experts)


def test_order_of_no_tokens(ctx):
    torch = torch_mod()
    order, token_of, offsets = ctx.moe_order(torch.empty((0, 4), dtype=torch.int32, device="cuda"), 7)
    assert order.numel() == 0 and token_of.numel() == 0 and offsets.tolist() == [0] * 8
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    order, token_of, offsets = ctx.moe_order(torch.zeros((400, 4), dtype=torch.int32, device="cuda"), 7, tokens_dev=live)
    assert (order == -1).all() and (token_of == -1).all() and offsets.tolist() == [0] * 8
