"""What the Python layer of the MX4 tensors hands to the library, on CPU tensors: the types between the steps of a routed layer."""
import copy
import ctypes as C

import pytest
import torch

from aotx_b200 import library
from aotx_b200.mx4 import Mx4Calls, Mx4Tensor

F32, F16, BF16 = 0, 1, 2


class Recorded(Mx4Calls):
    """Every call is written down and does nothing."""
    device = torch.device("cpu")
    _address = 1

    def __init__(self):
        self.lib = self
        self.calls = []
        for name in ("quantize", "dequant", "matmul", "linear", "order", "grouped"):
            setattr(self, "_mx4_%s_call" % name, lambda *args, name=name: self.calls.append((name, args)) or 0)

    def aotx_mx4_linear_workspace_bytes(self, ctx, n, k, m):
        return 64

    def moe_combine(self, proj, prob, ids, tokens_dev=None, out=None, out_dtype=None):
        self.calls.append(("combine", (proj.dtype, out_dtype)))
        return out

    def _stream(self):
        return 0


@pytest.mark.parametrize("kind,code", [(torch.float32, F32), (torch.float16, F16), (torch.bfloat16, BF16)])
def test_the_activation_of_a_routed_step_has_the_type_of_x(kind, code):
    """binary16 holds nothing above 65504: what a bfloat16 or float layer's gated unit gives may be larger."""
    c = Recorded()
    x, prob, ids = torch.zeros((6, 64), dtype=kind), torch.zeros((6, 4)), torch.zeros((6, 2), dtype=torch.int32)
    c.mx4_moe_ffn(Mx4Tensor.empty(4 * 2 * 96, 64, "cpu"), Mx4Tensor.empty(4 * 64, 96, "cpu"), 4, x, prob, ids)
    names = [name for name, _ in c.calls]
    assert names == ["order", "quantize", "grouped", "quantize", "grouped", "combine"]
    up, again, down = (c.calls[i][1] for i in (2, 3, 4))
    assert up[-2] == code and again[3] == code and down[-2] == F32
    assert up[-3] == again[2]            # the same rows


def own(rows, k):
    return torch.zeros((rows, k // 2), dtype=torch.uint8), torch.zeros(((k + 127) // 128, rows, 4), dtype=torch.uint8)


def passed(c):
    """The addresses of w and of x that the last product was given."""
    args = c.calls[-1][1]
    return args[2:4], args[6:8]


def places(t):
    return t.codes.data_ptr(), t.scales.data_ptr()


def test_a_tensor_is_read_where_it_is():
    """Storage that is put elsewhere is followed; it is the tensor's own for as long as the tensor lives, whatever its caller does
    with the two that it was made of."""
    c = Recorded()
    codes, scales = own(8, 64)
    w, x = Mx4Tensor(codes, scales), Mx4Tensor.empty(6, 64, "cpu")
    c.mx4_matmul(w, x)
    assert passed(c) == ((codes.data_ptr(), scales.data_ptr()), places(x)) == (places(w), places(x))
    # more room for either, which lies elsewhere then
    for t in (codes, scales, x.codes):
        before = t.data_ptr()
        t.untyped_storage().resize_(1 << 22)
        assert t.data_ptr() != before
    c.mx4_matmul(w, x)
    assert passed(c) == ((codes.data_ptr(), scales.data_ptr()), places(x))
    c.mx4_matmul(x, w)
    assert passed(c) == (places(x), (codes.data_ptr(), scales.data_ptr()))
    # other storage for the caller's tensors, and for what the properties gave; other shapes
    kept = passed(c)
    codes.fill_(7)
    w.codes.data, x.codes.data = own(3, 64)[0], own(3, 64)[0]
    codes.data, scales.data = own(8, 32)
    codes.resize_(2, 4)
    del codes, scales
    c.mx4_matmul(x, w)
    assert passed(c) == kept == (places(x), places(w)) and w.codes.shape == (8, 32) and (w.codes == 7).all()


def test_a_copy_is_read_where_the_copy_is():
    c = Recorded()
    w, x = copy.deepcopy(Mx4Tensor(*own(8, 64))), copy.deepcopy(Mx4Tensor.empty(6, 64, "cpu"))
    c.mx4_matmul(w, x)
    assert passed(c) == (places(w), places(x))


def test_released_storage_is_passed_on_as_a_null_pointer():
    """(Which the library refuses.)"""
    c = Recorded()
    w, x = Mx4Tensor(*own(8, 64)), Mx4Tensor.empty(6, 64, "cpu")
    x.codes.untyped_storage().resize_(0)
    c.mx4_matmul(w, x)
    assert passed(c)[1][0] == 0


def test_the_size_of_a_workspace_as_ctypes_gives_it():
    lib = library.load_library()
    call = library.native_call(lib, "aotx_mx4_linear_workspace_bytes")
    assert call.func.__name__ == "aotx_mx4_linear_workspace_bytes"
    ctx = C.cast(C.create_string_buffer(4096), C.c_void_p).value        # zeros: no SM, so nothing is quantised by the product
    for n, k, m in ((8, 64, 40), (1, 96, 1 << 24), (8, 33, 40), (0, 64, 40), (8, 64, 0), (1 << 20, 1 << 24, 1 << 20)):
        assert call(ctx, n, k, m) == lib.aotx_mx4_linear_workspace_bytes(ctx, n, k, m)
    assert call(ctx, 8, 64, 40) >= 40 * 32 + 40 * 4 and call(None, 8, 64, 40) == 0
    for wrong in ((ctx, 8, 64), (ctx, 8, 64, 40, 0), (ctx, 8.0, 64, 40), (ctx, None, 64, 40)):
        with pytest.raises(TypeError):
            call(*wrong)


class OnMeta(Recorded):
    """Tensors of any size, with nothing in them."""
    device = torch.device("meta")


def blank(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_sizes_past_the_limits_are_refused_and_not_cut_to_32_bits():
    """(The native calls take numbers modulo their width: 2^32 + 64 values would have been 64.)"""
    c = OnMeta()
    wide, far = (1 << 32) + 64, (1 << 32) + 5
    calls = [
        lambda: c.mx4_quantize(blank(1, wide, dtype=torch.float16)),
        lambda: c.mx4_quantize(blank(2, 64, dtype=torch.float16), rows=blank(far)),
        lambda: c.mx4_quantize(blank(2, 64, dtype=torch.float16), rows=blank(1 << 31)),
        lambda: Mx4Tensor.empty(1, wide, "meta"), lambda: Mx4Tensor.empty(1, (1 << 24) + 32, "meta"),
        lambda: Mx4Tensor.empty(far, 32, "meta"), lambda: Mx4Tensor.empty(1 << 31, 32, "meta"),
        lambda: Mx4Tensor(blank(far, 16, dtype=torch.uint8), blank(1, far, 4, dtype=torch.uint8)),
        lambda: Mx4Tensor(blank(1, wide // 2, dtype=torch.uint8), blank((wide + 127) // 128, 1, 4, dtype=torch.uint8)),
        lambda: c.moe_order(blank(far, 1), 8), lambda: c.moe_order(blank(1 << 30, 2), 8),
        lambda: c.moe_order(blank(4, 2), (1 << 32) + 8), lambda: c.moe_order(blank(4, 2), 257),
        lambda: c.mx4_matmul_grouped(Mx4Tensor.empty(0, 64, "meta"), far, Mx4Tensor.empty(4, 64, "meta"), blank(far + 1)),
        lambda: c.mx4_matmul_grouped(Mx4Tensor.empty(4, 64, "meta"), 2, Mx4Tensor.empty(4, 64, "meta"), blank(3), y_rows=blank(4),
                                     y=blank(far, 2, dtype=torch.float32)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            raise AssertionError("call %d went through" % i)
    assert c.calls == []
    # the limits themselves
    c.mx4_quantize(blank(1, 1 << 24, dtype=torch.float16))
    c.mx4_quantize(blank(2, 64, dtype=torch.float16), rows=blank((1 << 31) - 1))
    c.moe_order(blank((1 << 31) - 1, 1), 256)
    assert len(c.calls) == 3
