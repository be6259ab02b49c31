"""What the Python layer of the MX4 tensors hands to the library, on CPU tensors: the types between the steps of a routed layer."""
import pytest
import torch

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


def test_a_tensor_is_read_where_it_is():
    """Storage that is put elsewhere under an Mx4Tensor: the next call takes it from there, or refuses what no longer fits."""
    c = Recorded()
    codes, scales = own(8, 64)
    w, x = Mx4Tensor(codes, scales), Mx4Tensor.empty(6, 64, "cpu")
    c.mx4_matmul(w, x)
    assert passed(c) == ((codes.data_ptr(), scales.data_ptr()), (x.codes.data_ptr(), x.scales.data_ptr()))
    before = codes.data_ptr()
    codes.data, scales.data = own(8, 64)
    assert codes.data_ptr() != before
    c.mx4_matmul(w, x)
    assert passed(c)[0] == (codes.data_ptr(), scales.data_ptr())
    # an array of its own that grows, and moves
    kept = x.codes
    kept.untyped_storage().resize_(1 << 22)
    c.mx4_matmul(w, x)
    assert passed(c)[1] == (x.codes.data_ptr(), x.scales.data_ptr()) and x.codes.data_ptr() == kept.data_ptr()
    calls = len(c.calls)
    for change in (own(7, 64), own(8, 96), (own(8, 64)[0], own(8, 160)[1]), (codes[:4], scales), (codes.float(), scales),
                   (codes.t().contiguous().t(), scales)):
        moved = Mx4Tensor(*(t.clone() for t in own(8, 64)))
        moved.codes.data, moved.scales.data = change
        for call in (lambda: c.mx4_matmul(moved, x), lambda: c.mx4_matmul(x, moved), lambda: c.mx4_dequant(moved),
                     lambda: c.mx4_linear(moved, torch.zeros((6, 64))),
                     lambda: c.mx4_quantize(torch.zeros((8, 64)), out=moved),
                     lambda: c.mx4_matmul_grouped(moved, 2, x, torch.tensor([0, 3, 6], dtype=torch.int32))):
            with pytest.raises(ValueError):
                call()
    assert len(c.calls) == calls


def test_released_storage_is_passed_on_as_a_null_pointer():
    """(Which the library refuses.)"""
    c = Recorded()
    w, x = Mx4Tensor(*own(8, 64)), Mx4Tensor.empty(6, 64, "cpu")
    x.codes.untyped_storage().resize_(0)
    c.mx4_matmul(w, x)
    assert passed(c)[1][0] == 0
