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
