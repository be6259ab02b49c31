"""MX4 tensors on the CPU: the declared symbols, the refusals of the C interface and of the Python layer, the kernels' registers
and spills, and the plain forms that the GPU tests compare with."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import _mx4
import aotx_b200
from aotx_b200 import build as builder
from aotx_b200 import library
from aotx_b200.mx4 import Mx4Calls, Mx4Tensor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARGUMENT, WORKSPACE = 1, 5
F32, F16, BF16 = 0, 1, 2
STORE, ADD, SWIGLU = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    builder.build()
    return library.load_library()


@pytest.fixture(scope="module")
def ctx():
    """Zeros where a context would be: a refused call looks at nothing in it."""
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def test_every_declared_symbol_is_there(lib):
    with open(os.path.join(ROOT, "include", "aotx_mx4_b200.h")) as f:
        declared = set(re.findall(r"\b(aotx_mx4_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)))
    assert declared == set(library.MX4_SYMBOLS)
    for name in declared:
        assert hasattr(lib, name)


def test_kernels_spill_nothing():
    builder.build()
    usage = builder.resource_usage(builder.MX4_SOURCES)
    assert sum("mx4_" in name for name in usage) >= 10
    for name, use in usage.items():
        # (a frame of two words: the flag that the out-of-line wait is given)
        assert use["spill_stores"] == 0 and use["spill_loads"] == 0 and use["stack"] <= 8, (name, use)


P = 4096     # an aligned address that is never read

GOOD = {
    "aotx_mx4_quantize": dict(x=P, x_dtype=F16, x_rows=4, ldx=64, k=64, rows_of=None, rows=4, rows_dev=None, codes=P, scales=P),
    "aotx_mx4_dequant": dict(codes=P, scales=P, total_rows=4, k=64, first_row=0, rows=4, out=P, out_dtype=F16),
    "aotx_mx4_matmul": dict(w_codes=P, w_scales=P, n=4, k=64, x_codes=P, x_scales=P, m=4, m_dev=None, y=P, y_dtype=F32,
                            epilogue=STORE),
    "aotx_mx4_linear": dict(w_codes=P, w_scales=P, n=4, k=64, x=P, x_dtype=F16, ldx=64, m=4, m_dev=None, y=P, y_dtype=F32,
                            epilogue=STORE, workspace=P, workspace_bytes=1 << 20),
    "aotx_mx4_moe_order": dict(ids=P, tokens=4, tokens_dev=None, used=2, experts=8, order=P, token_of=P, offsets=P),
    "aotx_mx4_matmul_grouped": dict(w_codes=P, w_scales=P, experts=2, n=4, k=64, x_codes=P, x_scales=P, rows=4, offsets=P,
                                    y_rows_of=None, y_rows=4, y=P, y_dtype=F32, epilogue=STORE),
}
WRONG = [
    ("aotx_mx4_quantize", dict(x=0)), ("aotx_mx4_quantize", dict(x=P + 1)), ("aotx_mx4_quantize", dict(x=P + 2, x_dtype=F32)),
    ("aotx_mx4_quantize", dict(x_dtype=3)), ("aotx_mx4_quantize", dict(ldx=63)), ("aotx_mx4_quantize", dict(k=0)),
    ("aotx_mx4_quantize", dict(k=(1 << 24) + 32, ldx=1 << 25)),
    ("aotx_mx4_quantize", dict(k=48, ldx=48)), ("aotx_mx4_quantize", dict(rows=5)), ("aotx_mx4_quantize", dict(codes=P + 8)),
    ("aotx_mx4_quantize", dict(codes=0)), ("aotx_mx4_quantize", dict(scales=P + 2)), ("aotx_mx4_quantize", dict(scales=0)),
    ("aotx_mx4_quantize", dict(rows_of=P + 2)), ("aotx_mx4_quantize", dict(rows_dev=P + 1)),
    ("aotx_mx4_dequant", dict(first_row=1)), ("aotx_mx4_dequant", dict(rows=5)), ("aotx_mx4_dequant", dict(out=0)),
    ("aotx_mx4_dequant", dict(out=P + 2, out_dtype=F32)), ("aotx_mx4_dequant", dict(out_dtype=-1)),
    ("aotx_mx4_dequant", dict(k=33)), ("aotx_mx4_dequant", dict(first_row=2 ** 32 - 2)),
    ("aotx_mx4_matmul", dict(k=40)), ("aotx_mx4_matmul", dict(k=1 << 25)), ("aotx_mx4_matmul", dict(y_dtype=7)), ("aotx_mx4_matmul", dict(y=0)),
    ("aotx_mx4_matmul", dict(y=P + 2)), ("aotx_mx4_matmul", dict(w_codes=P + 4)), ("aotx_mx4_matmul", dict(x_codes=0)),
    ("aotx_mx4_matmul", dict(x_scales=P + 1)), ("aotx_mx4_matmul", dict(epilogue=3)), ("aotx_mx4_matmul", dict(epilogue=-1)),
    ("aotx_mx4_matmul", dict(epilogue=ADD, y_dtype=F16)), ("aotx_mx4_matmul", dict(epilogue=SWIGLU, n=5)),
    ("aotx_mx4_matmul", dict(m=1 << 25)), ("aotx_mx4_matmul", dict(n=1 << 31)), ("aotx_mx4_matmul", dict(m_dev=P + 2)),
    ("aotx_mx4_linear", dict(x=0)), ("aotx_mx4_linear", dict(ldx=32)), ("aotx_mx4_linear", dict(x_dtype=9)),
    ("aotx_mx4_linear", dict(epilogue=ADD, y_dtype=BF16)), ("aotx_mx4_linear", dict(k=16, ldx=16)),
    ("aotx_mx4_moe_order", dict(experts=0)), ("aotx_mx4_moe_order", dict(experts=257)), ("aotx_mx4_moe_order", dict(used=0)),
    ("aotx_mx4_moe_order", dict(ids=0)), ("aotx_mx4_moe_order", dict(offsets=0)), ("aotx_mx4_moe_order", dict(order=0)),
    ("aotx_mx4_moe_order", dict(tokens=1 << 30, used=2)), ("aotx_mx4_moe_order", dict(token_of=P + 2)),
    ("aotx_mx4_matmul_grouped", dict(experts=0)), ("aotx_mx4_matmul_grouped", dict(experts=300)),
    ("aotx_mx4_matmul_grouped", dict(epilogue=ADD)), ("aotx_mx4_matmul_grouped", dict(offsets=0)),
    ("aotx_mx4_matmul_grouped", dict(offsets=P + 2)), ("aotx_mx4_matmul_grouped", dict(y_rows_of=P + 2)),
    ("aotx_mx4_matmul_grouped", dict(experts=256, n=1 << 24)), ("aotx_mx4_matmul_grouped", dict(y=0)),
    ("aotx_mx4_matmul_grouped", dict(epilogue=SWIGLU, n=3)),
    ("aotx_mx4_matmul_grouped", dict(rows=1 << 24, n=(1 << 16) + 128)),
]


@pytest.mark.parametrize("name,change", WRONG)
def test_refused_before_anything_is_enqueued(lib, ctx, name, change):
    call = getattr(lib, name)
    assert call(ctx, None, *dict(GOOD[name], **change).values()) == ARGUMENT
    assert call(None, None, *GOOD[name].values()) == ARGUMENT


def test_nothing_to_do_is_no_error(lib, ctx):
    for name, empty in (("aotx_mx4_quantize", dict(rows=0)), ("aotx_mx4_dequant", dict(rows=0)), ("aotx_mx4_matmul", dict(m=0)),
                        ("aotx_mx4_matmul", dict(n=0)), ("aotx_mx4_linear", dict(m=0)), ("aotx_mx4_linear", dict(n=0)),
                        ("aotx_mx4_matmul_grouped", dict(rows=0)), ("aotx_mx4_matmul_grouped", dict(n=0))):
        assert getattr(lib, name)(ctx, None, *dict(GOOD[name], **empty).values()) == 0


def test_workspace_of_a_linear_call(lib, ctx):
    m, k = 300, 96
    n = GOOD["aotx_mx4_linear"]["n"]
    size = lib.aotx_mx4_linear_workspace_bytes(ctx, n, k, m)
    assert size >= m * k // 2 + m * 4
    call = dict(GOOD["aotx_mx4_linear"], m=m, k=k, ldx=k)
    for wrong in (dict(workspace=0), dict(workspace=P + 8), dict(workspace_bytes=size - 1)):
        assert lib.aotx_mx4_linear(ctx, None, *dict(call, **wrong).values()) == WORKSPACE


class OnCpu(Mx4Calls):
    """The Python layer on CPU tensors: every call is refused, or gets as far as the library."""
    device = torch.device("cpu")
    _address = 0

    class Reached(Exception):
        pass

    def __init__(self):
        def reached(*args):
            raise self.Reached()
        self.lib = self
        for name in ("quantize", "dequant", "matmul", "linear", "order", "grouped"):
            setattr(self, "_mx4_%s_call" % name, reached)

    def aotx_mx4_linear_workspace_bytes(self, ctx, n, k, m):
        return 64

    def _stream(self):
        return 0

    def _check(self, code):
        raise AssertionError("not reached")


def words(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_python_layer_refuses_and_passes_on():
    c = OnCpu()
    x, w = Mx4Tensor.empty(6, 64, "cpu"), Mx4Tensor.empty(8, 64, "cpu")
    rows = torch.zeros((6, 64))
    passes = [
        lambda: c.mx4_quantize(rows), lambda: c.mx4_quantize(rows, rows=words(5, 0), rows_dev=words(1)),
        lambda: c.mx4_quantize(torch.zeros((6, 100))[:, 4:68]), lambda: c.mx4_dequant(x, first_row=2, rows=4),
        lambda: c.mx4_matmul(w, x), lambda: c.mx4_matmul(w, x, epilogue=SWIGLU, y=torch.zeros((6, 4))),
        lambda: c.mx4_matmul(w, x, epilogue=ADD, y=torch.zeros((6, 8)), m_dev=words(3)), lambda: c.mx4_linear(w, rows),
        lambda: c.moe_order(torch.zeros((6, 2), dtype=torch.int32), 4),
        lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 3, 6)),
        lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 3, 6), y_rows=words(0, 1, 2, 3, 4, 5), y=torch.zeros((9, 4))),
    ]
    for call in passes:
        with pytest.raises(OnCpu.Reached):
            call()
    refused = [
        lambda: c.mx4_quantize(rows.double()), lambda: c.mx4_quantize(torch.zeros((2, 40))), lambda: c.mx4_quantize(rows.t()),
        lambda: c.mx4_quantize(rows, rows=torch.zeros(2)), lambda: c.mx4_quantize(rows, rows=words(1, 2, 3, 4)[::2]),
        lambda: c.mx4_quantize(rows, out=w), lambda: c.mx4_quantize(rows, rows_dev=words(1, 2)),
        lambda: c.mx4_quantize(torch.zeros((1, 64)).expand(3, 64)), lambda: c.mx4_quantize(rows.to("meta")),
        lambda: c.mx4_dequant(x, first_row=3, rows=4), lambda: c.mx4_dequant(x, out=torch.zeros((5, 64))),
        lambda: c.mx4_dequant(x, dtype=torch.int32), lambda: c.mx4_matmul(w, Mx4Tensor.empty(2, 96, "cpu")),
        lambda: c.mx4_matmul(w, x, y=torch.zeros((6, 4))), lambda: c.mx4_matmul(w, x, epilogue=ADD),
        lambda: c.mx4_matmul(w, x, epilogue=5), lambda: c.mx4_matmul(Mx4Tensor.empty(7, 64, "cpu"), x, epilogue=SWIGLU),
        lambda: c.mx4_matmul(w, x, y=torch.zeros((6, 16))[:, ::2]), lambda: c.mx4_matmul(w, x, m_dev=torch.zeros(1)),
        lambda: c.mx4_matmul(w, x, y=torch.zeros((6, 8)), y_dtype=torch.float16),
        lambda: c.mx4_linear(w, torch.zeros((6, 96))), lambda: c.mx4_linear(w, rows.to("meta")),
        lambda: c.moe_order(torch.zeros(6, dtype=torch.int32), 4), lambda: c.moe_order(torch.zeros((6, 2)), 4),
        lambda: c.mx4_matmul_grouped(w, 3, x, words(0, 1, 2, 3)), lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 6)),
        lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 3, 6), y_rows=words(0, 1)),
        lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 3, 6), y=torch.zeros((9, 4))),
        lambda: c.mx4_matmul_grouped(w, 2, x, words(0, 3, 6), epilogue=ADD, y=torch.zeros((6, 4))),
        lambda: Mx4Tensor(torch.zeros((2, 16), dtype=torch.uint8), torch.zeros((2, 2, 4), dtype=torch.uint8)),
        lambda: Mx4Tensor(torch.zeros((2, 8), dtype=torch.uint8), torch.zeros((1, 2, 4), dtype=torch.uint8)),
        lambda: Mx4Tensor(torch.zeros((2, 16)), torch.zeros((1, 2, 4), dtype=torch.uint8)),
        lambda: Mx4Tensor.empty(2, 33, "cpu"),
        lambda: c.mx4_moe_ffn(w, w, 2, rows, torch.zeros((6, 2)), torch.zeros((6, 1), dtype=torch.int32)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            raise AssertionError("call %d went through" % i)


def test_plain_form_rounds_as_the_format_says():
    # borders between codes, both signs, at three scales; what saturates; zeros; the smallest and largest floats
    values = np.array([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 0.2499, 0.2501])
    want = np.array([6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, 0.0, 0.5])
    for power in (-100, 0, 90):
        x = np.zeros((1, 32))
        x[0, :12], x[0, 12:24] = values, -values
        got = _mx4.values(*_mx4.quantize(np.ldexp(x, power)))
        assert np.array_equal(got[0, :24], np.ldexp(np.concatenate((want, -want)), power))
    edge = np.zeros((3, 32))
    edge[0, 0], edge[1, 0], edge[2, 0] = 2.0 ** -149, 2.0 ** 127 * (2 - 2.0 ** -23), 2.0 ** -126
    codes, scales = _mx4.quantize(edge)
    assert scales[0, :, 0].tolist() == [0, 252, 0]
    assert _mx4.values(codes, scales)[:, 0].tolist() == [0.0, 6 * 2.0 ** 125, 2.0 ** -126]


CALLS = {"aotx_mx4_quantize": (None, 0, 0, 1, 4, 64, 64, 0, 4, 0, 0, 0),
         "aotx_mx4_dequant": (None, 0, 0, 0, 4, 64, 0, 4, 0, 1),
         "aotx_mx4_matmul": (None, 0, 0, 0, 4, 64, 0, 0, 4, 0, 0, 0, 0),
         "aotx_mx4_linear": (None, 0, 0, 0, 4, 64, 0, 1, 64, 4, 0, 0, 0, 0, 0, 0),
         "aotx_mx4_moe_order": (None, 0, 0, 4, 0, 2, 8, 0, 0, 0),
         "aotx_mx4_matmul_grouped": (None, 0, 0, 0, 2, 4, 64, 0, 0, 4, 0, 0, 4, 0, 0, 0)}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_the_package_calls_the_library_as_ctypes_does(lib, name):
    call, good = library.native_call(lib, name), CALLS[name]
    assert call(*good) == getattr(lib, name)(*good) != 0      # no context
    for wrong in (good[:-1], good + (0,), (1.5,) + good[1:], ("x",) + good[1:]):
        with pytest.raises(TypeError):
            call(*wrong)
    for i, kind in enumerate(getattr(lib, name).argtypes):
        one = good[:i] + (None,) + good[i + 1:]
        if kind is C.c_void_p:
            assert call(*one) != 0
        else:
            with pytest.raises(TypeError):
                call(*one)


def test_every_argument_arrives_in_its_place():
    for name in CALLS:
        kinds = getattr(library.load_library(), name).argtypes
        seen = []
        answer = C.CFUNCTYPE(C.c_int, *kinds)(lambda *args: seen.append(args) or 7)
        stub = type("Library", (), {name: answer})
        wide = (C.c_void_p, C.c_uint64, C.c_size_t)
        sent = tuple(0x7F1234567000 + i if kind in wide else 100 + i for i, kind in enumerate(kinds))
        assert library.native_call(stub, name)(*sent) == 7
        assert seen == [sent]


def test_counted_stores_of_four_words_are_acquired_at_cluster_scope():
    """(What tests/test_counted_stores.py holds of the stores of one word.)"""
    with open(os.path.join(builder.CSRC, "mx4_product.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    counted = re.findall(r"store_counted_v4\([^;]*mapa_shared\((\w+), \w+\)\);", code)
    assert counted == ["exchanged"] and code.count("store_counted_v4(") == 1
    assert set(re.findall(r"(mbar_\w*(?:wait|test)\w*)\(\s*exchanged\b", code)) == {"mbar_wait_counted"}
