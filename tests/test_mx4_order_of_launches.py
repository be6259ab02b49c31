"""When the launch behind an MX4 call may start, on the CPU (tests/mx4_emu.cu: the quantisation's kernel and the C interface as
host code).  A product may read its weights without waiting for the work before it; whatever a public quantisation writes may
be such weights, so it lets nothing behind it start before it has ended: whichever rows it takes, whatever runs on other streams
or is captured in between, whatever context the product is on."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import _mx4
from aotx_b200 import library

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    path = str(tmp_path_factory.mktemp("emu") / "libmx4_emu.so")
    done = subprocess.run([nvcc, "-O1", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-fno-strict-aliasing", "-gencode",
                           "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "aotx_b200", "csrc"),
                           "-I", os.path.join(ROOT, "tests"), "-o", path, os.path.join(ROOT, "tests", "mx4_emu.cu")],
                          capture_output=True, text=True, timeout=900)
    assert done.returncode == 0, done.stderr[-3000:]
    lib = C.CDLL(path)
    library.declare_mx4(lib)
    lib.mx4_emu_context.restype = C.c_void_p
    lib.mx4_emu_release.argtypes = [C.c_void_p]
    lib.mx4_emu_released.restype = C.c_uint32
    lib.mx4_emu_product.argtypes = [C.c_void_p, C.c_size_t]
    lib.mx4_emu_product.restype = C.c_size_t
    return lib


@pytest.fixture
def ctx(emu):
    made = C.c_void_p(emu.mx4_emu_context())
    yield made
    emu.mx4_emu_release(made)


def memory(size, value=0):
    """`size` bytes on a 16-byte boundary."""
    whole = np.full(size + 16, value, np.uint8)
    skip = -whole.ctypes.data % 16
    return whole[skip:skip + size]


class Rows:
    """Values, and room for them in MX4."""

    def __init__(self, rows, k, seed, kind=np.float16):
        rng = np.random.Generator(np.random.PCG64(seed))
        self.rows, self.k = rows, k
        self.x = memory(rows * k * kind().itemsize).view(kind).reshape(rows, k)
        self.x[:] = rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-9, 9, (rows, 1))
        self.codes = memory(rows * k // 2, 0xA5).reshape(rows, k // 2)
        self.scales = memory((k + 127) // 128 * rows * 4, 0x5A).reshape((k + 127) // 128, rows, 4)

    def quantize(self, emu, ctx, stream=None, order=None):
        listed = None if order is None else np.ascontiguousarray(order, np.uint32)
        code = emu.aotx_mx4_quantize(ctx, stream, self.x.ctypes.data, F16 if self.x.dtype == np.float16 else F32, self.rows, self.k,
                                     self.k, None if order is None else listed.ctypes.data, self.rows, None,
                                     self.codes.ctypes.data, self.scales.ctypes.data)
        assert code == 0
        want = _mx4.quantize(self.x if order is None else self.x[listed])
        assert np.array_equal(self.codes, want[0]) and np.array_equal(self.scales, want[1])


@pytest.mark.parametrize("kind", [np.float16, np.float32])
@pytest.mark.parametrize("listed", [False, True])
def test_nothing_starts_beside_a_quantisation(emu, ctx, kind, listed):
    w = Rows(70, 96, 1, kind)
    order = np.random.Generator(np.random.PCG64(2)).permutation(70) if listed else None
    emu.mx4_emu_released()
    w.quantize(emu, ctx, order=order)
    assert emu.mx4_emu_released() == 0


def test_the_product_of_a_linear_call_starts_beside_its_own_quantisation(emu, ctx):
    """(It reads x in MX4 behind its wait; the count shows that the stand-in sees a launch let go.)"""
    w, x = Rows(8, 64, 1), Rows(40, 64, 2)
    size = emu.aotx_mx4_linear_workspace_bytes(ctx, 8, 64, 40)
    work, y = memory(size), memory(40 * 8 * 4)
    emu.mx4_emu_released()
    assert emu.aotx_mx4_linear(ctx, None, w.codes.ctypes.data, w.scales.ctypes.data, 8, 64, x.x.ctypes.data, F16, 64, 40, None,
                               y.ctypes.data, F32, 0, work.ctypes.data, size) == 0
    assert emu.mx4_emu_released() > 0


def launched(emu):
    """The description that the last product was launched by."""
    room = C.create_string_buffer(4096)
    size = emu.mx4_emu_product(room, 4096)
    return room.raw[:size]


@pytest.mark.parametrize("call", ["matmul", "linear", "grouped"])
def test_a_product_is_launched_alike_whatever_was_quantised_before(emu, ctx, call):
    """A model's weights are laid out once, its last matrix last: no later product of that matrix is slower for it."""
    w, x, other = Rows(8, 64, 1), Rows(4, 64, 2), Rows(8, 64, 3)
    y = memory(4 * 8 * 4)
    offsets = np.array([0, 4], np.int32)

    def multiply():
        if call == "matmul":
            code = emu.aotx_mx4_matmul(ctx, None, w.codes.ctypes.data, w.scales.ctypes.data, 8, 64, x.codes.ctypes.data,
                                       x.scales.ctypes.data, 4, None, y.ctypes.data, F32, 0)
        elif call == "linear":
            code = emu.aotx_mx4_linear(ctx, None, w.codes.ctypes.data, w.scales.ctypes.data, 8, 64, x.x.ctypes.data, F16, 64, 4,
                                       None, y.ctypes.data, F32, 0, None, 0)
        else:
            code = emu.aotx_mx4_matmul_grouped(ctx, None, w.codes.ctypes.data, w.scales.ctypes.data, 1, 8, 64,
                                               x.codes.ctypes.data, x.scales.ctypes.data, 4, offsets.ctypes.data, None, 4,
                                               y.ctypes.data, F32, 0)
        assert code == 0
        return launched(emu)

    x.quantize(emu, ctx)
    other.quantize(emu, ctx)
    before = multiply()
    w.quantize(emu, ctx)
    assert any(before) and multiply() == before
    assert multiply() == before
