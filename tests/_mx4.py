"""MX4 tensors in plain 64-bit arithmetic (test code only): the formulas of include/aotx_mx4_b200.h, no code of the package."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [rows][k] (any float type) -> codes, scales in the layout of the header.  Every step is exact in 64 bits."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    blocks = x.reshape(rows, k // 32, 32)
    bad = ~np.isfinite(blocks).all(axis=2)
    clean = np.where(bad[:, :, None], 0.0, blocks)
    largest = np.abs(clean).max(axis=2)
    exponent = np.where(largest > 0, np.frexp(np.where(largest > 0, largest, 1.0))[1] - 1 - 2, -127)
    exponent = np.maximum(exponent, -127)
    v = np.abs(np.ldexp(clean, -exponent[:, :, None]))
    # the nearest of the eight: above the middle of two, or on it if the upper one is even
    middle = (GRID[1:] + GRID[:-1]) / 2
    code = np.zeros(v.shape, np.uint8)
    for i, mid in enumerate(middle):
        code += (v >= mid) if (i + 1) % 2 == 0 else (v > mid)
    code = np.where(bad[:, :, None], 0, code + 8 * np.signbit(clean)).astype(np.uint8).reshape(rows, k)
    codes = code[:, 0::2] | code[:, 1::2] << 4
    chunks = (k + 127) // 128
    scales = np.zeros((rows, chunks * 4), np.uint8)
    scales[:, :k // 32] = np.where(bad, 255, exponent + 127)
    return codes, np.ascontiguousarray(scales.reshape(rows, chunks, 4).transpose(1, 0, 2))


def values(codes, scales):
    rows, half = codes.shape
    code = np.stack((codes & 15, codes >> 4), axis=2).reshape(rows, 2 * half)
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    byte = scales.transpose(1, 0, 2).reshape(rows, -1)[:, :half // 16].astype(np.int64)
    scale = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    return (v.reshape(rows, -1, 32) * scale[:, :, None]).reshape(rows, 2 * half)


def gated(y):
    """silu(gate) * up of columns that take turns."""
    gate, up = y[:, 0::2], y[:, 1::2]
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up


def half_step(dtype):
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]


def sum_bound(w, x):
    """How far a float sum of k products may be from its value: the products are exact, and each of the k additions may lose
    a step of a float (2^-23) of what has been summed so far, which is at most the sum of the magnitudes."""
    return np.abs(x) @ np.abs(w).T * (w.shape[1] * 2.0 ** -23)


def gated_bound(y, error, dtype):
    """The same behind the gated unit: silu has a slope below 1.1 and at most the size of its argument.  For a float result the
    unit's own arithmetic loses at most eight float steps (expf, sum, quotient, product: two each).  For 16 bits the
    exponential's argument, gate times a rounded constant, is off by 2^-23 of itself, which makes |gate| 2^-23 of the
    exponential; that is good to two units (2^-22), the reciprocal to one (2^-23), and there are three roundings more: in
    halves of a unit, 2^-24, 2 |gate| + 4 + 2 + 3."""
    gate, up = np.abs(y[:, 0::2]), np.abs(y[:, 1::2])
    e_gate, e_up = error[:, 0::2], error[:, 1::2]
    steps = 8 if dtype == "f32" else 9 + 2 * np.minimum(gate, 128)
    return 1.1 * e_gate * (up + e_up) + (gate + e_gate) * e_up + steps * 2.0 ** -24 * gate * up


def close(got, want, error, dtype):
    """A float sum within `error` of the value, then one rounding.  binary16: the smallest step is 2^-24, and what is 65520 or
    more (half a step above 65504, the largest) rounds to infinity, so where the float sum may be on either side of
    that border, either is right."""
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= error + (np.abs(want) + error) * half_step(dtype) + (2.0 ** -25 if dtype == "f16" else 0.0)
    if dtype != "f16":
        return near
    past = (np.copysign(np.inf, want) == got) & (np.abs(want) + error >= 65520)
    return past | (near & (np.abs(want) - error < 65520))
