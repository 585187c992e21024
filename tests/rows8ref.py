"""The definitions of the 8-bit activation operators in f64, and device rows,
for their tests."""
import numpy as np

import pywelvet
from tokmem import U, Dev

TINY = 2.0 ** -126
ACTS = ["linear", "relu", "silu", "gelu", "tanh", "sigmoid", "leakyrelu", "relu2"]


def codes_of(x):
    """x [n][width] (f64 of values that are exact in f32) -> codes (int64) and
    scales (f32).  The f64 quotient is within 2^-53 of the exact one, and the
    exact one is a half or at least 2^-34 of it away from one: (2 k + 1) s and
    2 x are whole multiples of a unit of 2^-33 or more of either."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x).all(1)
    top = np.where(fine, np.abs(np.where(np.isfinite(x), x, 0)).max(1, initial=0), 0)
    scale = (top.astype(np.float32) / np.float32(127)).astype(np.float32)
    s = scale.astype(np.float64)[:, None]
    q = np.rint(np.divide(x, s, out=np.zeros_like(x), where=(s > 0) & fine[:, None]))
    codes = np.where(fine[:, None], np.clip(q, -127, 127), 0).astype(np.int64)
    return codes, np.where(fine, scale, np.float32(np.nan)).astype(np.float32)


def values(codes, scales):
    with np.errstate(invalid="ignore"):
        return codes.astype(np.float64) * scales.astype(np.float64)[:, None]


def sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def act(x, name):
    if name == "relu":
        return np.maximum(x, 0)
    if name == "relu2":
        return np.maximum(x, 0) ** 2
    if name == "leakyrelu":
        return np.where(x < 0, x * 0.01, x)
    if name == "silu":
        return x * sigmoid(x)
    if name == "sigmoid":
        return sigmoid(x)
    if name == "tanh":
        return np.tanh(x)
    if name == "gelu":
        return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))
    return x


def act_prime(x, name):
    if name == "relu":
        return (x > 0) * 1.0
    if name == "relu2":
        return np.where(x > 0, 2 * x, 0)
    if name == "leakyrelu":
        return np.where(x > 0, 1.0, 0.01)
    if name == "silu":
        z = sigmoid(x)
        return z * (1 + x * (1 - z))
    if name == "sigmoid":
        z = sigmoid(x)
        return z * (1 - z)
    if name == "tanh":
        return 1 / np.cosh(np.clip(x, -300, 300)) ** 2
    if name == "gelu":
        a = np.sqrt(2 / np.pi)
        x = np.clip(x, -1e4, 1e4)
        z = sigmoid(2 * a * (x + 0.044715 * x ** 3))
        return z + x * z * (1 - z) * 2 * a * (1 + 0.134145 * x ** 2)
    return np.ones_like(x)


# The activations' own error.  Sigmoid: e^-|x| from an argument carried past f32
# and an exponential within 1 ulp, a sum, a reciprocal within 1 ulp: 4 ulp = 8 U
# of itself, and of its complement.  GELU's argument u is rounded four times, 4 U
# |u|, which moves z by z (1 - z) 4 U |u| <= 0.9 U, and the derivative's second
# term (at most 0.4, nothing past |u| = 20) by 80 U of it.  Then two to four
# roundings of values of at most |x| + 1.1.  tanhf is within 2 ulp.
ACT_ERR = 16 * U        # of |x| + 1
PRIME_ERR = 64 * U      # of 1


class Rows:
    """Rows in 8 bits on the device, filled with what must not matter."""

    def __init__(self, n, width, extra=0, codes=None, scales=None):
        self.n, self.width, self.stride = n, width, (width + 15) // 16 * 16 + 16 * extra
        host = np.full((n, self.stride), 77, np.int8)
        if codes is not None:
            host[:, :width] = codes
        self.codes = Dev(host)
        self.scales = Dev(np.full(n, 7.0, np.float32) if scales is None else scales.astype(np.float32))
        self.desc = pywelvet.rows8(self.codes.ptr, self.stride, self.scales.ptr)

    def get(self):
        """Codes and scales; the rest of each row as it has to be after a store."""
        raw = self.codes.get()
        end = (self.width + 15) // 16 * 16
        assert (raw[:, self.width:end] == 0).all() and (raw[:, end:] == 77).all()
        return raw[:, :self.width].astype(np.int64), self.scales.get()
