"""Device buffers of any numpy type, 16-bit floats and bounds for the tests of
the token-side operators (embedding, adapters, distillation)."""
import ctypes as C

import numpy as np

import devmem

U = 2.0 ** -24  # half an f32 ulp, relative
DT = {"float32": 1, "float16": 2, "bfloat16": 3}


def to_bits(a, dtype):
    """f32 values rounded (to nearest even) into a dtype's own array."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "float32":
        return a
    if dtype == "float16":
        return a.astype(np.float16)
    u = a.view(np.uint32)
    r = ((u >> 16) & 1) + np.uint32(0x7FFF)
    out = ((u + r) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), out).astype(np.uint16)


def to_f64(b, dtype):
    if dtype == "bfloat16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


class Dev:
    """A device copy of a numpy array; .get() reads it back.  `guard` values
    of 0xA5 bytes lie on either side, checked at every get."""
    GUARD = 256

    def __init__(self, a):
        a = np.ascontiguousarray(a)
        self.shape, self.dtype, self.nbytes = a.shape, a.dtype, a.nbytes
        p = C.c_void_p()
        devmem._ok(devmem.hip().hipMalloc(C.byref(p), a.nbytes + 2 * self.GUARD), "hipMalloc")
        self.base, self.ptr = p.value, p.value + self.GUARD
        raw = np.full(a.nbytes + 2 * self.GUARD, 0xA5, np.uint8)
        raw[self.GUARD:self.GUARD + a.nbytes] = a.reshape(-1).view(np.uint8)
        devmem._ok(devmem.hip().hipMemcpy(self.base, raw.ctypes.data, raw.nbytes, 1), "hipMemcpy H2D")

    def get(self):
        devmem._ok(devmem.hip().hipDeviceSynchronize(), "hipDeviceSynchronize")
        raw = np.empty(self.nbytes + 2 * self.GUARD, np.uint8)
        devmem._ok(devmem.hip().hipMemcpy(raw.ctypes.data, self.base, raw.nbytes, 2), "hipMemcpy D2H")
        assert (raw[:self.GUARD] == 0xA5).all() and (raw[self.GUARD + self.nbytes:] == 0xA5).all(), \
            "written outside the array"
        return raw[self.GUARD:self.GUARD + self.nbytes].copy().view(self.dtype).reshape(self.shape)

    def __del__(self):
        try:
            if self.base:
                devmem.hip().hipFree(self.base)
                self.base = None
        except Exception:
            pass


class Big:
    """Uninitialised device memory with writes and reads at byte offsets."""

    def __init__(self, nbytes):
        p = C.c_void_p()
        devmem._ok(devmem.hip().hipMalloc(C.byref(p), nbytes), "hipMalloc")
        self.ptr = p.value

    def put(self, at, a):
        a = np.ascontiguousarray(a)
        devmem._ok(devmem.hip().hipMemcpy(self.ptr + at, a.ctypes.data, a.nbytes, 1), "hipMemcpy H2D")

    def get(self, at, shape, dtype):
        out = np.empty(shape, dtype)
        devmem._ok(devmem.hip().hipDeviceSynchronize(), "hipDeviceSynchronize")
        devmem._ok(devmem.hip().hipMemcpy(out.ctypes.data, self.ptr + at, out.nbytes, 2), "hipMemcpy D2H")
        return out

    def free(self):
        devmem.hip().hipFree(self.ptr)


def strided(a, extra, fill=np.nan):
    """a [rows][cols] inside rows of cols + extra, the rest `fill`."""
    if not extra:
        return np.ascontiguousarray(a)
    fill = 0x7FC0 if a.dtype == np.uint16 else fill
    out = np.full((a.shape[0], a.shape[1] + extra), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def within(got, want, bound, what):
    """Element-wise |got - want| <= bound; NaN and infinities in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities"
    d = np.abs(got - want)[fine] - np.broadcast_to(bound, want.shape)[fine]
    assert d.size == 0 or d.max() <= 0, \
        f"{what}: {np.count_nonzero(d > 0)} of {d.size} past their bound, the worst by {d.max():.3e}"
