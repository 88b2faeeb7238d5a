"""Element types of the operators that take more than fp32, for tests: host arrays as the bits in memory, values in float64."""
import numpy as np

TYPES = ("f32", "f16", "bf16")
STORAGE = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # of a rounding, relative to the value
SMALLEST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}    # half a step of the subnormal numbers
U = 2.0 ** -24


def stored(values, type_):
    """float64 or float32 values as `type_` in memory, rounded to nearest even."""
    f = np.asarray(values, dtype=np.float32)
    if type_ != "bf16":
        with np.errstate(over="ignore"):
            return f.astype(STORAGE[type_])
    bits = f.view(np.uint32).astype(np.uint64)
    rounded = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7fc0), rounded).astype(np.uint16)


def values(array, type_):
    """What an array in memory holds, in float64."""
    if type_ != "bf16":
        return np.asarray(array, dtype=np.float64)
    return (np.asarray(array).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def place(ctx, matrix, type_, pad=0, shift=0, fill=77.0):
    """A device array that holds `matrix` (values) in rows `pad` places longer than its own, from its element `shift` on -> (the array, a view that starts there)."""
    rows, cols = matrix.shape
    flat = np.full(shift + rows * (cols + pad), fill, dtype=np.float32)
    flat[shift:].reshape(rows, cols + pad)[:, :cols] = matrix
    whole = ctx.array(stored(flat, type_), STORAGE[type_])
    return whole, whole.offset(shift)


def fetch(whole, rows, cols, type_, pad=0, shift=0):
    """(the matrix's values, what lies in the places before and behind its rows)."""
    flat = values(whole.download(), type_)
    body = flat[shift:].reshape(rows, cols + pad)
    return body[:, :cols], np.concatenate([flat[:shift], body[:, cols:].ravel()])


def place_apart(ctx, matrix, type_, stride):
    """A device array whose rows lie `stride` elements apart, nothing written between them."""
    rows, cols = matrix.shape
    whole = ctx.empty(((rows - 1) * stride + cols,), STORAGE[type_])
    for r in range(rows):
        line = np.ascontiguousarray(stored(matrix[r], type_))
        ctx._ck(ctx.lib.so_h2d(ctx.h, whole.offset(r * stride).ptr, line.ctypes.data, line.nbytes))
    return whole


def fetch_apart(ctx, whole, rows, cols, type_, stride):
    out = np.empty((rows, cols), STORAGE[type_])
    for r in range(rows):
        ctx._ck(ctx.lib.so_d2h(ctx.h, out[r].ctypes.data, whole.offset(r * stride).ptr, out[r].nbytes))
    return values(out, type_)
