"""Rows in 8 bits by their definition, in 64 bits on the host: what the tests hold the kernels to."""
import numpy as np

NUMBERS = np.array([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])  # e4m3, from 0 to 448


def nearest(v):
    """The index of the e4m3 number nearest to |v| (448 at most), of two equally near ones the even one."""
    size = np.abs(v)
    low = np.clip(np.searchsorted(NUMBERS, size, side="right") - 1, 0, len(NUMBERS) - 2)
    down, up = size - NUMBERS[low], NUMBERS[low + 1] - size
    return np.where(down < up, low, np.where(up < down, low + 1, low + (low & 1)))


def pack64(x):
    """(bytes of q, bytes of scale, values) of x [rows, cols] in float64."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    n, words = -(-cols // 32), -(-cols // 128)
    cells = np.zeros((rows, n, 32))
    cells.reshape(rows, -1)[:, :cols] = x
    fine = np.isfinite(cells)
    top = np.abs(np.where(fine, cells, 0.0)).max(2) if cells.size else np.zeros((rows, n))
    powers = 2.0 ** np.arange(-127, 128)
    byte = np.searchsorted(448.0 * powers, top)               # the first power that is large enough
    unit = powers[byte][:, :, None]
    code = nearest(np.where(fine, cells, 0.0) / unit)
    values = NUMBERS[code] * np.sign(np.where(fine, cells, 0.0)) * unit
    code = np.where(fine, code | np.where(np.signbit(cells), 0x80, 0), 0x7F).astype(np.uint8)
    values = np.where(fine, values, np.nan)
    scale = np.zeros((rows, 4 * words), np.uint8)
    scale[:, :n] = byte
    return code.reshape(rows, 32 * n), scale, values.reshape(rows, -1)[:, :cols]
