"""The 4-bit blocks of include/staleynet_fp4.h in numpy and 64 bits, from their definition."""
import numpy as np

BLOCK = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LARGEST_SCALE = 252


def blocks_of(inner):
    return -(-inner // BLOCK)


def quantize(rows):
    """[rows][inner] floats -> codes [rows][blocks * 16] and scales [rows][blocks], uint8."""
    rows = np.asarray(rows, np.float32)
    count, inner = rows.shape
    padded = np.zeros((count, blocks_of(inner) * BLOCK), np.float32)
    padded[:, :inner] = rows
    v = padded.reshape(count, -1, BLOCK).astype(np.float64)
    codes = np.zeros(v.shape, np.uint8)
    scales = np.zeros(v.shape[:2], np.uint8)
    for r in range(count):
        for b in range(v.shape[1]):
            block = v[r, b]
            if not np.isfinite(block).all():
                scales[r, b] = 255
                continue
            largest = np.abs(block).max()
            e = -127
            while e < 125 and largest >= 7 * 2.0 ** e:  # the smallest power of two of which it is under 7
                e += 1
            scales[r, b] = e + 127
            a = np.minimum(np.abs(block) / 2.0 ** e, 6.0)
            distance = np.abs(a[:, None] - MAGNITUDES[None, :])
            near = distance == distance.min(1, keepdims=True)
            # Of two at the same distance, the one with the even code.
            code = np.where(near.sum(1) > 1, (near & (np.arange(8) % 2 == 0)).argmax(1), near.argmax(1))
            codes[r, b] = code + 8 * np.signbit(block)
    codes = codes.reshape(count, -1)
    return codes[:, 0::2] | codes[:, 1::2] << 4, scales


def dequantize(codes, scales, inner=None):
    """The values, float64, [..., blocks * 32] (the first `inner` of a row)."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
    values = np.where(nibbles >= 8, -1.0, 1.0) * MAGNITUDES[nibbles & 7]
    factor = np.where(scales > LARGEST_SCALE, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    values = values * np.repeat(factor, BLOCK, -1)
    return values if inner is None else values[..., :inner]


class View:
    """Part of a device buffer as a tensor argument: what `offset` elements of it leave."""

    def __init__(self, tensor, offset, count, itemsize=4):
        self.pointer = tensor.pointer + offset * itemsize
        self.count = count
        self.owner = tensor

    def __len__(self):
        return self.count
