"""The 8-bit blocks of include/staleynet_fp8.h in numpy and 64 bits, from their definition."""
import numpy as np

BLOCK = 128
LEAST_SCALE, LARGEST_SCALE = 3, 246
CODES = np.arange(128)
MAGNITUDES = np.where(CODES < 8, CODES / 512.0, 2.0 ** (CODES // 8 - 7.0) * (1 + CODES % 8 / 8.0))
MAGNITUDES[127] = np.nan


def blocks_of(inner):
    return -(-inner // BLOCK)


def scale_stride(inner):
    return -(-blocks_of(inner) // 4) * 4


def quantize(rows):
    """[rows][inner] floats -> codes [rows][blocks * 128] and scales [rows][blocks, to fours], uint8."""
    rows = np.asarray(rows, np.float32)
    count, inner = rows.shape
    padded = np.zeros((count, blocks_of(inner) * BLOCK), np.float32)
    padded[:, :inner] = rows
    v = padded.reshape(count, -1, BLOCK).astype(np.float64)
    magnitude = np.abs(v)
    bad = ~np.isfinite(v).all(-1)
    with np.errstate(invalid="ignore"):
        largest = np.where(bad, 0, magnitude.max(-1))
        # Binades by comparison: the smallest power of two of which the largest is at most 464.
        factors = 2.0 ** np.arange(-124.0, 120.0)
        at = np.minimum(np.searchsorted(464 * factors, largest), len(factors) - 1)  # first of 464 f >= largest
    scales = np.where(bad, 255, at + LEAST_SCALE).astype(np.uint8)
    a = np.where(bad[..., None], 0, magnitude) / factors[at][..., None]
    # The nearest code: the first whose middle with the next is not below, ties to the even one.
    middles = (MAGNITUDES[:126] + MAGNITUDES[1:127]) / 2
    low = np.searchsorted(middles, a, side="left")      # ties stay with the lower code
    high = np.searchsorted(middles, a, side="right")    # ties go to the upper code
    code = np.where(low % 2 == 0, low, high)
    code = np.where(bad[..., None], 0, code + 128 * np.signbit(v)).astype(np.uint8)
    stored = np.zeros((count, scale_stride(inner)), np.uint8)
    stored[:, :scales.shape[1]] = scales
    return code.reshape(count, -1), stored


def factors_of(scales):
    s = np.maximum(np.asarray(scales).astype(np.float64), LEAST_SCALE)
    return np.where(np.asarray(scales) > LARGEST_SCALE, np.nan, 2.0 ** (s - 127))


def dequantize(codes, scales, inner=None):
    """The values, float64, [rows][blocks * 128] (the first `inner` of a row)."""
    codes = np.asarray(codes)
    values = np.where(codes >= 128, -1.0, 1.0) * MAGNITUDES[codes & 127]
    factors = np.repeat(factors_of(scales)[..., :codes.shape[-1] // BLOCK], BLOCK, -1)
    values = values * factors
    return values if inner is None else values[..., :inner]
