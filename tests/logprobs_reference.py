"""Log probabilities, entropies, the likeliest classes and the gradient (include/staleynet_logprobs.h) in numpy and 64
bits, from their definition."""
import numpy as np

EMPTY = 0xFFFFFFFF


def forward(z, tokens=None, scale=1.0, top=0):
    """z [rows][heads][classes] -> logprobs, entropies, stats, top classes, top log probabilities."""
    x = np.asarray(z, np.float64)
    classes = x.shape[-1]
    with np.errstate(all="ignore"):
        m = np.where(np.isnan(x).any(-1), np.nan, x.max(-1))
        m = np.where(np.isfinite(m), m, np.nan)
        shifted = (x - m[..., None]) * float(scale)
        p = np.exp(shifted)
        at = shifted.argmax(-1)[..., None]
        others = p.copy()
        np.put_along_axis(others, at, 0.0, -1)
        log_total = np.log1p(others.sum(-1))
        log_p = shifted - log_total[..., None]
        weighted = np.where(p > 0, p * -shifted, 0.0).sum(-1)
        entropies = log_total + weighted / p.sum(-1)
        logprobs = None
        if tokens is not None:
            t = np.asarray(tokens, np.uint32)
            inside = t < classes
            picked = np.take_along_axis(log_p, np.where(inside, t, 0).astype(np.int64)[..., None], -1)[..., 0]
            logprobs = np.where(t == EMPTY, 0.0, np.where(inside, picked, np.nan))
    key = np.where(np.isnan(x), np.inf, x)
    order = np.lexsort((np.broadcast_to(np.arange(classes), x.shape), -key, ~np.isnan(x)), axis=-1)[..., :top]
    ids = np.full(x.shape[:-1] + (top,), EMPTY, np.uint32)
    listed = np.full(ids.shape, -np.inf)
    ids[..., :order.shape[-1]] = order
    listed[..., :order.shape[-1]] = np.take_along_axis(log_p, order, -1)
    return logprobs, entropies, np.stack([m, log_total], -1), ids, listed


def backward(z, stats, entropies, tokens=None, d_logprobs=None, d_entropies=None, scale=1.0):
    x, stats = np.asarray(z, np.float64), np.asarray(stats, np.float64)
    with np.errstate(all="ignore"):
        log_p = (x - stats[..., :1]) * float(scale) - stats[..., 1:]
        p = np.exp(log_p)
        grad = np.zeros(x.shape)
        if d_logprobs is not None:
            t = np.asarray(tokens, np.uint32)[..., None]
            d = np.where(t == EMPTY, 0.0, np.asarray(d_logprobs, np.float64)[..., None])
            grad = grad + d * ((np.arange(x.shape[-1]) == t) - p)
        if d_entropies is not None:
            h = np.asarray(entropies, np.float64)[..., None]
            grad = grad - np.asarray(d_entropies, np.float64)[..., None] * np.where(p > 0, p * (log_p + h), p * 0)
    return grad * float(scale)
