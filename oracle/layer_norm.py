"""Layer norm and its gradients from the formulas, in 64 bits (numpy)."""

import numpy as np


def forward(h, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) of rows h [M, N]."""
    h = np.asarray(h, np.float64)
    mean = h.mean(1)
    d = h - mean[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        rstd = 1.0 / np.sqrt((d * d).mean(1) + eps)
        y = d * rstd[:, None]
    if weight is not None:
        y = y * np.asarray(weight, np.float64)
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
    return y, mean, rstd


def backward(dy, h, weight, mean, rstd, dsum=None):
    """(dx, dweight, dbias) for gradients dy of y, dsum of h."""
    dy, h = np.asarray(dy, np.float64), np.asarray(h, np.float64)
    rstd = np.asarray(rstd, np.float64)[:, None]
    xhat = (h - np.asarray(mean, np.float64)[:, None]) * rstd
    a = dy if weight is None else dy * np.asarray(weight, np.float64)
    dx = rstd * (a - a.mean(1, keepdims=True) - xhat * (a * xhat).mean(1, keepdims=True))
    if dsum is not None:
        dx = dx + np.asarray(dsum, np.float64)
    return dx, (dy * xhat).sum(0), dy.sum(0)
