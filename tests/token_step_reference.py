"""Plain 64-bit restatements of the token-step operators (rotary positions, KV append, sampling), and the
tolerances the tests hold the kernels to."""
from __future__ import annotations

import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def host(t) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


# --------------------------------------------------------------------------- rotary positions

def rope(x, positions, theta, interleaved=False, adjoint=False, magnitude=1.0):
    """x [B, S, H, D] (float64), positions [B, S], theta [R/2] -> (y, sum of the magnitudes each y adds up).
    The angles are formed in extended precision."""
    half = len(theta)
    phi = positions.astype(np.longdouble)[:, :, None] * theta.astype(np.longdouble)
    cos = np.cos(phi).astype(np.float64)[:, :, None, :]
    sin = np.sin(phi).astype(np.float64)[:, :, None, :] * (-1.0 if adjoint else 1.0)
    y, size = x.copy(), np.zeros_like(x)
    first = (Ellipsis, slice(0, 2 * half, 2)) if interleaved else (Ellipsis, slice(0, half))
    second = (Ellipsis, slice(1, 2 * half, 2)) if interleaved else (Ellipsis, slice(half, 2 * half))
    y[first] = magnitude * (x[first] * cos - x[second] * sin)
    y[second] = magnitude * (x[first] * sin + x[second] * cos)
    size[first] = size[second] = abs(magnitude) * (np.abs(x[first]) + np.abs(x[second]))
    return y, size


def rope_tolerance(want, size, dtype, largest_angle=0.0):
    """Sine and cosine: the F32 rounding of the fraction of a turn moves the angle by (pi/2) 2^-26 at most, the
    polynomials add their coefficients' and last step's roundings, 2^-23 in all; the magnitude, the two products
    and their sum round by 2^-24 each, so 2^-22 of |x1| + |x2| bounds the F32 value.  The 64-bit phase is 2^-52
    of the angle off, twice rounded.  Then half a step of the stored type."""
    half_step = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half the spacing of F16's subnormal values
    return size * (2.0 ** -22 + 2.0 ** -51 * largest_angle) + half_step * np.abs(want) * 1.01 + tiny


def assert_rope(got, want, size, dtype, largest_angle=0.0, what=""):
    err = np.abs(host(got) - want)
    tol = rope_tolerance(want, size, dtype, largest_angle)
    assert np.all(err <= tol), f"{what}: {int(np.sum(err > tol))} values off, worst {np.max(err - tol)}"


# --------------------------------------------------------------------------- sampling

def penalised(logits, recent=None, penalty=1.0, limit=0, ignore=None, streams=0):
    """F32 logits after the repetition penalty (F32 division) and the ignore list."""
    x = logits.detach().cpu().float().numpy().copy()
    rows, vocab = x.shape
    limit = vocab if limit <= 0 else min(limit, vocab)
    for r in range(rows):
        if recent is not None:
            ids = np.unique(np.asarray(recent[r]))
            ids = ids[(ids >= 0) & (ids < limit)]
            x[r, ids] = x[r, ids] / np.float32(penalty)
        if ignore is not None and (r % streams == 0 if streams > 0 else r == 0):
            ids = np.asarray(ignore)
            x[r, ids[(ids >= 0) & (ids < vocab)]] = -np.inf
    return x


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition for one row of F32 logits: (token, log of its share, its weight, the weight of what stayed,
    how near the uniform number comes to a border of its interval); None for a row without a token of weight."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return None
    order = np.argsort(-x, kind="stable")
    if temperature == 0:
        order = order[:1]
    if top_k > 0:
        order = order[:top_k]
    v = x[order].astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(v == top, 1.0, np.exp((v - float(top)) / (temperature or 1.0)))
    w[v == -np.inf] = 0.0
    w = np.rint(w * 2.0 ** 44) / 2.0 ** 44  # the documented unit: what is below half of it has no weight
    keep = np.ones(len(w), bool)
    if top_p < 1:
        keep = np.cumsum(w) - w < float(np.float32(top_p)) * w.sum()
    keep &= w >= float(np.float32(min_p))
    keep[0] = True
    keep &= w > 0
    w = w[:keep.sum()]  # the three conditions keep a prefix
    upto = np.cumsum(w)
    at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), len(w) - 1)
    near = np.min(np.abs(upto[:-1] - u * upto[-1])) / upto[-1] if len(w) > 1 else 1.0
    return int(order[at]), math.log(w[at] / upto[-1]), w[at], upto[-1], near


def logprob_tolerance(logprob, weight, total, vocab):
    """Each weight within one unit of 2^-44 of the reference's (both round an F64 exponential, good to 2^-42 of
    itself, and may round to neighbours), the logarithm rounded to F32."""
    return 2.0 ** -24 * abs(logprob) + 2.0 ** -44 / weight + vocab * 2.0 ** -44 / total + 2.0 ** -41
