"""Definitions in float64, on the CPU, of an 8-bit cache's rows and of the edits of
logits, and the error that the kernels may make, derived from their arithmetic."""

import math

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def nearest(u, codes):
    """The code nearest to u, even where two are as near, as a float64 value."""
    if codes == torch.int8:
        return torch.round(u)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(u / step) * step).clamp(-448.0, 448.0)


def half_step(u, codes):
    """The furthest that a value of magnitude u (in codes) is from the nearest code."""
    if codes == torch.int8:
        return torch.full_like(u, 0.5)
    return torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 4)


def values(cache_k, scale):
    """Rows that codes and scales stand for, float64."""
    return cache_k.double() * scale.double()[..., None]


def check_row(code, scale, y, slack, codes):
    """A stored row (code values, scale; float64) of y [.., dim] that the kernel has
    within `slack` of y: the scale is the row's, the codes are those of a row within
    that distance."""
    top = y.abs().amax(-1, keepdim=True)
    off = slack.amax(-1, keepdim=True)
    assert bool(((scale[..., None] - top / LARGEST[codes]).abs() <= off / LARGEST[codes] + 2.0 ** -23 * scale[..., None]).all())
    # quotient y M / a: y and a off by the slack, three roundings
    u = y * LARGEST[codes] / top
    d = slack * LARGEST[codes] / top + u.abs() * (off / top) * 1.01 + 4 * 2.0 ** -24 * u.abs()
    assert bool(((code >= nearest(u - d, codes)) & (code <= nearest(u + d, codes))).all())


def edit(x, history, prompt, repetition, presence, frequency, biases, allowed):
    """(row, sum of the magnitudes that went into each element): x float64 [vocab];
    history a list of tokens, the first `prompt` of them the prompt; biases a list of
    (token, value); allowed: bool [vocab] or None."""
    x = x.clone()
    mag = x.abs()
    vocab = len(x)
    seen = {t for t in history if 0 <= t < vocab}
    count = {}
    for t in history[max(0, prompt):]:
        if 0 <= t < vocab:
            count[t] = count.get(t, 0) + 1
    for t in seen:
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
        mag[t] = max(float(mag[t]), abs(float(x[t])))
    for t, c in count.items():
        x[t] -= frequency * c + presence
        mag[t] += abs(frequency * c) + abs(presence)
    for t, b in dict(biases).items():
        if 0 <= t < vocab:
            x[t] += b
            mag[t] += abs(b)
    if allowed is not None:
        x[~allowed] = -math.inf
    return x, mag
