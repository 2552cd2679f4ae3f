"""Plain 64-bit definitions of the packed operators, with the error that rounding may leave.

``eps`` below is the unit roundoff of the tensors' type: a rounding is off by at most ``eps`` of the
value, or, below the type's smallest normal number, by half of its constant spacing, which is ``eps``
of that number (2^-25 in fp16).  32-bit arithmetic adds less than ``SLACK`` of the same sums (accumulations of up to a few
thousand terms at 2^-24 each, the exponential's and the scores' last bits).
"""

import math

import torch

SLACK = 1e-4


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return unit(dtype) * torch.finfo(dtype).smallest_normal


def rotary(x, positions, inverse, amplitude=1.0, axis=None, interleaved=False):
    """(turned in FP64, bound of the error of a 32-bit turn rounded once to ``x.dtype``)."""
    slots = inverse.numel()
    where = positions.double().unsqueeze(-1) if axis is None else positions.double()[..., axis.long()]
    angle = (where * inverse).unsqueeze(-2)
    j = torch.arange(slots, device=x.device)
    first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + slots)
    out = x.double().clone()
    a, b = x.double()[..., first], x.double()[..., second]
    out[..., first] = amplitude * (a * torch.cos(angle) - b * torch.sin(angle))
    out[..., second] = amplitude * (a * torch.sin(angle) + b * torch.cos(angle))
    # The fraction of a turn is off by 2^-26 in 32 bits, 2 pi times that as an angle; sine and cosine
    # by at most 2 units of 2^-24, amplitude, product and sum by one each: 10 units in all.
    size = torch.zeros_like(out)
    size[..., first] = size[..., second] = a.abs() + b.abs()
    bound = unit(x.dtype) * out.abs() + tiny(x.dtype) + 10 * 2.0 ** -24 * amplitude * size
    if x.dtype == torch.float32:  # the rounding to the type is the sum's own, counted above
        bound = 10 * 2.0 ** -24 * amplitude * size
    return out, bound


def attention(q, k, v, spans, scale, grad=None):
    """``spans``: (first query row, rows, first key row, keys) of every sequence.

    Returns ``{"out": (value, bound), ...}`` with ``dq``, ``dk``, ``dv`` where ``grad`` is given.
    The kernels round p and ds to the type before a product, and every result once; delta is taken
    from the rounded out.
    """
    eps, group, least = unit(q.dtype), q.shape[1] // k.shape[1], tiny(q.dtype)

    def zeros(t):
        return torch.zeros(t.shape, dtype=torch.float64, device=t.device)

    res = {"out": (zeros(q), zeros(q))}
    if grad is not None:
        res.update(dq=(zeros(q), zeros(q)), dk=(zeros(k), zeros(k)), dv=(zeros(v), zeros(v)))
    for q0, rows, k0, keys in spans:
        if rows == 0 or keys == 0:
            continue
        seen = torch.arange(keys, device=q.device)[None] <= torch.arange(rows, device=q.device)[:, None] + keys - rows
        some = seen.any(-1)
        for h in range(q.shape[1]):
            g = h // group
            Q, K, V = q[q0:q0 + rows, h].double(), k[k0:k0 + keys, g].double(), v[k0:k0 + keys, g].double()
            s = (Q @ K.t() * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            p[~some] = 0
            o = p @ V
            # p is rounded before it is divided by its sum, which is at least 1
            o_err = (eps + SLACK) * (p @ V.abs()) + eps * o.abs() + least * (1 + seen.double() @ V.abs())
            res["out"][0][q0:q0 + rows, h] = o
            res["out"][1][q0:q0 + rows, h] = o_err
            if grad is None:
                continue
            dO = grad[q0:q0 + rows, h].double()
            delta = (dO * o).sum(-1, keepdim=True)
            ds = p * (dO @ V.t() - delta)
            size = p * (dO.abs() @ V.abs().t() + (dO * o).abs().sum(-1, keepdim=True))
            ds_err = eps * ds.abs() + least * seen + p * (dO.abs() * o_err).sum(-1, keepdim=True) + SLACK * size
            rows_, keys_ = slice(q0, q0 + rows), slice(k0, k0 + keys)
            for name, at, head, value, error in (
                    ("dq", rows_, h, scale * ds @ K, scale * ds_err @ K.abs()),
                    ("dk", keys_, g, scale * ds.t() @ Q, scale * ds_err.t() @ Q.abs()),
                    ("dv", keys_, g, p.t() @ dO, ((eps + SLACK) * p + least * seen).t() @ dO.abs())):
                res[name][0][at, head] += value
                res[name][1][at, head] += error
    for name, (value, bound) in res.items():
        if name != "out":
            bound += eps * value.abs() + least * (bound > 0)
    return res


def assert_close(actual, value, bound, name=""):
    off = (actual.double() - value).abs()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert torch.isfinite(actual).all(), f"{name}: not finite"
    assert worst <= 0, f"{name}: {worst:.3g} beyond its bound (largest error {off.max().item():.3g})"
