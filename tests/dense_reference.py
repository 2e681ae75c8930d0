"""The dense operators by index in 64 bits, from their definitions, and how far a sum in 32 bits may be off."""
import importlib

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS32 = 2.0 ** -24                                     # half a step, relative to the value
# half the smallest step of values near zero
FLOOR = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def ops_of(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def rounding(dtype, value):
    """Of one rounding of `value` to dtype."""
    return torch.finfo(dtype).eps / 2 * value.abs() + FLOOR[dtype]


def outside(got, want, tol):
    """How many values differ by more than `tol`, where infinities and NaN have to be the same."""
    got = got.double()
    bad = (got - want).abs() > tol
    fine = torch.isfinite(want)
    bad = torch.where(fine, bad | ~torch.isfinite(got), ~((got == want) | (torch.isnan(got) & torch.isnan(want))))
    return int(bad.sum())


def embedding(ids, table, scale):
    """(value, tolerance): one product in 32 bits, one rounding."""
    t = table.double()
    held = (ids >= 0) & (ids < t.shape[0])
    out = torch.zeros((*ids.shape, t.shape[1]), dtype=torch.float64, device=table.device)
    out[held] = t[ids[held].long()] * scale
    return out, rounding(table.dtype, out) * (1 + 2.0 ** -8) + EPS32 * out.abs()


def embedding_grad(ids, dout, rows, scale):
    """n additions and a product in 32 bits, one rounding."""
    held = (ids >= 0) & (ids < rows)
    at, d = ids[held].long(), dout[held].double()
    zero = torch.zeros((rows, dout.shape[-1]), dtype=torch.float64, device=dout.device)
    value = zero.index_add(0, at, d) * scale
    size = zero.index_add(0, at, d.abs()) * abs(scale)
    n = torch.bincount(at, minlength=rows)[:, None].double()
    return value, rounding(dout.dtype, value) * (1 + 2.0 ** -8) + (n + 1) * EPS32 * size


def _parts(offsets, rows):
    b = offsets.tolist()
    return [(g, s, e) for g, (s, e) in enumerate(zip(b, b[1:])) if e > s]


def _sum_tolerance(dtype, value, size, terms):
    # tensor cores may cut a term where an addition in 32 bits would round it: a whole step for each term
    return rounding(dtype, value) * (1 + 2.0 ** -8) + (terms + 2) * 2 * EPS32 * size


def grouped(X, W, offsets):
    x, w = X.double(), W.double()
    value = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device=X.device)
    size = torch.zeros_like(value)
    for g, s, e in _parts(offsets, x.shape[0]):
        value[s:e] = x[s:e] @ w[g]
        size[s:e] = x[s:e].abs() @ w[g].abs()
    return value, _sum_tolerance(X.dtype, value, size, x.shape[1])


def grouped_weight(X, dY, offsets):
    x, y = X.double(), dY.double()
    value = torch.zeros((offsets.numel() - 1, x.shape[1], y.shape[1]), dtype=torch.float64, device=X.device)
    tol = torch.zeros_like(value)
    for g, s, e in _parts(offsets, x.shape[0]):
        value[g] = x[s:e].T @ y[s:e]
        tol[g] = _sum_tolerance(X.dtype, value[g], x[s:e].T.abs() @ y[s:e].abs(), e - s)
    return value, tol


def _teacher(logits, ids, teacher, tau):
    """p, log p (0 where p is 0) and ids taken into the row."""
    t = teacher.double() / tau
    held = (ids >= 0) & (ids < logits.shape[-1]) & (teacher > -float("inf"))
    t = t.masked_fill(~held, -float("inf"))
    some = held.any(-1, keepdim=True)
    logp = torch.log_softmax(t.masked_fill(~some, 0.0), -1)
    p = torch.where(some & held, torch.exp(logp), 0.0)
    return p, torch.where(p > 0, logp, 0.0), torch.where(held, ids, 0).long(), some


def _share(columns):
    # of the sum over a row: ex2 is within 2^-22, the exponents within two roundings of values that weigh about log(V) in
    # the mean (2^-19 covers both), and the sum adds up `columns` / 256 terms in a thread, then 256 threads
    return (columns / 256 + 32) * EPS32 + 2.0 ** -19


def distill(logits, ids, teacher, tau):
    z = logits.double() / tau
    p, logp, at, some = _teacher(logits, ids, teacher, tau)
    logq = torch.log_softmax(z, -1).gather(-1, at)
    value = tau ** 2 * torch.where(p > 0, p * (logp - logq), 0.0).sum(-1)
    size = torch.where(p > 0, p * (logp.abs() + logq.abs()), 0.0).sum(-1)
    return value, tau ** 2 * (2 * _share(logits.shape[-1]) + 2.0 ** -20 * size)


def distill_grad(logits, ids, teacher, tau, dloss):
    z = logits.double() / tau
    p, _, at, some = _teacher(logits, ids, teacher, tau)
    q = torch.softmax(z, -1) * some
    q = torch.where(some, q, 0.0)
    named = torch.zeros_like(z).scatter_add_(-1, at, p)
    g = (dloss.double() * tau)[..., None]
    value = torch.where(some, g * (q - named), 0.0)
    # A single value of q or p is exp(-x) with x = (largest - it) / tau in three roundings (difference, log2(e) / tau,
    # product), so 3 x 2^-24 relative to it.  At tau = 0.05 and x = 100 that is 1.8e-5, nine times the 2^-19 that suffices
    # for sums, whose terms of large x weigh nothing.
    depth = 3 * EPS32 * (z.amax(-1, keepdim=True) - z)
    t = torch.where(p > 0, -torch.log(p), 0.0)
    named_off = torch.zeros_like(z).scatter_add_(-1, at, p * 3 * EPS32 * t)
    # (exponentials below the smallest normal number, 2^-126, count as 0: one in q, some in p)
    off = (1 + at.shape[-1]) * 2.0 ** -126 + (q + named) * 2 * _share(logits.shape[-1]) + torch.where(q > 0, q * depth, 0.0) + named_off
    tol = rounding(logits.dtype, value) * (1 + 2.0 ** -8) + g.abs() * off
    return value, tol
