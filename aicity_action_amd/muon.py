"""Orthogonalised updates for weight matrices: Newton-Schulz products and the Muon step, on csrc/newton_schulz.hip.

``orthogonalize`` pushes the singular values of matrices to about one; ``MuonMatrices`` renews the momenta of a set of weights and steps
each weight by its orthogonalised momentum, all matrices in the same launches whatever their sizes (one for a set of small ones, else 17 or a
few more; matrices of few rows or columns run ahead of larger ones).  ``solver.construct_optimizer`` builds a train step on it
(``SOLVER.OPTIMIZING_METHOD muon``); the reference's own methods are those of slowfast/models/optimizer.py:140-206.
Everything runs on the tensors' device and its current stream; there is no CPU fallback."""
import bisect
import functools
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _hip

QUINTIC = (3.4445, -4.7750, 2.0315)       # a, b, c of X <- a X + (b A + c A A) X: steep at zero, between 0.68 and 1.21 from 0.1 on after five steps
_REC = np.dtype([("u", "u8"), ("w", "u8"), ("m", "u8"), ("out", "u8"), ("rs", "i8"), ("cs", "i8"), ("rows", "i4"), ("cols", "i4"),
                 ("scale", "f4"), ("pad", "i4")])
_ROOM = 15.0                  # X, A and B are fp16 values times 2^12: 65504 / 4096, less a margin for their rounding
_ARITHMETIC = {"fp16": 0, "split": 1}


@functools.lru_cache(maxsize=64)
def _largest(steps, a, b, c):
    """The largest value that X, A or B can hold while ``steps`` are taken: no entry is larger than the largest singular value, those of X_0 are at
    most one, and every step is one polynomial of each.  (The last X is the result and not held.)"""
    top, most = 1.0, 1.0
    for _ in range(steps):
        t = top * top
        vertex = [-b / (2 * c)] if c else []
        disc = 9 * b * b - 20 * a * c
        ends = [(-3 * b + s * math.sqrt(disc)) / (10 * c) for s in (-1, 1)] if c and disc >= 0 else [-a / (3 * b)] if b and not c else []
        inside = lambda points: [p for p in points if 0 < p < t] + [t]  # noqa: E731
        most = max(most, top, t, max(abs(b * p + c * p * p) for p in inside(vertex)))
        top = max(abs(math.sqrt(p) * (a + b * p + c * p * p)) for p in inside(ends))
        if not most < _ROOM:
            break
    return most


def _check_iteration(steps, coefficients, eps, arithmetic):
    if not 1 <= int(steps) <= 100:
        raise ValueError("Newton-Schulz: 1 to 100 steps, got %r" % (steps,))
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError("Newton-Schulz: three finite coefficients, got %r" % (coefficients,))
    if not _largest(int(steps), *coefficients) < _ROOM:
        raise ValueError("Newton-Schulz: coefficients %r grow values of %.3g in %d steps, and the products hold up to %g"
                         % (tuple(coefficients), _largest(int(steps), *coefficients), steps, _ROOM))
    if not (math.isfinite(eps) and eps > 0.0):
        raise ValueError("Newton-Schulz: eps must be positive, got %r" % (eps,))
    if arithmetic not in _ARITHMETIC:
        raise ValueError("Newton-Schulz: arithmetic must be 'fp16' or 'split', got %r" % (arithmetic,))


def _library(half):
    return _hip.lib_with_record(half, "mvit_ns_matrix_bytes", _REC.itemsize)


def _workspace(L, rec, split, device):
    n = L.mvit_newton_schulz_workspace_bytes(rec.ctypes.data, len(rec), split)
    _hip.check(min(int(n), 0), "newton_schulz (sizes)")
    # from torch's allocator, per call: ordered with the stream, and a captured call owns its own
    return torch.empty(int(n), dtype=torch.uint8, device=device), int(n)


def orthogonalize(update, steps=5, coefficients=QUINTIC, eps=1e-7, dtype=torch.bfloat16, arithmetic=None):
    """Newton-Schulz orthogonalisation of one matrix, a batch [..., rows, columns] or a list of either (sizes may differ; one set of
    launches for all).  float32 / bfloat16 / float16, any strides.  Returns contiguous tensors of ``dtype``.  Coefficients under which a singular
    value or its polynomial would reach 15 on the way are refused.

    ``arithmetic``: "fp16" (default for 16-bit results) computes the products from fp16 operands, which leaves the result within 3e-3 of the
    exact one relative to its norm (five steps, these coefficients; about 1.4e-3 from a hundred rows on).  "split" (default for float32) computes them
    from pairs of fp16 values at three times the work: within 1e-4, and 1e-5 unless one direction of the update dominates all others.
    Matrices of at most 32 rows or columns always take pairs, whatever they stand beside.  A matrix of zeros stays zero; one with NaN or
    infinity gives NaN.  A matrix' last bits depend on the call it is in (which order its sums are taken in)."""
    many = isinstance(update, (list, tuple))
    ts = list(update) if many else [update]
    if arithmetic is None:
        arithmetic = "split" if dtype == torch.float32 else "fp16"
    _check_iteration(steps, coefficients, eps, arithmetic)
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("orthogonalize: dtype must be float32, bfloat16 or float16, got %s" % dtype)
    if not ts:
        return []
    for t in ts:
        if t.dim() < 2:
            raise ValueError("orthogonalize: matrices [..., rows, columns], got %s" % (tuple(t.shape),))
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("orthogonalize: float32, bfloat16 or float16, got %s" % t.dtype)
        if t.dtype != ts[0].dtype or t.device != ts[0].device:
            raise ValueError("orthogonalize: all updates must have one dtype and one device")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("orthogonalize has no backward pass: call it under torch.no_grad() or on detached updates")
    if forward_ad._current_level >= 0:
        _hip.refuse_tangents("orthogonalize", *ts)
    if not ts[0].is_cuda:
        raise RuntimeError("orthogonalize needs its updates on a gfx950 device; there is no CPU fallback")
    if ts[0].dtype != torch.float32 and dtype != torch.float32 and ts[0].dtype != dtype:
        ts = [t.float() for t in ts]                # bfloat16 and float16 are different libraries
    half = torch.float16 in (ts[0].dtype, dtype)
    with torch.cuda.device(ts[0].device), torch.no_grad():
        outs = [torch.empty(t.shape, dtype=dtype, device=t.device) for t in ts]
        rows = []
        for t, o in zip(ts, outs):
            if t.numel() == 0:
                continue
            size, osize = t.element_size(), o.element_size()
            r, c = t.shape[-2:]
            for i, at in enumerate(np.ndindex(*t.shape[:-2])):
                rows.append((t.data_ptr() + size * sum(a * s for a, s in zip(at, t.stride())), 0, 0, o.data_ptr() + osize * i * r * c,
                             t.stride(-2), t.stride(-1), r, c, 0.0, 0))
        if rows:
            rec = np.array(rows, dtype=_REC)
            L = _library("fp16" if half else "bf16")
            split = _ARITHMETIC[arithmetic]
            ws, n = _workspace(L, rec, split, ts[0].device)
            code = lambda d: _hip.F32 if d == torch.float32 else _hip.BF16  # noqa: E731
            _hip.check(L.mvit_newton_schulz(rec.ctypes.data, len(rec), code(ts[0].dtype), code(dtype), *[float(v) for v in coefficients],
                                            int(steps), float(eps), split, _hip.ptr(ws), n, torch.cuda.current_stream().cuda_stream),
                       "newton_schulz")
    return outs if many else outs[0]


def _apart(written, read=()):
    """Spans (first byte, byte behind the last one): what a step writes must not overlap, nor what it reads begin or end in it."""
    written = sorted(written)
    if any(a[1] > b[0] for a, b in zip(written, written[1:])):
        raise ValueError("MuonMatrices: parameters and momenta must not share memory (the same tensor twice?)")
    ends = [b for _, b in written]
    for a, b in read:
        i = bisect.bisect_right(ends, a)                 # the first span that ends behind the gradient's beginning
        if i < len(ends) and written[i][0] < b:
            raise ValueError("MuonMatrices.step: a gradient shares its memory with a parameter or a momentum")


class MuonMatrices(object):
    """A set of weight matrices and their momenta, stepped together.

    ``step``:  M <- mu M + (1 - mu) g;  U = (1 - mu) g + mu M (Nesterov) or M;  W <- W (1 - lr weight_decay) - lr rms sqrt(max(rows,
    columns)) NS(U).  ``rms`` 0.2 gives the update the size that AdamW's typically has, so that one learning rate and weight decay serve
    both.  Weights and momenta: contiguous float32 matrices, updated in place; gradients: float32, any strides, in memory of their own.

    ``arithmetic`` of the orthogonalisation, as in ``orthogonalize``: "fp16" leaves NS(U) within 3e-3 of the exact one although everything
    around it is float32 (an update is a small part of a weight, and the iteration itself stops up to 0.3 short of orthogonal), "split" within
    1e-4 at twice the time for a whole model's matrices (0.9 -> 1.7 ms for the video model's)."""

    def __init__(self, params, momenta=None, momentum=0.95, nesterov=True, weight_decay=0.0, rms=0.2, steps=5, coefficients=QUINTIC,
                 eps=1e-7, arithmetic="fp16"):
        self.params = list(params)
        if not self.params:
            raise ValueError("MuonMatrices: no parameters")
        _check_iteration(steps, coefficients, eps, arithmetic)
        if not (weight_decay >= 0.0 and math.isfinite(weight_decay)) or not (rms > 0.0 and math.isfinite(rms)):
            raise ValueError("MuonMatrices: weight_decay must not be negative and rms must be positive")
        if momenta is not None and len(momenta) != len(self.params):
            raise ValueError("MuonMatrices: %d momenta for %d parameters" % (len(momenta), len(self.params)))
        for p in self.params:
            self._check_matrix(p, "parameter")
        self.momenta = list(momenta) if momenta is not None else [torch.zeros_like(p, requires_grad=False) for p in self.params]
        for p, m in zip(self.params, self.momenta):
            self._check_matrix(m, "momentum")
            if m.shape != p.shape:
                raise ValueError("MuonMatrices: a momentum of shape %s for a parameter of shape %s" % (tuple(m.shape), tuple(p.shape)))
        _apart((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in self.params + self.momenta)
        self.weight_decay, self.rms, self.coefficients = float(weight_decay), float(rms), tuple(float(c) for c in coefficients)
        self.eps, self.arithmetic = float(eps), arithmetic
        self.configure(momentum, nesterov, steps)

    def configure(self, momentum, nesterov, steps):
        """Takes other values for the steps to come (a loaded state's)."""
        _check_iteration(steps, self.coefficients, self.eps, self.arithmetic)
        if not 0.0 <= momentum < 1.0:
            raise ValueError("MuonMatrices: momentum must be in [0, 1), got %r" % (momentum,))
        self.momentum, self.nesterov, self.steps = float(momentum), bool(nesterov), int(steps)

    def _check_matrix(self, t, what):
        if t.dim() != 2 or t.numel() == 0:
            raise ValueError("MuonMatrices: every %s must be a matrix, got shape %s" % (what, tuple(t.shape)))
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("MuonMatrices: every %s must be contiguous float32, got %s with strides %s" % (what, t.dtype, t.stride()))
        if t.device != self.params[0].device:
            raise ValueError("MuonMatrices: parameters and momenta must be on one device")

    def step(self, grads=None, lr=None, norm_coef=None, hyper=None):
        """One step with ``grads`` (default: each parameter's ``.grad``; a parameter whose gradient is None is left as it is).

        ``norm_coef``: two floats on the device, mvit_grad_norm's [norm, factor]: gradients are multiplied by the factor, and a norm or
        factor that is not finite leaves weights and momenta as they are.  ``hyper``: device floats whose first is the learning rate, read
        by the kernels in place of ``lr`` (a captured step is replayed with new values)."""
        if (lr is None) == (hyper is None):
            raise ValueError("MuonMatrices.step: give the learning rate either as lr or in hyper")
        if lr is not None and not math.isfinite(lr):
            raise ValueError("MuonMatrices.step: lr must be finite, got %r" % (lr,))
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError("MuonMatrices.step: %d gradients for %d parameters" % (len(grads), len(self.params)))
        device, rows, touched = self.params[0].device, [], []
        for t, n, what in ((norm_coef, 2, "norm_coef"), (hyper, 1, "hyper")):
            if t is not None and (t.dtype != torch.float32 or t.numel() < n or not t.is_contiguous() or t.device != device):
                raise ValueError("MuonMatrices.step: %s must be %d contiguous float32 values or more on %s" % (what, n, device))
        if forward_ad._current_level >= 0:
            _hip.refuse_tangents("MuonMatrices.step", norm_coef, hyper, *self.params, *self.momenta, *grads)
        for p, m, g in zip(self.params, self.momenta, grads):
            if g is None:
                continue
            if (p.dtype != torch.float32 or m.dtype != torch.float32 or p.device != device or m.device != device or m.shape != p.shape
                    or not (p.is_contiguous() and m.is_contiguous())):
                raise ValueError("MuonMatrices.step: a parameter or its momentum has changed its type, device, shape or strides")
            if g.shape != p.shape or g.dtype != torch.float32 or g.device != device:
                raise ValueError("MuonMatrices.step: a %s gradient of shape %s on %s for a float32 parameter of shape %s on %s"
                                 % (g.dtype, tuple(g.shape), g.device, tuple(p.shape), device))
            r, c = p.shape
            rows.append((g.data_ptr(), p.data_ptr(), m.data_ptr(), 0, g.stride(0), g.stride(1), r, c, self.rms * math.sqrt(max(r, c)), 0))
            touched += [p, m]
        if not rows:
            return
        _apart([(at, at + 4 * r * c) for _, p, m, _, _, _, r, c, _, _ in rows for at in (p, m)],
               [(g, g + 4 * (1 + (r - 1) * rs + (c - 1) * cs)) for g, _, _, _, rs, cs, r, c, _, _ in rows])
        if not self.params[0].is_cuda:
            raise RuntimeError("MuonMatrices needs its parameters on a gfx950 device; there is no CPU fallback")
        rec = np.array(rows, dtype=_REC)
        L, split = _library("bf16"), _ARITHMETIC[self.arithmetic]
        with torch.cuda.device(device):
            ws, n = _workspace(L, rec, split, device)
            _hip.check(L.mvit_muon_step(rec.ctypes.data, len(rec), float(lr or 0.0), self.weight_decay, self.momentum, int(self.nesterov),
                                        *self.coefficients, self.steps, self.eps, split, _hip.ptr(norm_coef), _hip.ptr(hyper), _hip.ptr(ws), n,
                                        torch.cuda.current_stream().cuda_stream), "muon_step")
        # written behind torch's back: whatever is cached by version (16-bit weight copies) is refreshed on its next use
        for t in touched:
            torch.autograd.graph.increment_version(t)
