"""Rotary positions with several axes (time, height, width) for the queries and keys of video and image tokens.

The reference model knows positions from the learned embeddings of its stem alone (slowfast/models/video_model_builder.py:1196-1223); a
rotary position instead turns pairs of channels of every query and key by an angle proportional to the token's place on one axis, so
that scores depend on differences of places and a model meets other grid sizes without interpolated tables.  ``HIP.ROTARY`` turns it on
in the model (models/mvit.py); this module is the operator itself::

    rot = AxialRotary(96)                                            # 32 channels for each of t, h, w
    q, k = rot(q, TokenGrid((8, 28, 28)), k, TokenGrid((8, 14, 14), step=(1, 2, 2)))

One kernel launch (csrc/rotary.hip) serves both tensors in each direction, on the tensors' device and its current stream; there is no
CPU fallback.
"""
import ctypes
import math
import struct

import torch
from torch.autograd import forward_ad

from . import _hip

_MAX_AXES, _MAX_PAIRS = 4, 256
_POS = {torch.int32: 1, torch.int64: 2, torch.float32: 3}
_LAYOUTS = {"half": 0, "interleaved": 1}
_RECORD = struct.Struct("@4P12qq3i4i8d")        # mvit_rotary_tensor of include/mvit_hip.h
_NO_GRID = (0,) * 4 + (0.0,) * 8


class TokenGrid(object):
    """Tokens in order on a grid, the last axis fastest (the model's token order: t, h, w).  Token (i_0, i_1, ...) stands at
    ``origin + step * i`` on each axis: keys pooled with stride s stand at every s-th place of the queries' grid (``step=(1, s, s)``)."""

    def __init__(self, sizes, step=None, origin=None):
        self.sizes = tuple(int(n) for n in sizes)
        self.step = tuple(float(s) for s in step) if step is not None else (1.0,) * len(self.sizes)
        self.origin = tuple(float(s) for s in origin) if origin is not None else (0.0,) * len(self.sizes)
        if not 1 <= len(self.sizes) <= _MAX_AXES or any(n < 1 or n >= 1 << 31 for n in self.sizes):
            raise ValueError("TokenGrid: 1 to %d axes of at least one token each, got %s" % (_MAX_AXES, self.sizes))
        if len(self.step) != len(self.sizes) or len(self.origin) != len(self.sizes):
            raise ValueError("TokenGrid: step and origin need one value for each of the %d axes" % len(self.sizes))
        if not all(math.isfinite(v) for v in self.step + self.origin):
            raise ValueError("TokenGrid: step and origin must be finite")
        self.tokens = math.prod(self.sizes)
        fill = lambda v, x: v + (x,) * (4 - len(v))  # noqa: E731
        self.record = fill(self.sizes, 0) + fill(self.origin, 0.0) + fill(self.step, 0.0)      # as in mvit_rotary_tensor

    def __repr__(self):
        return "TokenGrid(%s, step=%s, origin=%s)" % (self.sizes, self.step, self.origin)


class AxialRotary(object):
    """The plan of a head: which channels turn by which axis, and how fast.

    ``sections``: channels per axis, even; default: three axes of ``head_dim // 6 * 2`` channels.  Channels behind the sections pass
    through.  Pair i of a section of s channels turns by ``place * base ** (-2 i / s)``.  ``layout``: "half" pairs channel i of a section
    with i + s / 2, "interleaved" pairs 2i with 2i + 1."""

    def __init__(self, head_dim, sections=None, base=10000.0, layout="half"):
        self.head_dim = int(head_dim)
        self.sections = tuple(int(s) for s in sections) if sections is not None else (self.head_dim // 6 * 2,) * 3
        self.base, self.layout = float(base), layout
        if layout not in _LAYOUTS:
            raise ValueError("AxialRotary: layout must be 'half' or 'interleaved', got %r" % (layout,))
        if not 1 <= len(self.sections) <= _MAX_AXES or any(s < 2 or s % 2 for s in self.sections):
            raise ValueError("AxialRotary: 1 to %d sections of an even number of channels each, got %s" % (_MAX_AXES, self.sections))
        if sum(self.sections) > self.head_dim or sum(self.sections) > 2 * _MAX_PAIRS:
            raise ValueError("AxialRotary: sections %s need more than the %d channels of a head (at most %d turn)"
                             % (self.sections, self.head_dim, 2 * _MAX_PAIRS))
        if not (math.isfinite(self.base) and self.base > 0.0):
            raise ValueError("AxialRotary: base must be positive, got %r" % (base,))
        turns = [self.base ** (-2.0 * i / s) / (2.0 * math.pi) for s in self.sections for i in range(s // 2)]
        self._turns = (ctypes.c_double * len(turns))(*turns)
        self._sections = (ctypes.c_int * len(self.sections))(*self.sections)

    def __reduce__(self):                       # (models that hold a plan are copied and pickled)
        return AxialRotary, (self.head_dim, self.sections, self.base, self.layout)

    def __call__(self, x, positions, k=None, k_positions=None):
        """Turned copies of ``x`` (and ``k``), differentiable in reverse mode (a tensor or a gradient with a forward-mode tangent is refused).
        Tensors [batch, heads, tokens, head_dim], float32 / bfloat16 / float16, any strides with contiguous channels (a token-major buffer goes
        in as its transposed view).  Positions: a TokenGrid, or a tensor [tokens, axes] or [batch, tokens, axes] of int32 / int64 / float32 on
        the same device."""
        xs, ps = self._arguments(x, positions, k, k_positions)
        if torch.is_grad_enabled() and any(t.requires_grad for t in xs):
            held = [_leaf_on_one_stream(t) for t in xs]
            ys = _RotaryFn.apply(self, ps, False, *xs)
            del held                                # the graph holds the nodes now
        else:
            ys = self.turn(xs, ps)
        return tuple(ys) if k is not None else ys[0]

    def rotate_(self, x, positions, k=None, k_positions=None, inverse=False):
        """The same in place, without a graph (serving: queries and keys are turned where they stand, heads of one fused buffer for instance;
        they must not overlap each other, nor a tensor itself)."""
        xs, ps = self._arguments(x, positions, k, k_positions)
        for t in xs:
            if torch.is_grad_enabled() and t.requires_grad:
                raise RuntimeError("AxialRotary.rotate_: the tensor requires a gradient; use the plan's call, which makes a turned copy")
            if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
                raise ValueError("AxialRotary.rotate_: an expanded tensor (stride 0) cannot be turned in place")
        self.turn(xs, ps, outs=xs, inverse=inverse)
        for t in xs:                    # written behind torch's back
            torch.autograd.graph.increment_version(t)
        return tuple(xs) if k is not None else x

    # ---- checks ----------------------------------------------------------------------------------------------------------------------
    def _arguments(self, x, positions, k, k_positions):
        if (k is None) != (k_positions is None):
            raise ValueError("AxialRotary: k and k_positions go together")
        xs, ps = ([x], [positions]) if k is None else ([x, k], [positions, k_positions])
        for t, p in zip(xs, ps):
            self._check(t, p)
            if t.dtype != x.dtype or t.device != x.device:
                raise ValueError("AxialRotary: x and k must have one dtype and one device, got %s on %s and %s on %s"
                                 % (x.dtype, x.device, t.dtype, t.device))
        return xs, ps

    def _check(self, t, p):
        if forward_ad._current_level >= 0:      # (within a dual level)
            _hip.refuse_tangents("AxialRotary", t, p if isinstance(p, torch.Tensor) else None)
        if t.dim() != 4 or t.shape[3] != self.head_dim:
            raise ValueError("AxialRotary: expected [batch, heads, tokens, %d], got %s" % (self.head_dim, tuple(t.shape)))
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("AxialRotary: float32, bfloat16 or float16, got %s" % t.dtype)
        if t.stride(3) != 1:
            raise ValueError("AxialRotary: the channels of a head must be contiguous (stride %d)" % t.stride(3))
        if isinstance(p, TokenGrid):
            if len(p.sizes) != len(self.sections) or p.tokens != t.shape[2]:
                raise ValueError("AxialRotary: %r does not describe %d tokens on %d axes" % (p, t.shape[2], len(self.sections)))
        elif isinstance(p, torch.Tensor):
            if p.dtype not in _POS:
                raise TypeError("AxialRotary: positions must be int32, int64 or float32, got %s" % p.dtype)
            want = (t.shape[2], len(self.sections))
            if tuple(p.shape) != want and tuple(p.shape) not in ((t.shape[0],) + want, (1,) + want):
                raise ValueError("AxialRotary: positions must be [%d, %d] or [%d, %d, %d], got %s" % (want + (t.shape[0],) + want + (tuple(p.shape),)))
            if p.requires_grad:
                raise ValueError("AxialRotary: positions carry no gradient; detach them")
            if p.device != t.device:
                raise ValueError("AxialRotary: positions on %s, the tensor on %s" % (p.device, t.device))
        else:
            raise TypeError("AxialRotary: positions must be a TokenGrid or a tensor, got %s" % type(p).__name__)
        if not t.is_cuda:
            raise RuntimeError("AxialRotary needs its tensors on a gfx950 device; there is no CPU fallback")

    # ---- the launch --------------------------------------------------------------------------------------------------------------------
    def turn(self, xs, ps, outs=None, adds=None, inverse=False):
        """One launch over one or two checked tensors: outs[i] = rot(xs[i]) (+ adds[i]); fresh outputs where ``outs`` is None."""
        if outs is None:
            outs = [torch.empty_like(t) for t in xs]
            outs = [y if y.stride(3) == 1 else torch.empty(y.shape, dtype=y.dtype, device=y.device) for y in outs]
        _launch(xs, outs, adds, ps, self.head_dim, len(self.sections), self._sections, self._turns, _LAYOUTS[self.layout], inverse)
        return list(outs)


def add_(out, add, x=None):
    """out = (x or out) + add for [batch, heads, tokens, channels] views of any strides with contiguous channels: the rotary kernel with no
    axis."""
    _launch([out if x is None else x], [out], [add], [None], out.shape[3], 0, None, None, 0, False)
    torch.autograd.graph.increment_version(out)
    return out


def _raw_stream(index):
    """A device's current stream as the C entries take it.  torch.cuda.current_stream makes a Stream object for it: 4 us on the caller's thread
    and 16 on a backward thread, a tenth of a small call with its gradients."""
    return torch._C._cuda_getCurrentRawStream(index)


def _records(xs, outs, adds, ps):
    """The array of mvit_rotary_tensor that the C entries take."""
    rec = b""
    for i, (t, y, p) in enumerate(zip(xs, outs, ps)):
        add = adds[i] if adds is not None else None
        place, kind, steps, grid = 0, 0, (0, 0, 0), _NO_GRID
        if isinstance(p, TokenGrid):
            grid = p.record
        elif p is not None:
            place, kind, steps = p.data_ptr(), _POS[p.dtype], p.stride()
            steps = (0,) + steps if len(steps) == 2 else steps if p.shape[0] > 1 else (0,) + steps[1:]
        B, H, L, _ = t.shape
        rec += _RECORD.pack(t.data_ptr(), y.data_ptr(), add.data_ptr() if add is not None else 0, place, *t.stride()[:3], *y.stride()[:3],
                            *(add.stride()[:3] if add is not None else (0, 0, 0)), *steps, L, B, H, kind, *grid)
    return rec


def _launch(xs, outs, adds, ps, dim, axes, sections, turns, layout, inverse):
    x, rec = xs[0], _records(xs, outs, adds, ps)
    lib = _hip.lib_with_record("fp16" if x.dtype == torch.float16 else "bf16", "mvit_rotary_tensor_bytes", _RECORD.size)
    act = _hip.F32 if x.dtype == torch.float32 else _hip.BF16
    args = (rec, len(xs), dim, axes, sections, turns, layout, 1 if inverse else 0, act)
    at = x.device.index
    if at == torch.cuda.current_device():
        rc = lib.mvit_rotary(*args, _raw_stream(at))
    else:
        with torch.cuda.device(at):
            rc = lib.mvit_rotary(*args, _raw_stream(at))
    if rc == _hip.EINVAL and outs is xs:        # (everything else has been checked)
        raise ValueError("AxialRotary.rotate_: the tensors are the same memory in part, or one of them shares elements with itself; they "
                         "must not overlap")
    _hip.check(rc, "rotary")


def _leaf_on_one_stream(t):
    """A leaf's gradient node belongs to the stream it was made on and lives as long as any graph of the leaf.  A backward pass that is
    captured into a HIP graph while an eager graph of the same leaf is alive would make the capture wait for a stream outside it, which
    ends the process when the capture ends: refused here, as far as this operator has seen the leaf.  The first stream that a node is seen on
    is the one that counts: later calls on others (a warm-up before the capture) find the same node."""
    if not (t.is_leaf and t.requires_grad):
        return None
    node = torch.autograd.graph.get_gradient_edge(t).node
    stream = _raw_stream(t.device.index)
    if node.metadata.setdefault("rotary_stream", stream) != stream and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("AxialRotary: an eager graph of this leaf tensor is still alive while its backward pass is being captured; "
                           "drop it (its outputs, its loss) before the capture")
    return node


class _RotaryFn(torch.autograd.Function):
    """The turn is orthogonal: the gradient is turned back by the same angles (and a gradient's gradient forth again).  Nothing of the
    input is kept."""

    @staticmethod
    def forward(ctx, plan, ps, inverse, *xs):
        ctx.plan, ctx.inverse = plan, inverse
        ctx.ps = ps
        listed = [p for p in ps if not isinstance(p, TokenGrid)]
        if listed:                      # (kept by autograd, which notices a change of theirs in between)
            ctx.ps = [p if isinstance(p, TokenGrid) else None for p in ps]
            ctx.save_for_backward(*listed)
        return tuple(plan.turn(xs, ps, inverse=inverse))

    @staticmethod
    def backward(ctx, *grads):
        if forward_ad._current_level >= 0:
            _hip.refuse_tangents("AxialRotary", *grads)
        ps = ctx.ps
        if None in ps:
            saved = iter(ctx.saved_tensors)
            ps = [p if p is not None else next(saved) for p in ps]
        gs = [g if g.stride(3) == 1 else g.contiguous() for g in grads]
        if torch.is_grad_enabled():     # create_graph
            return (None, None, None) + _RotaryFn.apply(ctx.plan, ps, not ctx.inverse, *gs)
        return (None, None, None) + tuple(ctx.plan.turn(gs, ps, inverse=not ctx.inverse))
