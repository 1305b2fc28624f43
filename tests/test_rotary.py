"""Rotary positions (aicity_action_amd/rotary.py) against the definition in 64 bits, and its refusals (those run on the CPU)."""
import copy
import math
import pickle
import random

import pytest
import torch

from aicity_action_amd.rotary import AxialRotary, TokenGrid, add_

gpu = pytest.mark.gpu
DEV = "cuda:0"


def places_of(p, batch):
    if not isinstance(p, TokenGrid):
        return (p if p.dim() == 3 else p[None]).double().cpu().expand(batch, -1, -1)
    axes = [o + s * torch.arange(n, dtype=torch.float64) for n, s, o in zip(p.sizes, p.step, p.origin)]
    return torch.stack([g.reshape(-1) for g in torch.meshgrid(*axes, indexing="ij")], -1)[None].expand(batch, -1, -1)


def oracle(x, p, sections, base, layout, sign=1.0):
    """(rot(x), |x_a| + |x_b| of each channel's pair) in 64 bits, as complex numbers."""
    x = x.detach().double().cpu()
    at = places_of(p, x.shape[0])
    y, mag, first = x.clone(), x.abs().clone(), 0
    for axis, s in enumerate(sections):
        part = x[..., first:first + s]
        pair = part.unflatten(-1, (2, s // 2)).transpose(-1, -2) if layout == "half" else part.unflatten(-1, (s // 2, 2))
        f = torch.tensor([base ** (-2.0 * i / s) for i in range(s // 2)], dtype=torch.float64)
        ang = sign * at[:, None, :, axis, None] * f
        z = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(ang), ang)
        out, m = torch.view_as_real(z), pair.abs().sum(-1, keepdim=True).expand_as(pair)
        if layout == "half":
            out, m = out.transpose(-1, -2), m.transpose(-1, -2)
        y[..., first:first + s], mag[..., first:first + s] = out.flatten(-2), m.flatten(-2)
        first += s
    return y, mag


def check(got, x, p, sections, base, layout, sign=1.0, add=None):
    """One rounding to the result's type, and in 32 bits: the turn's fraction (2^-26 turns = 1e-7), sine and cosine (2 ulp = 2.4e-7), two
    products and a sum (1.2e-7): under 6e-7 of the pair's |x_a| + |x_b|."""
    want, mag = oracle(x, p, sections, base, layout, sign)
    tol = 6e-7 * mag
    if add is not None:
        want = want + add.detach().double().cpu()
        tol = tol + 2.0 ** -24 * want.abs()
    tol = tol * 1.01 + torch.finfo(got.dtype).eps / 2 * want.abs() + torch.finfo(got.dtype).tiny
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV).to(dtype)


CASES = [     # dim, sections, batch, heads, positions
    (96, (32, 32, 32), 2, 4, TokenGrid((2, 7, 5))),
    (96, (32, 32, 32), 1, 8, TokenGrid((1, 1, 1), origin=(5, 6, 7))),
    (96, (32, 32, 32), 3, 1, TokenGrid((3, 4, 4), step=(1, 8, 8))),
    (128, (32, 48, 48), 1, 2, TokenGrid((4, 9, 3), step=(0.5, 1.5, 2.0), origin=(-1.0, 0.25, 3.0))),
    (80, (24, 28, 26), 2, 3, TokenGrid((2, 3, 5))),
    (7, (2, 4), 2, 5, TokenGrid((3, 11))),
    (64, (64,), 1, 3, TokenGrid((257,))),
    (61, (8, 4, 12, 6), 2, 2, TokenGrid((2, 3, 2, 3))),
    (512, (256, 128, 128), 1, 1, TokenGrid((2, 2, 2))),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_backward(case, layout, dtype):
    dim, sections, B, H, grid = CASES[case]
    rot = AxialRotary(dim, sections, base=100.0, layout=layout)
    x = randn((B, H, grid.tokens, dim), dtype, case).requires_grad_(True)
    y = rot(x, grid)
    check(y, x, grid, sections, 100.0, layout)
    dy = randn(y.shape, dtype, case + 50)
    (dx,) = torch.autograd.grad(y, x, dy)
    check(dx, dy, grid, sections, 100.0, layout, sign=-1.0)


@gpu
@pytest.mark.parametrize("dtype,pos", [(torch.bfloat16, torch.int64), (torch.float32, torch.int32), (torch.float16, torch.float32)])
def test_listed_positions_query_and_key_token_major(dtype, pos):
    B, H, L, D, S = 2, 3, 131, 96, (16, 40, 40)
    buf = randn((B, L, 3 * H, D), dtype, 3)
    q, k = buf[:, :, :H].transpose(1, 2).requires_grad_(True), buf[:, ::2, H:2 * H].transpose(1, 2).requires_grad_(True)
    pq = torch.randint(-4, 1000, (B, L, 3), generator=torch.Generator().manual_seed(1)).to(DEV).to(pos)
    pk = torch.randint(0, 1000, (k.shape[2], 3), generator=torch.Generator().manual_seed(2)).to(DEV).to(pos)
    rot = AxialRotary(D, S)
    yq, yk = rot(q, pq, k, pk)
    check(yq, q, pq, S, 10000.0, "half")
    check(yk, k, pk, S, 10000.0, "half")
    dq, dk = randn(yq.shape, dtype, 5).transpose(2, 3).contiguous().transpose(2, 3), randn(yk.shape, dtype, 6)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))      # one gradient arrives with its channels apart
    check(gq, dq, pq, S, 10000.0, "half", sign=-1.0)
    check(gk, dk, pk, S, 10000.0, "half", sign=-1.0)


@gpu
def test_far_positions_keep_their_turn():
    p = torch.tensor([[10 ** 6 + 1, 2 ** 31 + 3, 7], [10 ** 7, 2 ** 40 + 1, 0], [-(2 ** 33), 1, 2]], device=DEV)
    x = randn((1, 2, 3, 48), torch.float32, 9)
    # in 64 bits the product place x turns is off by 2^-53 of itself: 2^40 / (2 pi) turns -> 2e-5 turns at the farthest place
    got, (want, mag) = AxialRotary(48, (16, 16, 16))(x, p), oracle(x, p, (16, 16, 16), 10000.0, "half")
    far = places_of(p, 1).abs().amax(-1)[:, None, :, None]
    assert ((got.double().cpu() - want).abs() <= mag * (1e-6 + far * 2.0 ** -51)).all()


@gpu
def test_gradient_against_differences():
    rot, grid = AxialRotary(12, (4, 4, 4), base=50.0), TokenGrid((2, 2, 3))
    x, w = randn((1, 2, 12, 12), torch.float32, 11), randn((1, 2, 12, 12), torch.float32, 12)
    v = randn(x.shape, torch.float32, 13)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad((rot(x, grid) * w).sum(), x)
    with torch.no_grad():                       # the map is linear: a wide difference is exact up to rounding
        d = ((rot(x + 8 * v, grid) * w).double().sum() - (rot(x - 8 * v, grid) * w).double().sum()) / 16
    # sums of 288 products of O(10) values, each 2^-23 off at most
    assert abs(d.item() - (g.double() * v.double()).sum().item()) <= 288 * 30 * 2.0 ** -23


@gpu
def test_gradient_of_a_gradient():
    rot, grid = AxialRotary(12, (4, 4, 4), base=50.0), TokenGrid((2, 1, 3))
    x = randn((1, 1, 6, 12), torch.float32, 14).requires_grad_(True)
    w = randn((1, 1, 6, 12), torch.float32, 15)
    y = rot(x, grid)
    (g,) = torch.autograd.grad((y * y * w).sum(), x, create_graph=True)        # g = R^T (2 w R x)
    (gg,) = torch.autograd.grad((g * g).sum(), x)                              # 2 R^T (2 w R (R^T (2 w R x)))
    forth = lambda t, s: oracle(t, grid, rot.sections, 50.0, "half", s)[0]  # noqa: E731
    wd = w.double().cpu()
    want = 2 * forth(2 * wd * forth(forth(2 * wd * forth(x, 1.0), -1.0), 1.0), -1.0)
    # four turns and three products, each 6e-7 of the pair at most
    assert (gg.double().cpu() - want).abs().max() <= 7 * 6e-7 * 2 * want.abs().max()


@gpu
def test_in_place_and_back_and_addend():
    rot, grid = AxialRotary(96), TokenGrid((2, 3, 3))
    buf = randn((2, 18, 5, 96), torch.bfloat16, 1)
    q, before = buf[:, :, 1:3].transpose(1, 2), buf.clone()
    want = rot(q, grid)
    assert rot.rotate_(q, grid) is q and torch.equal(q, want)
    assert torch.equal(buf[:, :, [0, 3, 4]], before[:, :, [0, 3, 4]])          # the neighbours in the buffer are as they were
    rot.rotate_(q, grid, inverse=True)                                          # two roundings, 2^-8 of the pair's length each
    assert (q - before[:, :, 1:3].transpose(1, 2)).abs().max() <= 2.01 * 2.0 ** -8 * before.abs().max() * 1.5
    a = randn((2, 2, 18, 96), torch.bfloat16, 2)
    y = torch.empty_like(a)
    rot.turn([a], [grid], outs=[y], adds=[want])
    check(y, a, grid, rot.sections, rot.base, "half", add=want)
    out = a.clone()
    add_(out, want)
    assert torch.equal(out, (a.float() + want.float()).to(torch.bfloat16))
    other = torch.empty_like(a)
    add_(other, want, x=a)
    assert torch.equal(other, out)


@gpu
def test_empty_expanded_and_wide_offsets():
    rot = AxialRotary(96)
    for shape in ((0, 2, 3, 96), (2, 0, 3, 96), (2, 2, 0, 96)):
        p = torch.zeros(shape[2], 3, dtype=torch.int64, device=DEV)
        x = torch.empty(shape, device=DEV, requires_grad=True)
        y = rot(x, p)
        assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    # an empty key tensor beside a full query tensor
    q = randn((1, 1, 4, 96), torch.float32, 1)
    yq, yk = rot(q, TokenGrid((1, 2, 2)), torch.empty(1, 1, 0, 96, device=DEV), torch.zeros(0, 3, device=DEV))
    check(yq, q, TokenGrid((1, 2, 2)), rot.sections, rot.base, "half")
    e = randn((1, 1, 1, 96), torch.float16, 2).expand(3, 2, 8, 96)
    check(rot(e, TokenGrid((2, 2, 2))), e, TokenGrid((2, 2, 2)), rot.sections, rot.base, "half")
    far = 2 ** 31 + 64
    buf = torch.empty(far + 4096, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((2, 1, 8, 96), (far, 0, 96, 1))
    x.copy_(randn(x.shape, torch.bfloat16, 3))
    src = x.clone()
    rot.rotate_(x, TokenGrid((2, 2, 2)))
    check(x, src, TokenGrid((2, 2, 2)), rot.sections, rot.base, "half")


@gpu
def test_side_stream_and_replayed_graph():
    rot, grid = AxialRotary(96), TokenGrid((2, 4, 4))
    x = randn((1, 2, 32, 96), torch.bfloat16, 21).requires_grad_(True)
    dy = randn(x.shape, torch.bfloat16, 22)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.autograd.grad(rot(x, grid), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rot(x, grid)
        (dx,) = torch.autograd.grad(y, x, dy)
    for i in range(3):
        with torch.no_grad():
            x.copy_(randn(x.shape, torch.bfloat16, 30 + i))
            dy.copy_(randn(x.shape, torch.bfloat16, 40 + i))
        graph.replay()
        torch.cuda.synchronize()
        check(y, x, grid, rot.sections, rot.base, "half")
        check(dx, dy, grid, rot.sections, rot.base, "half", sign=-1.0)


def test_capture_beside_a_living_eager_graph_is_refused(monkeypatch):
    from aicity_action_amd import rotary

    class Stream(object):
        cuda_stream = 1
    capturing = [False]
    monkeypatch.setattr(rotary, "_raw_stream", lambda index: Stream.cuda_stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    x = torch.zeros(3, requires_grad=True)
    node = rotary._leaf_on_one_stream(x)
    y = x * 2                                    # holds the node
    del node
    capturing[0], Stream.cuda_stream = True, 2
    with pytest.raises(RuntimeError, match="eager graph"):
        rotary._leaf_on_one_stream(x)
    del y                                        # the eager graph is gone, and its node with it
    y = x * 3 if rotary._leaf_on_one_stream(x) is not None else None
    assert rotary._leaf_on_one_stream(x) is not None
    assert rotary._leaf_on_one_stream(x * 2) is None and rotary._leaf_on_one_stream(torch.zeros(1)) is None


def test_a_warm_up_on_the_capture_stream_does_not_hide_a_living_eager_graph(monkeypatch):
    """Eager graph on stream 1, kept; warm-up on stream 2, dropped; capture on stream 2: the node is still stream 1's."""
    from aicity_action_amd import rotary
    stream, capturing = [1], [False]
    monkeypatch.setattr(rotary, "_raw_stream", lambda index: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    x = torch.zeros(3, requires_grad=True)

    def call():
        node = rotary._leaf_on_one_stream(x)
        return x * 2, node
    kept = call()[0]
    stream[0] = 2
    for _ in range(2):
        call()
    capturing[0] = True
    with pytest.raises(RuntimeError, match="eager graph"):
        call()
    del kept                                     # with the last graph of stream 1 the node goes, and the next one is stream 2's
    again = call()[0]
    assert call() and again is not None


def test_a_plan_is_copied_and_pickled():
    plan = AxialRotary(40, (8, 12, 20), base=77.0, layout="interleaved")
    for other in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert (other.head_dim, other.sections, other.base, other.layout) == (plan.head_dim, plan.sections, plan.base, plan.layout)
        assert list(other._turns) == list(plan._turns) and list(other._sections) == list(plan._sections)


def test_refusals():
    with pytest.raises(ValueError, match="layout"):
        AxialRotary(96, layout="split")
    for sections in ((), (31, 33, 32), (64, 64), (2, 2, 2, 2, 2), (0, 2, 2)):
        with pytest.raises(ValueError, match="sections"):
            AxialRotary(96, sections)
    for base in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="base"):
            AxialRotary(96, base=base)
    for bad in (dict(sizes=()), dict(sizes=(1, 2, 0)), dict(sizes=(1,) * 5), dict(sizes=(2, 2), step=(1,)), dict(sizes=(2,), origin=(math.nan,))):
        with pytest.raises(ValueError, match="TokenGrid"):
            TokenGrid(**bad)
    rot, x, grid = AxialRotary(96), torch.zeros(2, 1, 8, 96), TokenGrid((2, 2, 2))
    for t, p in ((x[0], grid), (x[..., :90], grid), (x, TokenGrid((2, 2, 3))), (x, TokenGrid((2, 4))), (x, torch.zeros(8, 2)),
                 (x, torch.zeros(3, 8, 3)), (x.transpose(2, 3).contiguous().transpose(2, 3), grid)):
        with pytest.raises(ValueError):
            rot(t, p)
    for t, p in ((x.double(), grid), (x, torch.zeros(8, 3, dtype=torch.float64)), (x, None), (x, (2, 2, 2))):
        with pytest.raises(TypeError):
            rot(t, p)
    with pytest.raises(ValueError, match="together"):
        rot(x, grid, x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rot(x, grid)
    assert rot.sections == (32, 32, 32) and AxialRotary(80).sections == (26, 26, 26)


@gpu
def test_refusals_on_the_device():
    rot, x, grid = AxialRotary(96), torch.zeros(2, 1, 8, 96, device=DEV), TokenGrid((2, 2, 2))
    with pytest.raises(ValueError, match="positions on"):
        rot(x, torch.zeros(8, 3))
    with pytest.raises(ValueError, match="one dtype"):
        rot(x, grid, x.half(), grid)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        rot.rotate_(x.clone().requires_grad_(True), grid)
    with pytest.raises(ValueError, match="expanded"):
        rot.rotate_(x[:1].expand(3, 1, 8, 96), grid)
    with pytest.raises(ValueError, match="no gradient"):
        rot(x, torch.zeros(8, 3, device=DEV, requires_grad=True))
    version = x._version
    rot.rotate_(x, grid)
    assert x._version > version
    with pytest.raises(ValueError, match="same memory"):
        rot.rotate_(x, grid, x, grid)


def test_forward_mode_tangents_are_refused(monkeypatch):
    """A dual tensor does not require a gradient, and a kernel's output has no tangent: torch would read zero.  With the launch replaced, on
    the host."""
    from torch.autograd import forward_ad

    from aicity_action_amd import rotary
    rot, grid = AxialRotary(96), TokenGrid((2, 2, 2))
    monkeypatch.setattr(rotary, "_launch", lambda *a: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    x, at = torch.zeros(1, 1, 8, 96), torch.zeros(8, 3)
    assert rot(x, grid).shape == x.shape and rot.rotate_(x, at) is x
    with forward_ad.dual_level():
        dual, places = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(at, torch.ones_like(at))
        for call in (lambda: rot(dual, grid), lambda: rot.rotate_(dual, grid), lambda: rot(x, grid, dual, grid), lambda: rot(x, places),
                     lambda: rot(dual.transpose(0, 1), grid)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert rot(dual.detach(), grid).shape == rot(x, grid).shape == x.shape


def _overlap(xs, outs=None, adds=None):
    from aicity_action_amd import _hip, rotary
    outs = xs if outs is None else outs
    rec = rotary._records(xs, outs, adds, [TokenGrid((t.shape[2], 1, 1)) if t.shape[2] else torch.zeros(0, 3) for t in xs])
    return _hip.lib().mvit_rotary_overlap(rec, len(xs), xs[0].shape[3], _hip.F32 if xs[0].dtype == torch.float32 else _hip.BF16)


def test_overlap_of_views_against_their_elements():
    """Random views of one buffer: an overlap is always found, and none is seen where there is none."""
    rng, flat = random.Random(1), torch.zeros(4000)

    def view(dim):
        sizes = [rng.choice([1, 1, 2, 3, 4]) for _ in range(3)]
        unit = dim if rng.random() < 0.6 else 1
        strides = [unit * rng.choice([1, 2, 3, 4, 6, 12, 24]) for _ in range(3)]
        return flat.as_strided(sizes + [dim], strides + [1], rng.randint(0, 30) * unit)

    def elements(t):
        return torch.arange(4000).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()
    seen = [0, 0]
    for _ in range(3000):
        dim = rng.choice([2, 4, 8])
        x, k = view(dim), view(dim)
        a, b = elements(x), elements(k)
        if len(set(a)) < len(a) or len(set(b)) < len(b):
            assert _overlap([x, k]) == 1
            continue
        want = int(bool(set(a) & set(b)))
        nested = all(_overlap([t]) == 0 for t in (x, k))     # (strides that neither nest nor collide count as a collision)
        assert _overlap([x, k]) == (want if nested else 1)
        seen[want] += nested
    assert min(seen) > 100
    # written, read, added
    x, y, z = flat[:96].view(1, 2, 6, 8), flat[96:192].view(1, 2, 6, 8), flat[8:104].view(1, 2, 6, 8)
    assert _overlap([x], [y]) == 0 and _overlap([x], [x], [x]) == 0 and _overlap([x], [y], [z]) == 1 and _overlap([x], [z]) == 1
    assert _overlap([x, y], [y, x]) == 1 and _overlap([x, x], [y, flat[192:288].view(1, 2, 6, 8)]) == 0


def test_heads_of_a_fused_buffer_do_not_overlap():
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.zeros(4, 784, 12, 96, dtype=dtype)
        q, k = buf[:, :, :4].transpose(1, 2), buf[:, :, 4:8].transpose(1, 2)
        assert _overlap([q, k]) == 0 and _overlap([q, buf[:, :, 3:5].transpose(1, 2)]) == 1
        assert _overlap([q, k[:, :, ::4]]) == 0 and _overlap([q, q[:, 3:, 5::4]]) == 1     # every fourth token
        assert _overlap([q[:2], k[1:]]) == 0 and _overlap([q[:2], q[2:]]) == 0 and _overlap([q[:2], q[1:]]) == 1
        assert _overlap([q[..., :48], q[..., 48:]]) == 0 and _overlap([q[..., :50], q[..., 46:]]) == 1
        assert _overlap([q[:, :0], q]) == 0 and _overlap([q[:, :, :, :2].expand(4, 4, 784, 2)]) == 0
        assert _overlap([q[:, :1].expand(4, 3, 784, 96)]) == 1 and _overlap([buf.as_strided((1, 1, 9, 96), (1, 1, 95, 1))]) == 1


@gpu
def test_in_place_turns_of_overlapping_views_are_refused():
    rot, grid = AxialRotary(96), TokenGrid((2, 2, 2))
    buf = randn((2, 8, 6, 96), torch.bfloat16, 4)
    before = buf.clone()
    views = lambda b: (b[:, :, :3].transpose(1, 2), b[:, :, 2:4].transpose(1, 2), b[:, :, 3:5].transpose(1, 2))  # noqa: E731
    q, near, k = views(buf)
    with pytest.raises(ValueError, match="must not overlap"):
        rot.rotate_(q, grid, near, grid)
    with pytest.raises(ValueError, match="must not overlap"):
        rot.rotate_(buf.as_strided((1, 1, 8, 96), (768, 768, 64, 1)), grid)
    assert torch.equal(buf, before)
    want = [rot(t, grid) for t in views(before)]
    rot.rotate_(q, grid, k, grid)
    assert torch.equal(q, want[0]) and torch.equal(k, want[2]) and torch.equal(buf[:, :, 5:], before[:, :, 5:])


def test_gradients_with_a_forward_mode_tangent_are_refused(monkeypatch):
    """Forward over reverse: the tangent comes with the gradient, not with the tensor."""
    from torch.autograd import forward_ad

    from aicity_action_amd import rotary
    rot, grid = AxialRotary(96), TokenGrid((2, 2, 2))
    monkeypatch.setattr(rotary, "_launch", lambda xs, outs, *a: [y.zero_() for y in outs])
    monkeypatch.setattr(rotary, "_leaf_on_one_stream", lambda t: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    x, w = torch.zeros(1, 1, 8, 96, requires_grad=True), torch.ones(1, 1, 8, 96)
    assert torch.autograd.grad(rot(x, grid), x, w)[0].shape == x.shape
    with forward_ad.dual_level():
        y = rot(x, grid)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(w, torch.ones_like(w)))
        assert torch.autograd.grad(rot(x, grid), x, w)[0].shape == x.shape
