"""Cases, plain forms and calls of the framework's rotary positions, its Newton-Schulz orthogonalisation and its Muon step."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = 10000.0
QUINTIC = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
STEPS = 5
MU = 0.95
DECAY = 1e-4
# a learning rate of the recipe's warm-up (it climbs from 2e-5 to 2e-3)
LR = 5e-5


# ---- cases --------------------------------------------------------------------------------------------------------------------------
def _rotary(name, dtype, batch, heads, dim, sections, layout, q, k, train, token_major=False, far=0):
    """q, k: token grids "TxHxW" (k as "grid/strides": its tokens stand at every stride-th place of q's grid), or a token count with
    positions of every token listed."""
    c = {"op": "rotary", "dtype": dtype, "batch": batch, "heads": heads, "dim": dim, "sections": sections, "layout": layout, "q": q,
         "k": k, "train": train, "token_major": token_major, "far": far}
    return dict(c, name=name) if name else c


def _orth(name, shape, batch, dtype):
    c = {"op": "orthogonalize", "shape": shape, "batch": batch, "dtype": dtype}
    return dict(c, name=name) if name else c


def _muon(name, shapes, nesterov=True):
    c = {"op": "muon", "shapes": shapes, "nesterov": nesterov}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token's query and key of one clip, as a streaming user rotates them: latency alone
        _rotary("rotary one token", "bf16", 1, 8, 96, "32,32,32", "half", "1", "1", False),
        # the block that most of the model's depth has (B = 8 clips at 448): four heads on 8 x 28 x 28, keys pooled by two
        _rotary("rotary stage 3", "bf16", 8, 4, 96, "32,32,32", "half", "8x28x28", "8x14x14/1x2x2", False),
        # the first block of a training step: one head on 8 x 112 x 112 tokens, keys pooled by eight, both directions
        _rotary("rotary stage 1 train", "bf16", 8, 1, 96, "32,32,32", "half", "8x112x112", "8x14x14/1x8x8", True),
        # exact arithmetic, images and videos of several sizes packed in one token-major batch, an odd number of tokens, odd sections
        _rotary("rotary packed fp32 train", "fp32", 3, 6, 80, "24,28,26", "interleaved", "4099", "4099", True, True, 512),
        # a long stream far from its beginning
        _rotary("rotary far fp16", "fp16", 2, 16, 128, "32,48,48", "half", "20011", "20011", False, False, 1000000),
        # one small weight's update: latency
        _orth("orthogonalize 96x288", "96x288", 1, "bf16"),
        # a batch of tall matrices of odd sizes
        _orth("orthogonalize 3x1000x257", "1000x257", 3, "bf16"),
        # an update that is wanted in single precision (the model's widest query / key / value weight)
        _orth("orthogonalize 2304x768 fp32", "2304x768", 1, "fp32"),
        # a large generic weight
        _orth("orthogonalize 4096x4096", "4096x4096", 1, "bf16"),
        # the weights of the model's first block
        _muon("muon first block", "288x96,96x96,384x96,96x384"),
        # odd and degenerate sizes: the class head, a single row, a single column, sizes that no tile divides
        _muon("muon ragged", "18x768,130x70,513x129,1x300,77x1,200x333", False),
        # every weight matrix of the model's blocks, as one training step updates them
        _muon("muon model", "model"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "orthogonalize", "muon"])
    if kind == "rotary":
        dtype, layout, train = rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["half", "interleaved"]), rng.random() < 0.5
        if rng.random() < 0.5:
            heads, s = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
            t, h, w = rng.randint(1, 16), _spread(rng, 1, 10) * s, _spread(rng, 1, 10) * s
            batch = max(1, min(8, _spread(rng, 1, 8), 60000000 // (heads * t * h * w * 96)))
            return _rotary("", dtype, batch, heads, 96, "32,32,32", layout, "%dx%dx%d" % (t, h, w),
                           "%dx%dx%d/1x%dx%d" % (t, h // s, w // s, s, s), train, rng.random() < 0.3)
        axes = rng.randint(1, 3)
        sections = [2 * rng.randint(2, 24) for _ in range(axes)]
        dim = sum(sections) + rng.choice([0, 0, 1, 6, 16])
        heads, tokens = rng.randint(1, 16), _spread(rng, 1, 30000)
        batch = max(1, min(4, 30000000 // (heads * tokens * dim)))
        return _rotary("", dtype, batch, heads, dim, ",".join(map(str, sections)), layout, str(tokens), str(tokens), train,
                       rng.random() < 0.5, rng.choice([0, 512, 1000000]))
    if kind == "orthogonalize":
        m, n = _spread(rng, 1, 2500), _spread(rng, 1, 2500)
        return _orth("", "%dx%d" % (m, n), rng.randint(1, 3), rng.choice(["bf16", "bf16", "fp32"]))
    shapes = ["%dx%d" % (_spread(rng, 1, 1600), _spread(rng, 1, 1600)) for _ in range(rng.randint(1, 12))]
    return _muon("", ",".join(shapes), rng.random() < 0.7)


# ---- what the texts of a case stand for -----------------------------------------------------------------------------------------------
def _ints(text, sep):
    return [int(v) for v in text.split(sep)]


def _grid(text):
    """(sizes, strides) of a token grid."""
    grid, _, strides = text.partition("/")
    sizes = _ints(grid, "x")
    return sizes, _ints(strides, "x") if strides else [1] * len(sizes)


def _tokens(text):
    return math.prod(_grid(text)[0])


def _shapes(text):
    if text != "model":
        return [tuple(_ints(s, "x")) for s in text.split(",")]
    found = []
    for i, o in [(96, 96), (96, 192), (192, 192), (192, 384)] + [(384, 384)] * 10 + [(384, 768), (768, 768)]:  # the blocks' widths in and out
        found += [(3 * o, i), (o, o), (4 * o, o), (o, 4 * o)] + ([(o, i)] if i != o else [])
    return found


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _update(rows, cols, batch, gen):
    """A weight gradient: products of activations and output gradients, whose spectrum falls off, and the noise of a batch under them."""
    r = min(rows, cols, 64)
    fall = torch.logspace(0, -2, r, device="cuda") if r > 1 else torch.ones(1, device="cuda")
    left = torch.randn(batch, rows, r, generator=gen, device="cuda") * fall
    return (left @ torch.randn(batch, r, cols, generator=gen, device="cuda") + 0.1 * torch.randn(batch, rows, cols, generator=gen, device="cuda")) * 1e-3


def _inputs(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "orthogonalize":
        u = _update(*_ints(case["shape"], "x"), case["batch"], gen)
        return {"case": case, "update": u if case["batch"] > 1 else u[0]}
    if case["op"] == "muon":
        shapes = _shapes(case["shapes"])
        ends = [0]
        for r, c in shapes:
            ends.append(ends[-1] + r * c)
        w, m = (torch.randn(ends[-1], generator=gen, device="cuda") * s for s in (0.02, 1e-4))
        grads = [_update(r, c, 1, gen)[0] for r, c in shapes]
        views = lambda flat: [flat[a:b].view(s) for a, b, s in zip(ends, ends[1:], shapes)]  # noqa: E731
        return {"case": case, "weights": w, "momenta": m, "w": views(w), "m": views(m), "g": grads}
    dtype, b, h, d = DTYPES[case["dtype"]], case["batch"], case["heads"], case["dim"]
    state = {"case": case}
    for part in ("q", "k"):
        n = _tokens(case[part])
        for name in (part, "d" + part):
            if case["token_major"]:  # a slice of a fused buffer: heads and channels of one token side by side
                x = torch.randn(b, n, 2 * h, d, generator=gen, device="cuda").to(dtype)[:, :, :h].transpose(1, 2)
            else:
                x = torch.randn(b, h, n, d, generator=gen, device="cuda").to(dtype)
            state[name] = x
        if "x" not in case[part]:
            axes = len(case["sections"].split(","))
            state[part + "_at"] = torch.randint(0, max(case["far"], 64), (b, n, axes), generator=gen, device="cuda")
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "rotary":
        from aicity_action_amd.rotary import AxialRotary, TokenGrid
        state["plan"] = AxialRotary(case["dim"], _ints(case["sections"], ","), base=BASE, layout=case["layout"])
        for part in ("q", "k"):
            if "x" in case[part]:
                state[part + "_at"] = TokenGrid(*_grid(case[part]))
    if own and case["op"] == "muon":
        from aicity_action_amd.muon import MuonMatrices
        state["plan"] = MuonMatrices(state["w"], state["m"], momentum=MU, nesterov=case["nesterov"], weight_decay=DECAY)
    if case["op"] == "rotary" and case["train"]:
        for part in ("q", "k"):
            state[part].requires_grad_(own)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "orthogonalize":
        return _plain_orthogonal(state["update"]).to(DTYPES[case["dtype"]])
    if case["op"] == "muon":
        return _plain_muon(state, case["nesterov"])
    q, k = (_plain_rotary(case, part, state[part], state.get(part + "_at"), 1.0) for part in ("q", "k"))
    if not case["train"]:
        return [q, k]
    return [q, k] + [_plain_rotary(case, part, state["d" + part], state.get(part + "_at"), -1.0) for part in ("q", "k")]


def _run_own(state, case):
    if case["op"] == "orthogonalize":
        from aicity_action_amd.muon import orthogonalize
        return orthogonalize(state["update"], dtype=DTYPES[case["dtype"]])
    if case["op"] == "muon":
        state["plan"].step(state["g"], lr=LR)
        return [state["weights"], state["momenta"]]
    q, k = state["plan"](state["q"], state["q_at"], state["k"], state["k_at"])
    if not case["train"]:
        return [q, k]
    return [q.detach(), k.detach()] + list(torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"])))


def _pairs(case, device):
    """Channels a, b of every pair, the axis it turns by, and its frequency (in 64 bits)."""
    a, b, axis, freq, first = [], [], [], [], 0
    for n, s in enumerate(_ints(case["sections"], ",")):
        i = torch.arange(s // 2, device=device)
        a.append(first + (i if case["layout"] == "half" else 2 * i))
        b.append(a[-1] + (s // 2 if case["layout"] == "half" else 1))
        axis.append(torch.full_like(i, n))
        freq.append(BASE ** (-2.0 * i.double() / s))
        first += s
    return torch.cat(a), torch.cat(b), torch.cat(axis), torch.cat(freq)


def _positions(case, part, at, device):
    """[1 or batch, tokens, axes] in 64 bits."""
    if at is not None:
        return at.double()
    sizes, strides = _grid(case[part])
    lines = [torch.arange(n, device=device).double() * s for n, s in zip(sizes, strides)]
    return torch.stack(torch.meshgrid(*lines, indexing="ij"), -1).reshape(1, -1, len(sizes))


def _plain_rotary(case, part, x, at, sign):
    a, b, axis, freq = _pairs(case, x.device)
    angle = _positions(case, part, at, x.device)[:, None][..., axis] * freq  # far positions: an angle in 32 bits has lost its turn
    cos, sin = torch.cos(angle).float(), sign * torch.sin(angle).float()
    xf = x.float()
    xa, xb = xf[..., a], xf[..., b]
    y = xf.clone()
    y[..., a] = xa * cos - xb * sin
    y[..., b] = xa * sin + xb * cos
    return y.to(x.dtype)


def _plain_orthogonal(u):
    x = u.float()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().float() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(STEPS):
        s = x @ x.mT
        x = QUINTIC[0] * x + (QUINTIC[1] * s + QUINTIC[2] * (s @ s)) @ x
    return x.mT if tall else x


def _plain_muon(state, nesterov):
    for w, m, g in zip(state["w"], state["m"], state["g"]):
        m.mul_(MU).add_((1 - MU) * g)
        o = _plain_orthogonal((1 - MU) * g + MU * m if nesterov else m)
        w.mul_(1 - LR * DECAY).sub_(LR * 0.2 * math.sqrt(max(w.shape)) * o)
    return [state["weights"], state["momenta"]]


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def _orth_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m ** 3 + 2 * m * m * n)  # X X^T and A A are symmetric: half of each


def work(case):
    if case["op"] == "orthogonalize":
        r, c = _ints(case["shape"], "x")
        size = 2 if case["dtype"] != "fp32" else 4
        return {"bytes": case["batch"] * r * c * (4 + size), "flops": case["batch"] * _orth_flops(r, c)}
    if case["op"] == "muon":
        shapes = _shapes(case["shapes"])
        return {"bytes": 20 * sum(r * c for r, c in shapes), "flops": sum(_orth_flops(r, c) for r, c in shapes)}
    size, ways = 2 if case["dtype"] != "fp32" else 4, 2 if case["train"] else 1
    numel = case["batch"] * case["heads"] * case["dim"] * (_tokens(case["q"]) + _tokens(case["k"]))
    at = sum(8 * case["batch"] * _tokens(case[p]) * len(case["sections"].split(",")) for p in ("q", "k") if "x" not in case[p])
    return {"bytes": ways * (2 * size * numel + at), "flops": ways * 3 * numel}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------------------------
def _exact_rotary(case, x, text, at, sign):
    """Every section as complex numbers, multiplied by exp(i p f)."""
    sections = _ints(case["sections"], ",")
    if at is None:
        sizes, strides = _grid(text)
        n = torch.arange(math.prod(sizes), device=x.device)
        inner = [math.prod(sizes[i + 1:]) for i in range(len(sizes))]
        at = torch.stack([(n // step) % size * stride for step, size, stride in zip(inner, sizes, strides)], -1)[None]
    y, first = x.double(), 0
    out = y.clone()
    for axis, s in enumerate(sections):
        part = y[..., first:first + s]
        pairs = part.unflatten(-1, (2, s // 2)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (s // 2, 2))
        f = torch.exp(torch.arange(0, s, 2, device=x.device, dtype=torch.float64) * (-math.log(BASE) / s))
        angle = sign * at[:, None, :, axis, None].double() * f
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
        out[..., first:first + s] = (z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2)
        first += s
    return out


def _exact_orthogonal(u):
    u = u.double()
    x = u / (torch.linalg.matrix_norm(u, keepdim=True) + EPS)
    short = x.shape[-2] <= x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=u.device)
    for _ in range(STEPS):
        s = x @ x.mT.contiguous() if short else x.mT.contiguous() @ x
        p = QUINTIC[0] * eye + s @ (QUINTIC[1] * eye + QUINTIC[2] * s)
        x = p @ x if short else x @ p
    return x


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "orthogonalize":
        return _exact_orthogonal(state["update"])
    if case["op"] == "muon":
        ws, ms = [], []
        for w, m, g in zip(state["w"], state["m"], state["g"]):
            m = MU * m.double() + (1 - MU) * g.double()
            o = _exact_orthogonal((1 - MU) * g.double() + MU * m if case["nesterov"] else m)
            ws.append(((1 - LR * DECAY) * w.double() - LR * 0.2 * math.sqrt(max(w.shape)) * o).flatten())
            ms.append(m.flatten())
        return [torch.cat(ws), torch.cat(ms)]
    ways = [("q", "q", 1.0), ("k", "k", 1.0)] + ([("dq", "q", -1.0), ("dk", "k", -1.0)] if case["train"] else [])
    return [_exact_rotary(case, state[x], case[p], state.get(p + "_at"), s) for x, p, s in ways]
