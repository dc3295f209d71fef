"""What stands between two layers of a model on node features, as cases that can be timed: layer norm, dropout, and
layer norm -> ReLU -> dropout in one, forward alone (inference) or with the gradients (training).

Rows are node features after a propagation or a Linear: a spread and an offset of their own per row, so that the
statistics have something to take away.  Every random number of a case is an input: the seed and the offset that a
training step keys its masks with.
"""
import concurrent.futures
import functools
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float64": torch.float64, "float16": torch.float16, "bfloat16": torch.bfloat16}
LARGEST = 2449029 * 256  # elements


def _case(name, op, rows, width, dtype, grad, params="same", relu=False, p=0.0):
    return dict(name=name, op=op, rows=rows, width=width, dtype=dtype, params=params, grad=grad, relu=relu, p=p)


def listed():
    return [
        # One node is asked for: the smallest call there is.
        _case("norm_node", "norm", 1, 128, "float32", False),
        # A training step on a citation graph, full batch: a few microseconds of work.
        _case("norm_citation", "norm", 2708, 128, "float32", True),
        # Wide raw features of a sampled batch, no whole packs, 16-bit rows under 32-bit parameters.
        _case("norm_wide_odd", "norm", 49784, 602, "bfloat16", True, params="float32"),
        # The input features of the large configuration: 2.4 M rows of 100.
        _case("norm_large", "norm", 2449029, 100, "float32", True),
        # Inference over rows that no single wavefront holds.
        _case("norm_infer_long", "norm", 4096, 4096, "float16", False),
        # The hidden rows of one mini-batch.
        _case("drop_batch", "drop", 1024, 64, "float32", False, p=0.5),
        # Class scores of the benchmark's graph: narrow odd rows.
        _case("drop_odd", "drop", 325557, 47, "float32", True, p=0.2),
        # Double precision, as for checks of gradients.
        _case("drop_double", "drop", 100003, 33, "float64", True, p=0.5),
        # The most masks that a model of the large configuration draws, 16-bit rows.
        _case("drop_large", "drop", 2449029, 256, "bfloat16", True, p=0.5),
        # Between the two layers of a citation-size GCN.
        _case("block_citation", "block", 2708, 128, "float32", True, relu=True, p=0.5),
        # Between the layers of a mid-size model in half precision, one feature more than whole packs.
        _case("block_half_odd", "block", 325557, 257, "float16", True, params="float32", relu=True, p=0.3),
        # Between the layers of the large configuration.
        _case("block_large", "block", 2449029, 256, "float32", True, relu=True, p=0.5),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, uniform in its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(("norm", "drop", "block"))
    width = _spread(rng, 1, 8192)
    if rng.random() < 0.5:
        width = max(8, width // 8 * 8)
    dtype = rng.choice(("float32", "float32", "bfloat16", "float16", "float64"))
    rows = min(_spread(rng, 1, 2449029), max(1, LARGEST // (2 * width * (2 if dtype == "float64" else 1))))
    params = rng.choice(("same", "float32")) if op != "drop" and dtype in ("float16", "bfloat16") else "same"
    return dict(op=op, rows=rows, width=width, dtype=dtype, params=params, grad=rng.random() < 0.7,
                relu=op == "block" and rng.random() < 0.7, p=round(rng.uniform(0.05, 0.9), 3) if op != "norm" else 0.0)


# ------------------------------------------------------------------------------ inputs --
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + case["rows"] + 31 * case["width"])
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    x = normal(rows, width).mul_(0.5 + torch.rand(rows, 1, device="cuda", generator=gen)).add_(normal(rows, 1) * 0.3)
    state = dict(case=case, x=x.to(dtype), seed=0x9E3779B9 * (seed + 1), offset=(5 << 32) + 7 * seed)
    if case["op"] != "drop":
        kind = dtype if case["params"] == "same" else TYPES[case["params"]]
        state["weight"] = (1 + 0.2 * normal(width)).to(kind)
        state["bias"] = (0.2 * normal(width)).to(kind)
    if case["grad"]:
        state["grad"] = (0.1 * normal(rows, width)).to(dtype)
        for name in ("x", "weight", "bias"):
            if name in state:
                state[name].requires_grad_()
    return state


EPS = 1e-5


# ----------------------------------------------------------- the framework's operators --
@functools.lru_cache(None)
def _calls():
    import compressgnn_amd.layer._paths  # noqa: F401  (the package's modules are imported by bare name)
    from CompressgnnDropout import dropout
    from CompressgnnNorm import layer_norm, norm_act_dropout
    return layer_norm, dropout, norm_act_dropout


def _run_own(state):
    layer_norm, dropout, norm_act_dropout = _calls()
    case = state["case"]
    if case["op"] == "drop":
        leaves = (state["x"],)
        out = dropout(state["x"], case["p"], state["seed"], state["offset"])
    else:
        leaves = (state["x"], state["weight"], state["bias"])
        if case["op"] == "norm":
            out = layer_norm(*leaves, EPS)
        else:
            out = norm_act_dropout(*leaves, EPS, "relu" if case["relu"] else None, case["p"], state["seed"], state["offset"])
    if not case["grad"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, leaves, state["grad"])]


# ------------------------------------------------------------------ their plain forms --
def _keep(rows, width, p, seed, offset, device):
    """(truth values [rows, width], scale): Philox4x32-10 numbers of eight elements of a row each, 16 bits an element."""
    kept = math.floor((1 - p) * 65536 + 0.5)
    blocks = -(-width // 8)
    low32 = 0xFFFFFFFF
    n = torch.arange(rows * blocks, device=device)
    c0, c1 = n & low32, n >> 32
    c2, c3 = torch.full_like(n, offset & low32), torch.full_like(n, (offset >> 32) & low32)
    k0, k1 = seed & low32, (seed >> 32) & low32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64 bits: what wraps keeps its bits
        c0, c1, c2, c3 = ((b >> 32) & low32) ^ c1 ^ k0, b & low32, ((a >> 32) & low32) ^ c3 ^ k1, a & low32
        k0, k1 = (k0 + 0x9E3779B9) & low32, (k1 + 0xBB67AE85) & low32
    words = torch.stack((c0, c1, c2, c3), dim=1).to(torch.int32)
    draws = torch.stack((words & 0xFFFF, (words >> 16) & 0xFFFF), dim=2).view(rows, blocks * 8)
    return draws[:, :width] < kept, 65536 / kept if kept else 0.0


def _run_plain(state):
    case = state["case"]
    x, dtype = state["x"].detach(), TYPES[case["dtype"]]
    narrow = torch.float64 if dtype == torch.float64 else torch.float32
    keep = None
    if case["op"] == "drop" or case["p"] > 0:
        keep, scale = _keep(case["rows"], case["width"], case["p"], state["seed"], state["offset"], x.device)
        zero = torch.zeros((), dtype=narrow, device=x.device)
    if case["op"] == "drop":
        out = torch.where(keep, x.to(narrow) * scale, zero).to(dtype)
        if not case["grad"]:
            return [out]
        return [out, torch.where(keep, state["grad"].to(narrow) * scale, zero).to(dtype)]
    # which side of zero a sum is on decides whether its gradient passes: in 64 bits where there is a ReLU
    wide = torch.float64 if case["relu"] else narrow
    w, b = state["weight"].detach(), state["bias"].detach()
    width = case["width"]
    centred = x.to(wide)
    centred = centred - centred.sum(1, keepdim=True) / width
    rstd = 1 / torch.sqrt((centred * centred).sum(1, keepdim=True) / width + EPS)
    h = centred * rstd
    y = h * w.to(wide) + b.to(wide)
    del centred
    if case["relu"]:
        off = y <= 0
        y = y.masked_fill(off, 0)
    h, rstd, y = h.to(narrow), rstd.to(narrow), y.to(narrow)
    out = (y if keep is None else torch.where(keep, y * scale, zero)).to(dtype)
    if not case["grad"]:
        return [out]
    del y
    g = state["grad"].to(narrow)
    if keep is not None:
        g = torch.where(keep, g * scale, zero)
    if case["relu"]:
        g = g.masked_fill(off, 0)
    dw, db = (g * h).sum(0), g.sum(0)
    g = g * w.to(narrow)
    dx = rstd * (g - g.sum(1, keepdim=True) / width - h * ((g * h).sum(1, keepdim=True) / width))
    return [out, dx.to(dtype), dw.to(w.dtype), db.to(b.dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- work --
def work(case):
    item = {"float64": 8, "float32": 4}.get(case["dtype"], 2)
    n = case["rows"] * case["width"]
    # forward: x in, out out; with gradients the output's gradient in and x's out too
    moved = n * item * (4 if case["grad"] else 2)
    flops = 0
    if case["op"] != "drop":
        param = 4 if case["params"] == "float32" else item
        moved += 2 * case["width"] * param * (2 if case["grad"] else 1)
        flops += n * (8 + (14 if case["grad"] else 0))
    if case["op"] == "drop" or case["p"] > 0:
        flops += n * 12 * (2 if case["grad"] else 1)  # a tenth of a generator call's steps, a comparison, a product
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------- the same in 64 bits --
def _exact_keep(rows, width, p, seed, offset):
    """The mask on the host, from the generator's definition, block by block of rows."""
    kept = math.floor((1 - p) * 65536 + 0.5)
    blocks = -(-width // 8)
    mask = np.empty((rows, width), dtype=bool)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    step = max(1, (1 << 17) // blocks)

    def part(first):
        last = min(rows, first + step)
        number = np.arange(first * blocks, last * blocks, dtype=np.uint64)
        c = [number & low, number >> shift, np.full_like(number, offset & 0xFFFFFFFF), np.full_like(number, offset >> 32 & 0xFFFFFFFF)]
        for r in range(10):
            key = [np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
            p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(p1 >> shift) ^ c[1] ^ key[0], p1 & low, (p0 >> shift) ^ c[3] ^ key[1], p0 & low]
        draws = np.stack([half for word in c for half in (word & np.uint64(0xFFFF), word >> np.uint64(16))], axis=1)
        mask[first:last] = (draws < kept).reshape(last - first, blocks * 8)[:, :width]

    with concurrent.futures.ThreadPoolExecutor(8) as pool:
        list(pool.map(part, range(0, rows, step)))
    return mask, 65536 / max(kept, 1)


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].detach().double()
    factor = torch.ones((), dtype=torch.float64, device=x.device)
    if case["op"] == "drop" or case["p"] > 0:
        mask, scale = _exact_keep(case["rows"], case["width"], case["p"], state["seed"], state["offset"])
        factor = torch.from_numpy(mask).to(x.device).double().mul_(scale)
    if case["op"] == "drop":
        return [x * factor] + ([state["grad"].double() * factor] if case["grad"] else [])
    w, b = state["weight"].detach().double(), state["bias"].detach().double()
    h = torch.addcmul(x, x.mean(1, keepdim=True), torch.full((1, 1), -1.0, dtype=torch.float64, device=x.device))
    deviation = torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    h = h / deviation
    y = torch.addcmul(b, h, w)
    if case["relu"]:
        factor = factor * (y > 0)
    out = [y * factor]
    if case["grad"]:
        g = state["grad"].double() * factor
        t = g * w
        dx = (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True)) / deviation
        out += [dx, (g * h).sum(0), g.sum(0)]
    return out
