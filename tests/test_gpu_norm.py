"""Layer norm, dropout and both behind a ReLU on the GPU, against the formulas in 64 bits on the host; masks bit for bit."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import compressgnn_runtime as rt
from compressgnn_amd import abi
from CompressgnnDropout import Compressgnn_Dropout, dropout
from CompressgnnNorm import Compressgnn_LayerNorm, layer_norm, norm_act_dropout
from rows_reference import Reference, assert_near, factors, host, mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
TYPES = [F32, F64, F16, BF16]
# one row and one column, ends inside and at the packs and lane groups of every type, rows of many waves, rows longer than any group holds
SHAPES = [(1, 1), (3, 1), (5, 2), (2, 3), (300, 4), (7, 5), (1000, 7), (65, 8), (13, 9), (40, 15), (257, 16), (33, 17), (100, 31), (64, 33),
          (1000, 47), (129, 64), (31, 65), (2708, 128), (50, 129), (100, 255), (300, 256), (41, 257), (9, 511), (20, 513), (33, 602),
          (5, 1023), (6, 1025), (700, 1024), (3, 1030), (5, 1500), (7, 1200), (17, 2047), (4, 2050), (4, 2600), (5, 3050), (3, 4096), (2, 4103), (5, 8191), (2, 8200), (1, 12345),
          (2, 16384), (3, 20001),
          # more rows than lanes at once, each width of the above but the longest
          (270000, 5), (70003, 17), (40000, 40), (20000, 70), (20000, 130), (9000, 200), (5000, 390), (2600, 601), (1100, 1100), (1030, 700),
          (1030, 900)]


def features(rows, width, dtype, seed, offset=0.3):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=gen, dtype=F64) * (0.5 + torch.rand(rows, 1, generator=gen, dtype=F64)) + offset
    return x.to(dtype).to(DEV)


def parameters(width, dtype, seed):
    gen = torch.Generator().manual_seed(1000 + seed)
    w, b = 1 + 0.3 * torch.randn(width, generator=gen), 0.2 * torch.randn(width, generator=gen)
    return w.to(dtype).to(DEV), b.to(dtype).to(DEV)


def leaves(*tensors):
    return [None if t is None else t.detach().requires_grad_() for t in tensors]


# ------------------------------------------------------------------------- dropout --
def check_dropout(got, x, factor):
    """A product by the scale, rounded to float (double), and once to the type: bit for bit what the host computes."""
    wide = F64 if x.dtype == F64 else F32
    kept = torch.from_numpy(factor > 0)
    scale = torch.tensor(factor.max() if factor.size else 0.0, dtype=wide)
    want = torch.where(kept, x.detach().cpu().to(wide) * scale, torch.zeros((), dtype=wide)).to(x.dtype)
    assert torch.equal(got.detach().cpu(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [s for s in SHAPES if s[0] * s[1] < 20000])
def test_dropout_is_its_definition(dtype, rows, width):
    for p, seed, offset in [(0.5, 1, 0), (0.1, (1 << 62) + 5, 1 << 40), (0.9, -7, -3)]:
        x = features(rows, width, dtype, rows + width).requires_grad_()
        factor = factors(rows, width, p, seed, offset)
        out = dropout(x, p, seed, offset)
        assert out.dtype == dtype and out.shape == x.shape and out.is_contiguous()
        check_dropout(out, x, factor)
        grad = features(rows, width, dtype, 5)
        (dx,) = torch.autograd.grad(out, x, grad)
        check_dropout(dx, grad, factor)
        check_dropout(abi.dropout(x.detach(), p, seed, offset), x, factor)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_of_everything_and_of_nothing(dtype):
    x = features(37, 50, dtype, 1)
    assert not dropout(x, 1.0, 3).any() and torch.equal(dropout(x, 0.0, 3), x) and torch.equal(dropout(x, 1e-7, 3), x)
    for shape in [(0,), (0, 5), (5, 0), (2, 0, 3), (0, 0)]:
        empty = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
        out = dropout(empty, 0.5, 1)
        assert out.shape == empty.shape
        (dx,) = torch.autograd.grad(out, empty, torch.zeros_like(out))
        assert dx.shape == empty.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_dropped_elements_are_zero_whatever_they_hold(dtype):
    kept = mask(20, 33, 0.5, 9, 0)
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max, -0.0):
        out = dropout(torch.full((20, 33), value, dtype=dtype, device=DEV), 0.5, 9).cpu()
        assert not out[~torch.from_numpy(kept)].any()
        want = torch.full((), value, dtype=F64 if dtype == F64 else F32).mul(2).to(dtype)
        assert torch.equal(torch.nan_to_num(out[torch.from_numpy(kept)], nan=7.0), torch.nan_to_num(want, nan=7.0).expand(int(kept.sum())))


def layouts(x):
    """The same values in other places: rows further apart, not at a multiple of 16 bytes, transposed, more dimensions"""
    rows, width = x.shape
    for pad, shift in [(3, 0), (5, 1), (64, 3)]:
        wide = torch.full((rows, width + pad), 7.0, dtype=x.dtype, device=x.device)
        view = wide[:, shift:shift + width]
        view.copy_(x)
        yield view
    flat = torch.empty(rows * width + 1, dtype=x.dtype, device=x.device)[1:].view(rows, width)
    yield flat.copy_(x)
    yield x.t().contiguous().t()
    yield x.repeat_interleave(2, dim=1)[:, ::2]
    yield x.repeat_interleave(3, dim=0)[::3]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 7), (23, 1), (50, 64), (33, 602), (6, 1030), (3, 8200)])
def test_rows_anywhere_give_the_same_bits(dtype, rows, width):
    x, grad = features(rows, width, dtype, 1), features(rows, width, dtype, 2)
    w, b = parameters(width, dtype, 3)
    call = (1e-5, "relu", 0.4, 11, 5)
    want = norm_act_dropout(*(l := leaves(x, w, b)), *call)
    want_grads = torch.autograd.grad(want, l, grad)
    want_drop = dropout(x, 0.4, 11, 5)
    for there, grad_there in zip(layouts(x), reversed(list(layouts(grad)))):
        assert torch.equal(dropout(there, 0.4, 11, 5), want_drop)
        l = leaves(there, w.repeat_interleave(2)[::2], b)
        out = norm_act_dropout(*l, *call)
        assert out.is_contiguous() and torch.equal(out, want)
        for got, should in zip(torch.autograd.grad(out, l, grad_there), want_grads):
            assert torch.equal(got, should)
    cube = leaves(x.view(1, rows, 1, width))[0]
    out = norm_act_dropout(cube, w, b, *call)
    assert torch.equal(out.view(rows, width), want) and out.shape == cube.shape
    assert torch.equal(torch.autograd.grad(out, cube, grad.view(cube.shape))[0].view(rows, width), want_grads[0])
    line = leaves(x[0])[0]
    out = norm_act_dropout(line, w, b, *call)
    assert torch.equal(out, want[0])
    assert torch.equal(torch.autograd.grad(out, line, grad[0])[0], want_grads[0][0])


def test_a_gradient_that_is_one_number_for_all_elements():
    x, = leaves(features(50, 33, F32, 1))
    w, b = leaves(*parameters(33, F32, 1))
    (layer_norm(x, w, b) * 1.0).sum().backward()
    got = x.grad.clone(), w.grad.clone(), b.grad.clone()
    for g, want in zip(got, torch.autograd.grad(layer_norm(x, w, b), (x, w, b), torch.ones(50, 33, device=DEV))):
        assert torch.equal(g, want)
    layer_norm(x, w, b).sum().backward()  # expanded: all strides 0
    assert torch.equal(w.grad, 2 * got[1])


# ---------------------------------------------------------------------- layer norm --
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype,params", [(F32, F32), (F64, F64), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_norm_and_gradients_match_the_formulas(dtype, params, rows, width):
    for relu, p in [(False, 0.0), (True, 0.0), (False, 0.3), (True, 0.5)]:
        x, grad = features(rows, width, dtype, rows + width), features(rows, width, dtype, 7, offset=0.0)
        w, b = parameters(width, params, width)
        factor = factors(rows, width, p, 21, 2)
        want = Reference(x, w, b, 1e-5, relu, factor, grad)
        assert want.nearest_zero > 1e-12  # which side of zero the reference is on is no matter of rounding
        l = leaves(x, w, b)
        if p:
            out = norm_act_dropout(*l, 1e-5, "relu" if relu else None, p, 21, 2)
        else:
            out = norm_act_dropout(*l, activation="relu") if relu else layer_norm(*l)
        assert out.dtype == dtype and out.shape == x.shape
        assert_near(out, want.out, want.out_bound, "out")
        dx, dw, db = torch.autograd.grad(out, l, grad)
        assert dx.dtype == dtype and dw.dtype == params and db.dtype == params
        assert_near(dx, want.dx, want.dx_bound, "dx")
        assert_near(dw, want.dweight, want.dweight_bound, "dweight")
        assert_near(db, want.dbias, want.dbias_bound, "dbias")
        drop = abi.drop_struct(p, 21, 2)
        same, stats = abi.layer_norm(x, w, b, 1e-5, relu, drop)
        assert torch.equal(same, out)
        for got, should in zip(abi.layer_norm_backward(grad, x, stats, w, b, relu, drop), (dx, dw, db)):
            assert torch.equal(got, should)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 100, 2050, 8200])
def test_parameters_that_are_not_there(dtype, width):
    rows = 19
    x, grad = features(rows, width, dtype, 3), features(rows, width, dtype, 4)
    w, b = parameters(width, dtype, 5)
    for weight, bias in [(None, None), (w, None), (None, b)]:
        want = Reference(x, weight, bias, 1e-3, True, factors(rows, width, 0.2, 1, 1), grad)
        l = leaves(x, weight, bias)
        out = norm_act_dropout(*l, 1e-3, "relu", 0.2, 1, 1)
        assert_near(out, want.out, want.out_bound, "out")
        grads = torch.autograd.grad(out, [t for t in l if t is not None], grad)
        for got, should, bound in zip(grads, [want.dx] + [want.dweight] * (weight is not None) + [want.dbias] * (bias is not None),
                                      [want.dx_bound] + [want.dweight_bound] * (weight is not None) + [want.dbias_bound] * (bias is not None)):
            assert_near(got, should, bound, "gradient")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 64), (500, 40), (64, 2050), (5, 9000)])
def test_gradients_one_at_a_time_are_those_of_all(dtype, rows, width):
    x, grad = features(rows, width, dtype, 3), features(rows, width, dtype, 4)
    w, b = parameters(width, F32, 5)
    call = (1e-5, "relu", 0.5, 4, 4)
    every = torch.autograd.grad(norm_act_dropout(*(l := leaves(x, w, b)), *call), l, grad)
    for k in range(3):
        l = [x, w, b]
        l[k] = l[k].detach().requires_grad_()
        out = norm_act_dropout(*l, *call)
        assert torch.equal(torch.autograd.grad(out, l[k], grad)[0], every[k])
    l = leaves(x, w, b)
    out = norm_act_dropout(*l, *call)
    for k in (2, 0, 1):
        assert torch.equal(torch.autograd.grad(out, l[k], grad, retain_graph=True)[0], every[k])
    with torch.no_grad():
        assert not norm_act_dropout(*l, *call).requires_grad
    assert torch.equal(norm_act_dropout(x, w, b, *call), out)


@pytest.mark.parametrize("rows,width", [(3, 5), (4, 8), (2, 33)])
def test_gradients_match_differences(rows, width):
    x, (w, b) = features(rows, width, F64, 3), parameters(width, F64, 5)
    l = leaves(x, w, b)
    for activation, p in [(None, 0.0), (None, 0.5), ("relu", 0.4)]:
        assert torch.autograd.gradcheck(lambda *a: norm_act_dropout(*a, 1e-5, activation, p, 3, 1), l, eps=1e-6, atol=1e-6, rtol=1e-5)
    assert torch.autograd.gradcheck(lambda a: dropout(a, 0.5, 3, 1), l[:1])


def test_many_rows_are_summed_without_loss():
    """The parameters' sums over 600,000 rows: no further from 64 bits than the bound for chains of 1,024 additions."""
    for dtype, width in [(F32, 12), (F16, 30)]:
        x, grad = features(600001, width, dtype, 3), features(600001, width, dtype, 4, offset=0.5)
        w, b = parameters(width, F32, 1)
        want = Reference(x, w, b, 1e-5, True, np.ones((600001, width)), grad)
        l = leaves(x, w, b)
        got = torch.autograd.grad(norm_act_dropout(*l, 1e-5, "relu"), l, grad)
        assert_near(got[0], want.dx, want.dx_bound, "dx")
        assert_near(got[1], want.dweight, want.dweight_bound, "dweight")
        assert_near(got[2], want.dbias, want.dbias_bound, "dbias")


@pytest.mark.parametrize("width", [1, 4, 100, 1000, 3000, 9001])
def test_rows_that_hold_one_value(width):
    """Nothing to normalise: the output is the bias, the gradient of x what the formula leaves of it, no division by zero."""
    w, b = parameters(width, F32, 2)
    x = torch.tensor([[0.0], [1.5], [-3e4], [1e30]], device=DEV).expand(4, width).contiguous()
    l = leaves(x, w, b)
    out = layer_norm(*l, 1e-5)
    assert torch.equal(out, b.expand(4, width))
    grad = features(4, width, F32, 3)
    dx, dw, db = torch.autograd.grad(out, l, grad)
    assert not dw.any() and torch.isfinite(dx).all()
    want = Reference(x, w, b, 1e-5, False, np.ones((4, width)), grad)
    assert_near(db, want.dbias, want.dbias_bound, "dbias")
    # eps 0: 1 / sqrt(0) times 0 is no number, as in the formula; the other rows stay
    x[1:] = features(3, width, F32, 1)
    out = layer_norm(x, w, b, 0.0)
    assert torch.isnan(out[0]).all() and (width == 1 or torch.isfinite(out[1:]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_one_element_have_no_gradient(dtype):
    """Nothing of a row is left when its mean is taken away: zeros, not the rest of a cancellation."""
    for rows in (1, 3, 500, 70001):
        x, grad = features(rows, 1, dtype, 3), features(rows, 1, dtype, 4)
        l = leaves(x, *parameters(1, dtype, 2))
        for activation, p in ((None, 0.0), ("relu", 0.4)):
            dx, dw, _ = torch.autograd.grad(norm_act_dropout(*l, 1e-5, activation, p, 5), l, grad)
            assert not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 64, 300, 2500, 9000])
def test_rows_without_a_finite_mean_stay_among_themselves(dtype, width):
    x, grad = features(9, width, dtype, 1), features(9, width, dtype, 2)
    w, b = parameters(width, dtype, 1)
    clean = norm_act_dropout(*(l := leaves(x, w, b)), 1e-5, "relu", 0.5, 3)
    clean_dx = torch.autograd.grad(clean, l[0], grad)[0]
    broken = x.clone()
    broken[1, 0], broken[4, width // 2], broken[8, -1] = float("nan"), float("inf"), -float("inf")
    l = leaves(broken, w, b)
    out = norm_act_dropout(*l, 1e-5, "relu", 0.5, 3)
    dx = torch.autograd.grad(out, l[0], grad)[0]
    good = [0, 2, 3, 5, 6, 7]
    assert torch.equal(out[good], clean[good]) and torch.equal(dx[good], clean_dx[good])
    kept = torch.from_numpy(mask(9, width, 0.5, 3, 0)).to(DEV)
    for r in (1, 4, 8):
        assert torch.isnan(out[r][kept[r]]).all() and not out[r][~kept[r]].any()


@pytest.mark.parametrize("width", [16, 200, 1500, 10000])
def test_small_spread_on_a_large_offset(width):
    """Values whose spread is a millionth of their mean: sums in float would leave nothing of it."""
    gen = torch.Generator().manual_seed(1)
    x = (1e4 + 0.01 * torch.randn(7, width, generator=gen, dtype=F64)).to(F32).to(DEV)
    w, b = parameters(width, F32, 1)
    want = Reference(x, w, b, 1e-8, False, np.ones((7, width)), grad := features(7, width, F32, 4))
    l = leaves(x, w, b)
    out = layer_norm(*l, 1e-8)
    assert_near(out, want.out, want.out_bound, "out")
    assert_near(torch.autograd.grad(out, l[0], grad)[0], want.dx, want.dx_bound, "dx")
    huge = features(3, width, F32, 2) * 1e37  # squares beyond float
    want = Reference(huge, w, b, 1e-5, False, np.ones((3, width)))
    assert_near(layer_norm(huge, w, b), want.out, want.out_bound, "out of huge rows")
    tiny = features(3, width, F32, 2, offset=0.0) * 1e-30  # squares below float
    want = Reference(tiny, w, b, 0.0, False, np.ones((3, width)))
    assert_near(layer_norm(tiny, w, b, 0.0), want.out, want.out_bound, "out of tiny rows")


def test_rows_beyond_32_bit_offsets():
    rows, width = (1 << 31) // 257 + 100, 257
    x = torch.empty(rows, width, dtype=BF16, device=DEV)
    x.normal_(generator=torch.Generator(DEV).manual_seed(1))
    out = dropout(x, 0.5, 3, 1)
    at = torch.tensor([0, rows // 2, rows - 2, rows - 1], device=DEV)
    for r in at.tolist():
        kept = torch.from_numpy(mask(1, width, 0.5, 3, 1, first_row=r)[0]).to(DEV)
        assert torch.equal(out[r], torch.where(kept, x[r] * 2, torch.zeros((), dtype=BF16, device=DEV)))
    del out
    l = leaves(x)
    out = layer_norm(l[0])
    small = leaves(x[at])[0]
    small_out = layer_norm(small)
    assert torch.equal(out[at], small_out)
    dx = torch.autograd.grad(out, l[0], x)[0]
    assert torch.equal(dx[at], torch.autograd.grad(small_out, small, x[at])[0])


@pytest.mark.parametrize("rows,dtype", [((1 << 21) + 77, BF16), (300007, F32)])
def test_matrices_beyond_the_caches(rows, dtype):
    """Whole lines, more of them than the last-level cache holds: other stores, and from a gigabyte on another way through the rows."""
    width = 256
    gen = torch.Generator(DEV).manual_seed(1)
    x, grad = (torch.randn(rows, width, device=DEV, generator=gen, dtype=F32).to(dtype) for _ in range(2))
    w, b = parameters(width, F32, 1)
    out = dropout(x, 0.5, 3, 1)
    zero = torch.zeros((), dtype=dtype, device=DEV)
    assert bool(((out == zero) | (out == x * 2)).all())
    at = torch.cat([torch.arange(0, 300), torch.arange(rows // 2, rows // 2 + 100), torch.arange(rows - 300, rows)]).to(DEV)
    for first, last in ((0, 300), (rows // 2, rows // 2 + 100), (rows - 300, rows)):
        kept = torch.from_numpy(mask(last - first, width, 0.5, 3, 1, first_row=first)).to(DEV)
        assert torch.equal(out[first:last], torch.where(kept, x[first:last] * 2, zero))
    del out
    l = leaves(x, w, b)
    out = norm_act_dropout(*l, 1e-5, "relu")
    dx, dw, db = torch.autograd.grad(out, l, grad)
    small = leaves(x[at], w, b)
    small_out = norm_act_dropout(*small, 1e-5, "relu")
    assert torch.equal(out[at], small_out)
    assert torch.equal(dx[at], torch.autograd.grad(small_out, small[0], grad[at])[0])
    off, sums = 0.0, [torch.zeros(width, dtype=F64, device=DEV) for _ in range(4)]
    for first in range(0, rows, 1 << 18):  # every row against 64 bits, the sums against theirs
        X, G = x[first:first + (1 << 18)].double(), grad[first:first + (1 << 18)].double()
        h = X - X.mean(1, keepdim=True)
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
        v = h * w.double() + b.double()
        G = G * (v > 0)
        off = max(off, float((out[first:first + (1 << 18)].double() - v.clamp_min(0)).abs().max()))
        for total, part in zip(sums, (G * h, (G * h).abs(), G, G.abs())):
            total += part.sum(0)
    # a value of at most 32: half a step of its type and a few of float
    assert off <= 32 * ({BF16: 2.0 ** -8, F32: 2.0 ** -24}[dtype] + 8 * 2.0 ** -24)
    for got, want, size in ((dw, sums[0], sums[1]), (db, sums[2], sums[3])):
        assert bool(((got.double() - want).abs() <= (1024 + 68) * 2.0 ** -24 * size).all())


# -------------------------------------------------------------- streams, graphs, autograd --
def test_other_streams_and_repeated_calls_give_the_same_bits():
    x, grad = features(3000, 130, F32, 1), features(3000, 130, F32, 2)
    w, b = parameters(130, F32, 1)
    call = (1e-5, "relu", 0.5, 8, 8)

    def step():
        l = leaves(x, w, b)
        out = norm_act_dropout(*l, *call)
        return [out.detach(), *torch.autograd.grad(out, l, grad)]

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(step())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(g, t) for g, t in zip(got, want))


def test_captured_steps_replay():
    """Forward and gradients in a graph, with eager work of the same operators between the replays."""
    x, grad = features(777, 65, F32, 1), features(777, 65, F32, 2)
    w, b = parameters(65, F32, 1)
    call = (1e-5, "relu", 0.25, 8, 8)

    def step(inputs):
        l = leaves(*inputs)
        out = norm_act_dropout(*l, *call)
        return [out.detach(), *torch.autograd.grad(out, l, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step((x, w, b))
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step((x, w, b)))
        graphs.append(graph)
    for k in range(4):
        x.copy_(features(777, 65, F32, 10 + k))
        for graph in graphs:
            graph.replay()
        want = step((x, w, b))
        torch.cuda.synchronize()
        for got in held:
            assert all(torch.equal(g, t) for g, t in zip(got, want)), k


def test_masks_of_a_captured_module_differ_from_replay_to_replay():
    x = torch.ones(64, 40, device=DEV)
    drop = Compressgnn_Dropout(0.5, seed=5)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            drop(x)
    drop.to(DEV)
    eager = drop(x)
    assert torch.equal(eager, torch.from_numpy(factors(64, 40, 0.5, 5, 0)).to(F32).to(DEV))
    graph = torch.cuda.CUDAGraph()
    leaf = x.clone().requires_grad_()
    with torch.cuda.graph(graph):
        first, second = drop(leaf), drop(leaf)
        (dx,) = torch.autograd.grad(second, leaf, x)
    for k in range(3):
        graph.replay()
        for n, got in ((2 * k, first), (2 * k + 1, second), (2 * k + 1, dx)):
            assert torch.equal(got.detach(), torch.from_numpy(factors(64, 40, 0.5, 5, (1 << 62) + n)).to(F32).to(DEV)), (k, n)
    assert drop.calls == 1
    assert torch.equal(drop(x), torch.from_numpy(factors(64, 40, 0.5, 5, 1)).to(F32).to(DEV))


def test_a_counter_on_the_device_is_added_to_the_offset():
    x = features(30, 20, F32, 1).requires_grad_()
    counter = torch.tensor([1 << 33], device=DEV)
    out = dropout(x, 0.5, 4, -5, counter)
    check_dropout(out, x, factors(30, 20, 0.5, 4, (1 << 33) - 5))
    normed = norm_act_dropout(x, p=0.5, seed=4, offset=-5, counter=counter)
    assert torch.equal(normed == 0, out == 0)
    counter += 1
    for late in (out, normed):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(late.sum(), x)
    for bad in (torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(1, device=DEV), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(RuntimeError, match="counter has to be"):
            dropout(x, 0.5, 4, 0, bad)
        with pytest.raises(RuntimeError, match="counter has to be"):
            norm_act_dropout(x, p=0.5, counter=bad)


def test_autograd_contract():
    x, (w, b) = features(20, 12, F32, 1), parameters(12, F32, 1)
    l = leaves(x, w, b)
    for out in (norm_act_dropout(*l, 1e-5, "relu", 0.5, 3), dropout(l[0], 0.5, 3)):
        (dx,) = torch.autograd.grad(out.sum(), l[0], create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            dx.sum().backward()
    # what is kept may not be written to before the gradient
    for k in (0, 1, 2):
        l = leaves(x, w, b)
        inner = [t * 1.0 for t in l]
        out = norm_act_dropout(*inner, 1e-5, "relu", 0.5, 3)
        with torch.no_grad():
            inner[k].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), l[0])
    out = norm_act_dropout(*(l := leaves(x, w, b)), 1e-5, "relu", 0.5, 3)
    out.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    # forward-mode tangents and the transforms of torch.func are refused, not answered wrongly
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: dropout(t, 0.5, 3), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layer_norm(t))(x.view(4, 5, 12))
    # under saved-tensor hooks nothing of the size of x is kept but x
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel()) or t, lambda t: t):
        norm_act_dropout(*leaves(x, w, b), 1e-5, "relu", 0.5, 3)
    assert sorted(sizes) == [12, 12, 40, 240]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel()) or t, lambda t: t):
        dropout(leaves(x)[0], 0.5, 3)
    assert len(sizes) == 4


def test_a_trace_records_the_operators():
    x = features(20, 12, F32, 1)
    norm = Compressgnn_LayerNorm(12, activation="relu").to(DEV)
    traced = torch.jit.trace(norm, (x,), check_trace=False)
    y = features(20, 12, F32, 2)
    assert torch.equal(traced(y), norm(y))


def test_refusals_on_the_device():
    x, (w, b) = features(4, 6, F32, 1), parameters(6, F32, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(RuntimeError, match="p has to lie"):
            dropout(x, p, 1)
        with pytest.raises(RuntimeError, match="p has to lie"):
            norm_act_dropout(x, p=p)
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="eps has to be"):
            layer_norm(x, eps=eps)
    for weight in (w[:5], w.double(), w.half(), w.view(1, 6), w.cpu(), torch.ones(6, dtype=torch.int64, device=DEV)):
        with pytest.raises(RuntimeError, match="weight has to be a vector"):
            layer_norm(x, weight, b)
    with pytest.raises(RuntimeError, match="of one type"):
        layer_norm(x.half(), w, b.half())
    with pytest.raises(RuntimeError, match="no last dimension"):
        layer_norm(x[0, 0])
    with pytest.raises(RuntimeError, match="has to be a float32"):
        dropout(x.to(torch.int32), 0.5, 1)
    out, stats = rt.layer_norm_forward(x, w, b, 1e-5)
    for grad, s in [(x[:3], stats), (x.half(), stats), (x, stats[:3]), (x, stats.float()), (x.cpu(), stats)]:
        with pytest.raises(RuntimeError):
            rt.layer_norm_backward(grad, x, s, w, b)


def test_no_rows_and_no_columns():
    for dtype in TYPES:
        for shape in [(0, 5), (0,), (3, 0), (0, 0), (2, 0, 4)]:
            x = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
            w, b = leaves(*parameters(shape[-1], dtype, 1))
            out = norm_act_dropout(x, w, b, 1e-5, "relu", 0.5, 1)
            assert out.shape == x.shape
            dx, dw, db = torch.autograd.grad(out, (x, w, b), torch.zeros_like(out))
            assert dx.shape == x.shape and dw.shape == w.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("width", [2100, 2700, 3500])
def test_many_wide_16_bit_rows_are_what_few_are(width, dtype):
    """Few rows, whose values the formulas check above, are spread over more lanes.  Two roundings of half a step each, of values that are
    2^-20 of the bias apart at most; below the least normal number of float16 half a step is 2^-25."""
    rows, few = 4100, 200
    x = features(rows, width, dtype, 1)
    w, b = parameters(width, F32, 1)

    def near(many, one):
        bound = torch.finfo(dtype).eps * one.double().abs() + 2.0 ** -20 * b.abs().max().double() + 2.0 ** -24
        assert ((many.double() - one.double()).abs() <= bound).all()

    call = (w, b, 1e-5, "relu")
    near(norm_act_dropout(x, *call, 0.5, 3, 1)[:few], norm_act_dropout(x[:few], *call, 0.5, 3, 1))
    near(norm_act_dropout(x, *call)[-few:], norm_act_dropout(x[-few:], *call))
    near(layer_norm(x, w, b)[-few:], layer_norm(x[-few:], w, b))


# ---------------------------------------------------------------------------- modules --
def test_modules():
    x = features(50, 24, F32, 1)
    drop = Compressgnn_Dropout(0.25, seed=77)
    for n in range(3):
        check_dropout(drop(x), x, factors(50, 24, 0.25, 77, n))
    again = Compressgnn_Dropout(0.25, seed=0)
    again.load_state_dict(drop.state_dict())
    assert torch.equal(again(x), drop(x))
    drop.eval()
    assert drop(x) is x
    norm = Compressgnn_LayerNorm(24, activation="relu", p=0.5, seed=9).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(parameters(24, F32, 1)[0])
        norm.bias.copy_(parameters(24, F32, 1)[1])
    for n in range(2):
        assert torch.equal(norm(x), norm_act_dropout(x, norm.weight, norm.bias, 1e-5, "relu", 0.5, 9, n))
        assert torch.equal(norm(x.half()), norm_act_dropout(x.half(), norm.weight, norm.bias, 1e-5, "relu", 0.5, 9, 2 * n + 1)) or n
        norm.calls = n + 1
    norm.eval()
    assert torch.equal(norm(x), norm_act_dropout(x, norm.weight, norm.bias, 1e-5, "relu"))
    plain = Compressgnn_LayerNorm(24, affine=False, dtype=F64)
    assert torch.equal(plain(x.double()), layer_norm(x.double()))


@pytest.mark.parametrize("reentrant", [False, True])
def test_activations_computed_again(reentrant):
    """Masks with names are the same the second time; a module, which counts its calls, refuses the second one."""
    x, grad = features(90, 40, F32, 1), features(90, 40, F32, 2)
    w, b = parameters(40, F32, 1)

    def block(x, w, b):
        return dropout(norm_act_dropout(x, w, b, 1e-5, "relu", 0.25, 3, 1), 0.5, 3, 2)

    l, k = leaves(x, w, b), leaves(x, w, b)
    want = torch.autograd.grad(block(*l), l, grad)
    out = torch.utils.checkpoint.checkpoint(block, *k, use_reentrant=reentrant)
    out.backward(grad)
    assert all(torch.equal(t.grad, g) for t, g in zip(k, want))
    drop, norm = Compressgnn_Dropout(0.5, seed=4).to(DEV), Compressgnn_LayerNorm(40, p=0.5).to(DEV)
    for module in (drop, norm, lambda x: drop(x).square()):
        (k,) = leaves(x)
        calls = drop.calls
        out = torch.utils.checkpoint.checkpoint(module, k, use_reentrant=reentrant)
        if module is drop and not reentrant:  # keeps no tensor, so nothing is computed again
            out.backward(grad)
            assert torch.equal(k.grad, dropout(grad, 0.5, 4, calls))
            continue
        with pytest.raises(RuntimeError, match="within a backward pass"):
            out.backward(grad)
    plain = Compressgnn_LayerNorm(40, activation="relu").to(DEV)
    (l,), (k,) = leaves(x), leaves(x)
    plain(l).backward(grad)
    torch.utils.checkpoint.checkpoint(plain, k, use_reentrant=reentrant).backward(grad)
    assert torch.equal(l.grad, k.grad)


def test_the_fused_operator_is_the_two_in_a_row():
    """In double nothing is rounded between them; the mask is the same in any type."""
    x, (w, b) = features(70, 50, F64, 1), parameters(50, F64, 1)
    grad = features(70, 50, F64, 2)
    l = leaves(x, w, b)
    fused = norm_act_dropout(*l, 1e-5, "relu", 0.4, 3, 2)
    fused_grads = torch.autograd.grad(fused, l, grad)
    apart = dropout(layer_norm(*l).relu(), 0.4, 3, 2)
    assert torch.allclose(fused, apart, rtol=1e-15, atol=0)
    for a, c in zip(fused_grads, torch.autograd.grad(apart, l, grad)):
        assert torch.allclose(a, c, rtol=1e-12, atol=1e-13)


def test_between_the_layers_of_a_model():
    """propagate -> cluster -> Linear -> norm + ReLU on the representatives -> reconstruct -> dropout -> propagate ->
    norm -> Linear, with its gradients, against the same in 64 bits of plain torch operators."""
    import compressgnn_offline as off
    from CompressgnnCluster import Compressgnn_Cluster
    from CompressgnnData import CompressgnnData
    from CompressgnnReconstruct import Compressgnn_Reconstruct
    from KPropagate import KPropagate
    v, e = off.gen_chung_lu(2708, 10500, 2.5, 0)
    V, F, H, C = 2708, 40, 24, 7
    m = np.ones(V, dtype=bool)
    data = CompressgnnData(np.zeros((V, F), np.float32), (v, e), np.zeros(V, np.int64), m, m, m, graph_type="csr", min_pair_frequency=3)
    data.edge_index.to(DEV)
    v2, e2 = off.add_self_loop_csr(v, e)  # as the loader does, with the weights it gives the edges
    degree = off.get_norm_degree(e2, V).astype(np.float64)
    rows = np.repeat(np.arange(V), np.diff(v2))
    src, dst = torch.from_numpy(rows).to(DEV), torch.from_numpy(e2.astype(np.int64)).to(DEV)
    weights = torch.from_numpy(degree[rows] * degree[e2]).to(DEV).unsqueeze(1)

    def plain_propagate(t):
        return torch.zeros_like(t).index_add_(0, dst, weights * t.index_select(0, src))

    P = KPropagate()

    def hop(t):
        return P(t, data.edge_index, None, data.vertex_cnt, data.rule_cnt)

    torch.manual_seed(1)
    x = torch.randn(V, F, device=DEV, requires_grad=True)
    cluster = Compressgnn_Cluster(in_feature=F, param_H=9, training=True, cache=True, refresh_interval=1).to(DEV)
    reconstruct, lin, out_lin = Compressgnn_Reconstruct(), torch.nn.Linear(F, H).to(DEV), torch.nn.Linear(H, C).to(DEV)
    norm = Compressgnn_LayerNorm(H, activation="relu").to(DEV)
    drop, last = Compressgnn_Dropout(0.5, seed=4), Compressgnn_LayerNorm(H, activation="relu", p=0.25, seed=6).to(DEV)
    reps, index = cluster(hop(x), epoch=0)
    hidden = drop(reconstruct(norm(lin(reps)), index))
    out = out_lin(last(hop(hidden)))
    grad = torch.randn(V, C, device=DEV)
    params = [x, *lin.parameters(), *norm.parameters(), *last.parameters(), *out_lin.parameters()]
    got = torch.autograd.grad(out, params, grad)

    wide = [t.detach().double().requires_grad_() for t in params]
    x64, w1, b1, nw, nb, lw, lb, w2, b2 = wide

    def plain_norm(t, w, b):
        c = t - t.mean(1, keepdim=True)
        return (c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w + b).relu()

    t = plain_propagate(x64)
    groups = int(index.max()) + 1
    counts = torch.bincount(index, minlength=groups).clamp_min(1).double()
    t = torch.zeros(groups, F, dtype=F64, device=DEV).index_add_(0, index, t) / counts[:, None]
    # rows that are copies are normalised alike: the plain model normalises every row behind the gather
    t = plain_norm((t @ w1.t() + b1).index_select(0, index), nw, nb) * torch.from_numpy(factors(V, H, 0.5, 4, 0)).to(DEV)
    t = plain_norm(plain_propagate(t), lw, lb) * torch.from_numpy(factors(V, H, 0.25, 6, 0)).to(DEV)
    want_out = t @ w2.t() + b2
    want = torch.autograd.grad(want_out, wide, grad.double())
    for a, c in zip([out, *got], [want_out, *want]):
        scale = float(c.detach().abs().max())
        assert float((a.detach().double() - c.detach()).abs().max()) <= 1e-4 * scale
