"""Layer norm and dropout on the GPU at the ends of their range: sizes, sums and shapes that single steps of them are chosen by."""
import numpy as np
import pytest
import torch

import compressgnn_runtime as rt
from CompressgnnDropout import Compressgnn_Dropout, dropout
from CompressgnnNorm import Compressgnn_LayerNorm, norm_act_dropout
from row_shapes import SPREAD, many
from rows_reference import SMALLEST, UNIT, factors, mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


def normal(shape, dtype, seed):
    """Made in the type itself: no copy of a large matrix in another."""
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(seed))


def test_sums_of_more_columns_than_one_launch_has_threads_for():
    """65 rows are two parts, whose sums over 2^25 + 24 columns of the weight's and the bias's gradient take workgroups of several sixteens.
    A part's lane adds 16 rows, four of them a part, and the two parts are added in 64 bits."""
    rows, width = 65, (1 << 25) + 24
    x, grad = normal((rows, width), BF16, 1), normal((rows, width), BF16, 2)
    _, stats = rt.layer_norm_forward(x, None, None, 1e-5)
    _, dw, db = rt.layer_norm_backward(grad, x, stats, None, None)
    assert dw.dtype == BF16 and dw.shape == db.shape == (width,)
    mean, rstd = stats[:, :1], stats[:, 1:]
    for first in range(0, width, 1 << 21):
        columns = slice(first, min(width, first + (1 << 21)))
        g, h = grad[:, columns].double(), (x[:, columns].double() - mean) * rstd
        for got, terms in ((dw, g * h), (db, g)):
            want = terms.sum(0)
            off = (16 + 4 + 4) * 2.0 ** -24 * terms.abs().sum(0)  # chain, groups, and four roundings of a term
            bound = off + 2.0 ** -8 * (want.abs() + off) + 2.0 ** -133
            assert bool(((got[columns].double() - want).abs() <= bound).all()), first


def test_masks_of_more_rows_than_one_launch_has_threads_for():
    """A column of 2^33 + 1,000: the mask of a row is that of its place in the whole matrix, in the second launch and further ones too."""
    rows = (1 << 33) + 1000
    out = dropout(torch.ones(rows, 1, dtype=BF16, device=DEV), 0.5, 3, 1)
    launch = (1 << 31) // 256 * 512  # rows
    for first in [0, (1 << 32) - 100] + [k * launch - 100 for k in range(1, 3)] + [rows - 500]:
        kept = mask(200, 1, 0.5, 3, 1, first_row=first)
        assert torch.equal(out[first:first + 200].cpu(), torch.from_numpy(kept).to(BF16) * 2), first
    assert bool((out[-300:].cpu() == torch.from_numpy(mask(300, 1, 0.5, 3, 1, first_row=rows - 300)).to(BF16) * 2).all())
    for first in range(0, rows, 1 << 31):
        part = out[first:first + (1 << 31)].view(torch.int16)
        share = (part == 0x4000).sum(dtype=torch.int64) + (part == 0).sum(dtype=torch.int64)  # 2 or 0
        assert int(share) == part.numel(), first


@pytest.mark.parametrize("dtype,width", [(F32, 20_000_003), (BF16, 24_000_001), (F16, 9000), (F32, 8200)])
def test_sums_along_wide_rows_do_not_lose_with_the_width(dtype, width):
    """A gradient that is one number everywhere: its mean takes all of it away again, so what a chain of float additions along the row loses
    stays in dx.  Sums of a pack or two in float (16 additions at most), the rest in 64 bits: a bound without the width in it."""
    rows = 2
    x, g = normal((rows, width), dtype, 1), torch.full((rows, width), 0.1, dtype=dtype, device=DEV)
    g[1] *= 0.25
    _, stats = rt.layer_norm_forward(x, None, None, 1e-5)
    dx, _, _ = rt.layer_norm_backward(g, x, stats, None, None)
    G = g.double()
    X = x.double()
    mean = X.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((X - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    h = (X - mean) * rstd
    m1, m2, c1, c2 = G.mean(1, keepdim=True), (G * h).abs().mean(1, keepdim=True), G.mean(1, keepdim=True), (G * h).mean(1, keepdim=True)
    want = rstd * (G - c1 - h * c2)
    u = 2.0 ** -24
    # a value takes a handful of roundings, a sum 16 and a few more; 64-bit sums of 20 million terms in lanes of 20,000 lose 2^-36 at most
    off = rstd * (8 * u * (G + m1 + h.abs() * m2) + 20 * u * (m1 + h.abs() * m2)) + 2.0 ** -36 * rstd * (m1 + h.abs() * m2)
    bound = off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + 2.0 ** -24 * (dtype == F16) + 2.0 ** -133
    over = (dx.double() - want).abs() - bound
    assert float(over.max()) <= 0, (float((dx.double() - want).abs().max()), float(bound.min()))


@pytest.mark.parametrize("width", [3, 33, 100, 257, 1024, 1500, 4100, 8192, 20001])
@pytest.mark.parametrize("rows", [2, 2000])
def test_float64_statistics_with_an_outlier_in_front(rows, width):
    """The first element a million deviations of the others off: differences to it alone would leave log2(width) bits less of the variance.
    Lanes add up to width / 64 terms (longer rows: width / 1,024 and 16 waves' sums), then six steps across lanes; a square or a difference
    has two roundings."""
    x = normal((rows, width), F64, 1)
    x[:, 0] = 1e6
    _, stats = rt.layer_norm_forward(x, None, None, 0.0)
    exact = x[:2].cpu().numpy().astype(np.longdouble)  # 64 bits of mantissa
    mean = exact.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((exact - mean) ** 2).mean(1))
    got = stats[:2].cpu().numpy()
    steps = 4 + 24 + min(width, 4096) / 64 + width / 1024
    assert (np.abs(got[:, 0] - mean[:, 0]) <= steps * 2.0 ** -53 * np.abs(exact).mean(1)).all()
    assert (np.abs(got[:, 1] / rstd - 1) <= steps * 2.0 ** -53).all(), np.abs(got[:, 1] / rstd - 1) * 2.0 ** 53
    assert bool((stats[:, 1] - stats[0, 1]).abs().max() < 1e-3 * stats[0, 1])


# ------------------------------------------------------------------------- modules --
def test_a_module_in_training_is_not_traced():
    x = normal((20, 12), F32, 1)
    for module in (Compressgnn_Dropout(0.5).to(DEV), Compressgnn_LayerNorm(12, activation="relu", p=0.5).to(DEV)):
        with pytest.raises(RuntimeError, match="a trace would draw"):
            torch.jit.trace(module, (x,), check_trace=False)
        module.eval()
        traced = torch.jit.trace(module, (x,), check_trace=False)
        assert torch.equal(traced(2 * x), module(2 * x))
    # what the message names instead: masks that a counter on the device tells apart
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)
    traced = torch.jit.trace(lambda x, counter: dropout(x, 0.5, 3, 0, counter), (x, counter), check_trace=False)
    for n in range(3):
        counter.fill_(n)
        assert torch.equal(traced(x, counter), dropout(x, 0.5, 3, n))


# -------------------------------------------------------------------------- shapes --
def check(got, want, off, dtype, what):
    """Within `off` of the formula, and half a step of the type that it is rounded to."""
    bound = off + UNIT[dtype] * (want.abs() + off) + SMALLEST[dtype]
    over = (got.double() - want).abs() - bound
    assert got.dtype == dtype and got.shape == want.shape and bool(torch.isfinite(got).all()), what
    assert float(over.max()) <= 0, (what, float(over.max()), int((over > 0).sum()))


@pytest.mark.parametrize("dtype,params", [(F32, F32), (F64, F64), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("number", range(len(SPREAD)), ids=["%dx%d" % shape for shape in SPREAD])
def test_rows_of_several_packs_a_lane_match_the_formulas(dtype, params, number):
    """Outputs and gradients of matrices with more rows than the chip holds at a pack a lane, by formulas in 64 bits on the device and the bounds
    of rows_reference.Reference; masks from the host's generator."""
    for _, rows, width in many(dtype)[2 * number:2 * number + 2]:
        x = normal((rows, width), F32, width).mul_(0.5 + torch.rand(rows, 1, device=DEV, generator=torch.Generator(DEV).manual_seed(5))).add_(0.3).to(dtype)
        grad = normal((rows, width), dtype, 7)
        w, b = (1 + 0.3 * normal((width,), F32, 3)).to(params), (0.2 * normal((width,), F32, 4)).to(params)
        X, W, B, u = x.double(), w.double(), b.double(), 2.0 ** -53 if dtype == F64 else 2.0 ** -24
        mean = X.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt(((X - mean) ** 2).mean(1, keepdim=True) + 1e-5)
        h = (X - mean) * rstd
        h_off = (width + 16) * 2.0 ** -53 * (2 * rstd * X.abs().mean(1, keepdim=True) + 2 * h.abs())
        pre = h * W + B
        assert float(pre.abs().min()) > 1e-12  # which side of zero the formula is on is no matter of rounding
        for relu, p in [(False, 0.0), (True, 0.0), (False, 0.3), (True, 0.5)]:
            what = (rows, width, relu, p)
            factor = torch.from_numpy(factors(rows, width, p, 21, 2)).to(DEV) if p else torch.ones((), dtype=F64, device=DEV)
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            out = norm_act_dropout(*leaves, 1e-5, "relu" if relu else None, p, 21, 2)
            dx, dw, db = torch.autograd.grad(out, leaves, grad)
            gate = (pre > 0) * factor if relu else factor.expand(rows, width)
            check(out, pre * gate, factor * (8 * u * ((h * W).abs() + B.abs()) + h_off * W.abs()), dtype, ("out", *what))
            g = grad.double() * gate
            gw = g * W
            c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
            m1, m2 = gw.abs().mean(1, keepdim=True), (gw * h).abs().mean(1, keepdim=True)
            want = rstd * (gw - c1 - h * c2)
            off = rstd * (8 * u * (gw.abs() + m1 + h.abs() * m2) + (width / 64 + 16) * u * (m1 + h.abs() * m2) + 2 * h_off * m2
                          + h_off.mean(1, keepdim=True) * m1 * h.abs()) + want.abs() * (width + 16) * 2.0 ** -52
            check(dx, want, off, dtype, ("dx", *what))
            chain = min(rows, 1024) + 64 + 4
            check(dw, (g * h).sum(0), chain * u * (g * h).abs().sum(0) + (g.abs() * h_off).sum(0), params, ("dweight", *what))
            check(db, g.sum(0), chain * u * g.abs().sum(0), params, ("dbias", *what))
