"""Layer norm, ReLU and dropout of rows in 64 bits on the host, and how far a kernel may be from them: shared by the tests."""
import numpy as np
import torch

LOW = np.uint64(0xFFFFFFFF)
UNIT = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def philox(counter, key):
    """Philox4x32-10: four words for the four words of `counter` (arrays) and the two of `key`."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [int(w) for w in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept_share(p):
    return int(np.floor((1 - p) * 65536 + 0.5))


def mask(rows, width, p, seed, offset, first_row=0):
    """Truth values [rows, width]: which elements are kept."""
    blocks = -(-width // 8)
    n = np.arange(first_row * blocks, (first_row + rows) * blocks, dtype=np.uint64)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    words = philox([n & LOW, n >> np.uint64(32), np.full_like(n, offset & 0xFFFFFFFF), np.full_like(n, offset >> 32)],
                   [seed & 0xFFFFFFFF, seed >> 32])
    draws = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=-1)
    return (draws < kept_share(p)).reshape(rows, blocks * 8)[:, :width]


def factors(rows, width, p, seed, offset):
    share = kept_share(p)
    return np.where(mask(rows, width, p, seed, offset), 65536.0 / share if share else 0.0, 0.0)


def host(t):
    return t.detach().cpu().double().numpy()


class Reference:
    """Outputs and gradients of drop(relu(layer_norm(x))) in 64 bits, and bounds on the distance of a kernel that holds row
    statistics in 64 bits and computes the rest in float (double for double rows), rounded once to the type of an output.

    One float step is u = 2^-24.  A normalised value takes a handful of roundings (difference, product with the deviation,
    weight, bias, scale): 8 u of its largest term.  Sums over a row of F take at most F / 64 + 16 additions in one
    chain, sums over the rows at most 1,024 + 64."""

    def __init__(self, x, weight, bias, eps, relu, factor, grad=None):
        X = host(x)
        rows, width = X.shape
        w = np.ones(width) if weight is None else host(weight)
        b = np.zeros(width) if bias is None else host(bias)
        u = 2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -24
        mean = X.mean(1, keepdims=True)
        centred = X - mean
        rstd = 1 / np.sqrt((centred ** 2).mean(1, keepdims=True) + eps)
        h = centred * rstd
        # the mean itself is off by the additions of 64 bits that make it, here and there
        h_off = rstd * (width + 16) * 2.0 ** -53 * np.abs(X).mean(1, keepdims=True) * 2 + np.abs(h) * (width + 16) * 2.0 ** -52
        pre = h * w + b
        opened = ~(pre <= 0) if relu else np.ones_like(pre, dtype=bool)
        self.out = np.where(opened, pre, 0.0) * factor
        out_off = np.where(factor > 0, factor * (8 * u * (np.abs(h * w) + np.abs(b)) + h_off * np.abs(w)), 0.0)
        self.out_bound = self._rounded(self.out, out_off, x.dtype)
        self.nearest_zero = np.abs(pre).min() if pre.size else 1.0
        if grad is None:
            return
        g = np.where(opened, host(grad) * factor, 0.0)
        gw = g * w
        c1, c2 = gw.mean(1, keepdims=True), (gw * h).mean(1, keepdims=True)
        self.dx = rstd * (gw - c1 - h * c2)
        chain = width / 64 + 16
        m1, m2 = np.abs(gw).mean(1, keepdims=True), np.abs(gw * h).mean(1, keepdims=True)
        off = rstd * (8 * u * (np.abs(gw) + m1 + np.abs(h) * m2) + chain * u * (m1 + np.abs(h) * m2) + h_off * 2 * m2 + h_off.mean(1, keepdims=True) * m1 * np.abs(h))
        self.dx_bound = self._rounded(self.dx, off + np.abs(self.dx) * (width + 16) * 2.0 ** -52, x.dtype)
        kind = x.dtype if weight is None and bias is None else (weight if weight is not None else bias).dtype
        chain = min(rows, 1024) + 64
        self.dweight, self.dbias = (g * h).sum(0), g.sum(0)
        self.dweight_bound = self._rounded(self.dweight, (chain + 4) * u * np.abs(g * h).sum(0) + (np.abs(g) * h_off).sum(0), kind)
        self.dbias_bound = self._rounded(self.dbias, (chain + 4) * u * np.abs(g).sum(0), kind)

    @staticmethod
    def _rounded(value, off, dtype):
        return off + UNIT[dtype] * (np.abs(value) + off) + SMALLEST[dtype]


def assert_near(got, want, bound, what):
    got = host(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.isfinite(got).all(), what
    over = np.abs(got - want) - bound
    if over.size and over.max() > 0:
        at = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError("%s at %s: got %r, want %r, bound %.3e (%d of %d over theirs)" % (
            what, at, got[at], want[at], bound[at], int((over > 0).sum()), over.size))
