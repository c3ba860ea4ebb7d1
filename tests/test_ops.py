"""The encoder-layer operators (gnn_model_explainer_amd/ops.py): layer norm, counter-based dropout and the two in one pass, forward and backward, against their
definitions in 64 bits, at the sizes where they can go wrong; their refusals; the encoders that call them.  On two backends: the HIP library (GPU) runs every case, the
emulator build of the sources (CPU) the smaller ones, each in one type, with one of every launch shape among them.

Tolerances are a priori.  u = 2^-24 is the relative error of one fp32 operation, h = finfo(type).eps / 2 that of the one rounding at the store (plus half of the
type's smallest subnormal), L the longest chain of additions of a row sum, of which the kernels have at most cols / 64 + 16 (64 lanes or more share a row of more
than 64 sixteen-byte pieces; shorter rows: at most 8 in a lane and 6 between lanes).  Writing e(z) for the bound on z's error before the store:
  e(mean)  = (L + 2) u mean|v|
  e(xhat)  = rstd e(mean) + |xhat| ((L + 8) / 2 + 6) u     (the shift by e(mean) changes the variance in second order only: (e(mean) rstd)^2 / 2 |xhat|)
  e(y)     = |w| e(xhat) + 2 u |xhat w| + u |y|
  backward, mean and rstd given: e(xhat) = 3 u |xhat|, e(dy) = 3 u (|dh| + |dd| / (1 - p)), e(g) = |w| e(dy) + u |g|,
  e(c1)    = mean e(g) + (L + 2) u mean|g|,  e(c2) = mean(e(g) |xhat| + |g| e(xhat)) + (L + 3) u mean|g xhat|
  e(dx)    = rstd (e(g) + e(c1) + |xhat| e(c2) + |c2| e(xhat) + 3 u (|g| + |c1| + |xhat c2|)) + u |dx|
  e(dw)    = sum(e(dy) |xhat| + |dy| e(xhat)) + (rows + 8) u sum|dy xhat|,  e(db) = sum e(dy) + (rows + 8) u sum|dy|
  dropout: two roundings (1 / (1 - p) and the product) before the store's.
All bounds are widened by 1 % for the second-order terms."""
import argparse

import numpy as np
import pytest
import torch

from gnn_model_explainer_amd import engine, models, ops

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


class _Backend:
    def __init__(self, name):
        self.name = name
        if name == "emu":
            from emu.emu_engine import emu_library
            self.lib, self.device = emu_library(), "cpu"
        else:
            assert torch.cuda.is_available(), "the gpu twins need an MI355X"
            self.lib, self.device = None, "cuda:0"


@pytest.fixture(params=["emu", pytest.param("gpu", marks=pytest.mark.gpu)])
def be(request, monkeypatch):
    b = _Backend(request.param)
    monkeypatch.setitem(ops._ENGINE, "lib", b.lib)
    return b


# ---------------------------------------------------------------- definitions in 64 bits ----------------------------------------------------------------
def philox(c, k):
    """The four words of Philox-4x32-10 (Salmon et al., SC 2011) for counter words c (uint64 arrays) under the key words k."""
    m, c, k = np.uint64(0xFFFFFFFF), list(c), list(k)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & m, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def philox_words(seed, step, rows, cols):
    """uint32 [len(rows), cols]: the word of every element."""
    rows = np.asarray(rows, np.uint64)[:, None]
    blocks = (cols + 3) // 4
    full = lambda a: np.broadcast_to(a, (len(rows), blocks))
    c = philox([full(np.arange(blocks, dtype=np.uint64)[None]), full(rows & np.uint64(0xFFFFFFFF)), full(rows >> np.uint64(32)), full(np.uint64(step))],
               [seed & 0xFFFFFFFF, seed >> 32])
    return np.stack(c, axis=2).reshape(len(rows), 4 * blocks)[:, :cols].astype(np.uint32)


def keep_mask(p, seed, step, rows, cols):
    return torch.from_numpy(philox_words(seed, step, rows, cols).astype(np.uint64) >= np.uint64(round(p * 2 ** 32)))


def drop64(v, p, keep):
    return torch.where(keep, v / (1.0 - p) if p < 1.0 else torch.zeros_like(v), torch.zeros_like(v))


def f64(t):
    return None if t is None else t.detach().cpu().double()


class Norm64:
    """The forward and backward formulas and the bounds of this file's head."""

    def __init__(self, x, w, b, eps, relu, stats=None):
        self.x, self.w, self.relu = f64(x), f64(w), relu
        v = self.x.clamp_min(0.0) if relu else self.x
        F = v.shape[1]
        self.L = F / 64 + 16
        mean = v.mean(1, keepdim=True)
        rstd = ((v - mean).square().mean(1, keepdim=True) + eps).rsqrt()
        if stats is not None:
            mean, rstd = (f64(s)[:, None] for s in stats)
        self.rstd, self.mean = rstd, mean
        self.xhat = (v - mean) * rstd
        self.ww = torch.ones(F, dtype=torch.float64) if w is None else self.w
        self.y = self.xhat * self.ww + (0.0 if b is None else f64(b))
        self.e_mean = (self.L + 2) * U * v.abs().mean(1, keepdim=True)
        e_xhat = rstd * self.e_mean + self.xhat.abs() * ((self.L + 8) / 2 + 6) * U + 0.5 * (rstd * self.e_mean) ** 2 * self.xhat.abs()
        self.e_rstd = rstd * (((self.L + 8) / 2 + 4) * U + 0.5 * (rstd * self.e_mean) ** 2)
        self.e_y = self.ww.abs() * e_xhat + 2 * U * (self.xhat * self.ww).abs() + U * self.y.abs()

    def backward(self, dh, dd, p, keep):
        a = torch.zeros_like(self.x) if dh is None else f64(dh)
        bb = torch.zeros_like(self.x) if dd is None else drop64(f64(dd), p, keep)
        dy, R = a + bb, self.x.shape[0]
        e_dy, e_xhat = 3 * U * (a.abs() + bb.abs()), 3 * U * self.xhat.abs()
        g = dy * self.ww
        e_g = self.ww.abs() * e_dy + U * g.abs()
        mean = lambda t: t.mean(1, keepdim=True)
        c1, c2 = mean(g), mean(g * self.xhat)
        e_c1 = mean(e_g) + (self.L + 2) * U * mean(g.abs())
        e_c2 = mean(e_g * self.xhat.abs() + g.abs() * e_xhat) + (self.L + 3) * U * mean((g * self.xhat).abs())
        dx = self.rstd * (g - c1 - self.xhat * c2)
        e_dx = self.rstd * (e_g + e_c1 + self.xhat.abs() * e_c2 + c2.abs() * e_xhat + 3 * U * (g.abs() + c1.abs() + (self.xhat * c2).abs())) + U * dx.abs()
        if self.relu:
            dx, e_dx = dx.masked_fill(self.x <= 0, 0.0), e_dx.masked_fill(self.x <= 0, 0.0)
        dw, db = (dy * self.xhat).sum(0), dy.sum(0)
        e_dw = (e_dy * self.xhat.abs() + dy.abs() * e_xhat).sum(0) + (R + 8) * U * (dy * self.xhat).abs().sum(0)
        e_db = e_dy.sum(0) + (R + 8) * U * dy.abs().sum(0)
        return (dx, e_dx), (dw, e_dw), (db, e_db)


def assert_close(got, want, bound, what):
    t = got.dtype
    tol = 1.01 * bound + torch.finfo(t).eps / 2 * (want.abs() + 1.01 * bound) + TINY[t] / 2
    err = (f64(got) - want).abs()
    worst = float((err / tol.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert got.shape == want.shape and bool((err <= tol).all()), "%s: %.3f of the bound" % (what, worst)


def make(be, rows, cols, dtype, wtype, pad=0, seed=0, params=("w", "b")):
    """x (rows with a level of their own, one empty row, columns of different weight), dy, dd inside wider tensors, w, b"""
    g = torch.Generator().manual_seed(1000 * rows + cols + seed)
    def inside(t):
        base = torch.full((rows, cols + pad), 7.0)
        base[:, pad // 2:pad // 2 + cols] = t
        return base.to(dtype).to(be.device)[:, pad // 2:pad // 2 + cols]
    x = torch.randn(rows, cols, generator=g) * (1 + 4 * (torch.rand(cols, generator=g) < 0.1)) + torch.randn(rows, 1, generator=g)
    if rows > 2:
        x[1] = 0.0
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wtype or dtype).to(be.device) if "w" in params else None
    b = (0.3 * torch.randn(cols, generator=g)).to(wtype or dtype).to(be.device) if "b" in params else None
    return inside(x), inside(torch.randn(rows, cols, generator=g)), inside(torch.randn(rows, cols, generator=g)), w, b


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 20), (70, 20), (33, 33), (4, 64), (3, 257), (2, 1000), (5, 1283), (2, 2049), (1, 4100), (2, 4133)]
BIG = [(1, 8192), (3, 8193), (17, 16385), (2, 32769), (2, 65537), (1, 131073), (5, 300007), (9, 4096), (1000, 60), (4099, 20), (300, 513), (40000, 3), (513, 2048), (33, 4095)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _cases():
    out = []
    for i, s in enumerate(SHAPES):
        out.append(pytest.param("emu", *s, TYPES[i % 3], id="emu-%dx%d-%s" % (s + (str(TYPES[i % 3])[6:],))))
    for i, s in enumerate(SHAPES + BIG):
        for t in TYPES:
            out.append(pytest.param("gpu", *s, t, id="gpu-%dx%d-%s" % (s + (str(t)[6:],)), marks=pytest.mark.gpu))
    return out


@pytest.fixture
def on(monkeypatch):
    def pick(name):
        b = _Backend(name)
        monkeypatch.setitem(ops._ENGINE, "lib", b.lib)
        return b
    return pick


@pytest.mark.parametrize("name,rows,cols,dtype", _cases())
def test_layer_norm_forward_and_backward_against_64_bits(on, name, rows, cols, dtype):
    be = on(name)
    for relu, pad, wtype, params in ((True, 0, torch.float32, ("w", "b")), (False, 6, dtype, ("w", "b")), (False, 1, dtype, ())):
        x, dy, _, w, b = make(be, rows, cols, dtype, wtype, pad, params=params)
        ref = Norm64(x, w, b, 1e-5, relu)
        y, mean, rstd = ops.layer_norm_forward(x, w, b, relu=relu)
        assert y.is_contiguous() and y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32 and mean.shape == (rows,)
        assert_close(y, ref.y, ref.e_y, "y")
        assert_close(mean, ref.mean[:, 0], ref.e_mean[:, 0], "mean")
        assert_close(rstd, ref.rstd[:, 0], ref.e_rstd[:, 0], "rstd")
        assert torch.equal(ops.layer_norm(x, w, b, relu=relu), y)
        back = Norm64(x, w, b, 1e-5, relu, (mean, rstd)).backward(dy, None, 0.0, None)
        got = ops.layer_norm_backward(dy, x, mean, rstd, w, relu=relu)
        assert (got[1] is None) == (got[2] is None) == (w is None)
        for g, (want, bound), what in zip(got, back, ("dx", "dw", "db")):
            if g is not None:
                assert_close(g, want, bound, what)


# one of every launch shape: each number of lanes and pieces per lane of the forward pass, the backward pass's workgroups of few and many waves and of two pieces per lane,
# long rows in chunks (several rows per walk), more than 16 partial rows of dw and db
LAUNCHES = [(3, 4, torch.float32), (5, 6, torch.float32), (3, 13, torch.float32), (3, 30, torch.float32), (2, 61, torch.float32), (2, 125, torch.float32),
            (2, 250, torch.float32), (2, 511, torch.float32), (2, 767, torch.float32), (2, 1021, torch.float32), (2, 2047, torch.float32), (2, 3001, torch.float32),
            (2, 4095, torch.float32), (2, 5000, torch.float32), (3, 8193, torch.float32), (700, 3, torch.float16), (1500, 9, torch.bfloat16), (2, 8193, torch.bfloat16),
            (3, 16383, torch.bfloat16), (5, 16387, torch.float16)]


@pytest.mark.parametrize("rows,cols,dtype", LAUNCHES)
def test_every_launch_shape_on_the_emulator(on, rows, cols, dtype):
    test_layer_norm_forward_and_backward_against_64_bits(on, "emu", rows, cols, dtype)
    test_layer_norm_dropout_against_64_bits(on, "emu", rows, cols, dtype)
    test_dropout_against_its_definition(on, "emu", rows, cols, dtype)


def _whole_numbers(be, rows, cols, dtype, seed=0):
    """x, dh, dd of small whole numbers on the device: with mean 0 and rstd 1 given (and p = 1/2, whose scale is 2) every product and every partial sum of dw and db is a
    whole number below 2^24, exact in fp32 in whatever order."""
    g = torch.Generator(device=be.device).manual_seed(1000 * rows + cols + seed)
    assert rows * 3 * 9 < 1 << 24
    return [torch.randint(-3, 4, (rows, cols), generator=g, device=be.device).to(dtype) for _ in range(3)]


MANY = [(40000, 3), (300000, 3), (300000, 7), (40000, 20), (99997, 20), (99997, 60), (20000, 130), (20000, 513), (5000, 4095), (3000, 8190), (700, 16385), (200, 65537)]


def _many_cases():
    out = [pytest.param("emu", r, c, t, id="emu-%dx%d-%s" % (r, c, str(t)[6:]))
           for r, c, t in ((4000, 3, torch.float32), (3000, 7, torch.bfloat16), (1500, 9, torch.bfloat16), (1100, 20, torch.float32), (90, 513, torch.float16),
                           (9, 5000, torch.float32), (9, 8193, torch.bfloat16))]
    return out + [pytest.param("gpu", r, c, t, id="gpu-%dx%d-%s" % (r, c, str(t)[6:]), marks=pytest.mark.gpu) for r, c in MANY for t in TYPES]


@pytest.mark.parametrize("name,rows,cols,dtype", _many_cases())
def test_no_row_is_lost_or_counted_twice_in_the_parameters_gradients(on, name, rows, cols, dtype):
    """dw and db, exact: one row more or less, in any lane's or workgroup's share, shows."""
    be = on(name)
    x, dh, dd = _whole_numbers(be, rows, cols, dtype)
    mean, rstd, w = torch.zeros(rows, device=be.device), torch.ones(rows, device=be.device), torch.ones(cols, device=be.device)
    sums = lambda dy: ((dy.double() * x.double()).sum(0), dy.double().sum(0))
    _, dw, db = ops.layer_norm_backward(dh, x, mean, rstd, w)
    for got, want in zip((dw, db), sums(dh)):
        assert torch.equal(got.double(), want)
    kept = ops.dropout(torch.ones_like(x), 0.5, 7, 3).double()            # 2 or 0: ops.dropout against its definition is a test of its own
    _, dw, db = ops.layer_norm_dropout_backward(dh, dd, x, mean, rstd, w, 0.5, 7, 3)
    for got, want in zip((dw, db), sums(dh.double() + dd.double() * kept)):
        assert torch.equal(got.double(), want)
    # one row alone
    for r in {0, rows // 2, rows - 1}:
        one = torch.zeros_like(dh)
        one[r] = dh[r]
        _, dw, db = ops.layer_norm_backward(one, x, mean, rstd, w)
        assert torch.equal(dw, dh[r].float() * x[r].float()) and torch.equal(db, dh[r].float())


@pytest.mark.parametrize("name,rows,cols,dtype", [c for c in _many_cases() if c.values[1] * c.values[2] < 1 << 24])
def test_the_parameters_gradients_of_many_rows_against_64_bits(on, name, rows, cols, dtype):
    """As above with ordinary numbers.  A column's longest chain of additions is a lane's walk over its share of the rows (at most rows / parts, the workgroups that leave a
    partial row each), at most 6 + 4 additions across the lanes and waves of a workgroup, and the join of the partial rows: parts / 32 + 36 (or up to 16 one by one)."""
    be = on(name)
    lib = be.lib or engine.get_library()
    x, dy, _, w, _ = make(be, rows, cols, dtype, torch.float32)
    _, mean, rstd = ops.layer_norm_forward(x, w)
    _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    nbytes = lib.gnnx_layer_norm_workspace_bytes(TYPES.index(dtype), rows, cols, 1)
    parts = nbytes // (8 * cols)                                          # (long rows keep a little more there: at least this many workgroups' share)
    if cols > 8192:
        parts = 1
    chain = -(-rows // parts) + parts / 32 + 64
    xd, dyd, md, rd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    xhat = (xd - md) * rd
    # each term: xhat's two roundings, the product fused into the sum, and the chain's
    for got, terms, each in ((dw, dyd * xhat, 3), (db, dyd, 0)):
        want, size = terms.sum(0), terms.abs().sum(0)
        assert got.dtype == torch.float32 and bool(((got.double() - want).abs() <= 1.01 * (chain + each) * U * size + 2.0 ** -149).all())


@pytest.mark.parametrize("name,rows,cols,dtype", _cases())
def test_layer_norm_dropout_against_64_bits(on, name, rows, cols, dtype):
    be = on(name)
    for relu, pad, wtype, p, row0 in ((True, 0, torch.float32, 0.5, 0), (False, 5, dtype, 0.1, (1 << 32) - 2)):
        x, dh, dd, w, b = make(be, rows, cols, dtype, wtype, pad, seed=1)
        draws = dict(p=p, seed=0x1234567890ABCDEF, step=77, row_offset=row0)
        keep = keep_mask(p, draws["seed"], 77, row0 + np.arange(rows), cols)
        ref = Norm64(x, w, b, 1e-5, relu)
        h, d, mean, rstd = ops.layer_norm_dropout_forward(x, w, b, relu=relu, **draws)
        assert_close(h, ref.y, ref.e_y, "h")
        assert torch.equal(h, ops.layer_norm(x, w, b, relu=relu))
        assert_close(d, drop64(ref.y, p, keep), (ref.e_y + 2 * U * ref.y.abs()) / (1 - p) * keep, "d")
        assert bool((d.cpu()[~keep] == 0).all())
        h2, d2 = ops.layer_norm_dropout(x, w, b, relu=relu, **draws)
        assert torch.equal(h2, h) and torch.equal(d2, d)
        n64 = Norm64(x, w, b, 1e-5, relu, (mean, rstd))
        for first, second in ((dh, dd), (None, dd), (dh, None)):
            got = ops.layer_norm_dropout_backward(first, second, x, mean, rstd, w, relu=relu, **draws)
            for g, (want, bound), what in zip(got, n64.backward(first, second, p, keep), ("dx", "dw", "db")):
                assert_close(g, want, bound, what)


@pytest.mark.parametrize("name,rows,cols,dtype", _cases())
def test_dropout_against_its_definition(on, name, rows, cols, dtype):
    be = on(name)
    for p, pad, step, row0 in ((0.5, 0, 0, 0), (0.1, 3, (1 << 32) - 1, (1 << 32) - 1)):
        x = make(be, rows, cols, dtype, None, pad)[0]
        keep = keep_mask(p, 42, step, row0 + np.arange(rows), cols)
        y = ops.dropout(x, p, 42, step, row0)
        want = drop64(f64(x), p, keep)
        assert y.is_contiguous() and bool((y.cpu()[~keep] == 0).all())
        assert_close(y, want, 2 * U * want.abs(), "y")
        state = torch.tensor([42, step], dtype=torch.int64, device=be.device)
        assert torch.equal(ops.dropout(x, p, state, 0, row0), y)


def test_philox_known_answers():
    """This file's form of the generator against the vectors published with it (Random123, philox4x32-10)."""
    for c, k, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                       ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                       ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v[0]) for v in philox([np.array([v], np.uint64) for v in c], k)) == want


def test_dropout_keeps_and_drops_everything_at_the_ends(be):
    x = torch.tensor([[1.5, float("inf"), float("nan"), -2.0, 3.0]], device=be.device)
    y = ops.dropout(x, 0.0, 7)
    assert torch.equal(torch.nan_to_num(y, 9.0, 8.0), torch.nan_to_num(x, 9.0, 8.0)) and y.data_ptr() != x.data_ptr()
    assert bool((ops.dropout(x, 1.0, 7) == 0).all())
    assert torch.equal(torch.nan_to_num(ops.dropout(x, 2.0 ** -34, 7), 9.0, 8.0), torch.nan_to_num(x, 9.0, 8.0))      # a threshold of zero
    w = torch.full((5,), 2.0, device=be.device)
    z = torch.tensor([[1.5, -1.0, 0.25, -2.0, 3.0]], device=be.device)
    h, d = ops.layer_norm_dropout(z, w, w, 0.0, 7)
    assert torch.equal(h, d) and torch.equal(h, ops.layer_norm(z, w, w))
    h, d, mean, rstd = ops.layer_norm_dropout_forward(z, w, w, 1.0, 7)
    assert bool((d == 0).all()) and torch.equal(h, ops.layer_norm(z, w, w))
    got = ops.layer_norm_dropout_backward(h, h, z, mean, rstd, w, 0.0, 7)
    both = ops.layer_norm_backward(2 * h, z, mean, rstd, w)
    assert all(torch.equal(a, b) for a, b in zip(got, both))
    got = ops.layer_norm_dropout_backward(h, h, z, mean, rstd, w, 1.0, 7)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.layer_norm_backward(h, z, mean, rstd, w)))


def test_infinities_and_nan_stay_in_their_rows_and_out_of_dropped_places(be):
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(3))
    clean = x.clone()
    x[2, 7], x[4, 3] = float("nan"), float("inf")
    keep = keep_mask(0.5, 11, 0, np.arange(6), 40)
    x, clean = x.to(be.device), clean.to(be.device)
    y = ops.dropout(x, 0.5, 11).cpu()
    assert bool((y[~keep] == 0).all()) and bool(torch.isnan(y[2, 7]) == keep[2, 7]) and bool(torch.isinf(y[4, 3]) == keep[4, 3])
    for relu in (False, True):
        h, mean, rstd = ops.layer_norm_forward(x, relu=relu)
        want, _, _ = ops.layer_norm_forward(clean, relu=relu)
        rows = [0, 1, 3, 5]
        assert torch.equal(h[rows], want[rows]) and bool(torch.isnan(h[2]).all()) and bool(torch.isnan(h[4, 3]))
        dx, _, _ = ops.layer_norm_backward(clean, x, mean, rstd, relu=relu)
        assert bool(torch.isfinite(dx[rows]).all())


def test_views_strides_and_broadcast_gradients(be):
    """Leading dimensions, a column slice, a transposed and a permuted tensor, rows that are one row, a gradient that is one number broadcast."""
    g = torch.Generator().manual_seed(5)
    base = torch.randn(4, 6, 50, generator=g).to(be.device)
    w, b = torch.rand(20, generator=g).to(be.device) + 0.5, torch.rand(20, generator=g).to(be.device)
    views = [base[:, :, 10:30], base[:, 2:5, 10:30], base[1:2, :, 10:30], base[::2, 3:4, 30:50], base[:, :, :20].transpose(0, 1),
             base[:, 0, :40:2], base[0, 0, 7:27], base[0, :1, 7:27].expand(5, 20), base.permute(2, 0, 1)[:, :, :1].expand(50, 4, 20), base[..., None].expand(4, 6, 50, 20)]
    for v in views:
        dense = v.contiguous()
        y, mean, rstd = ops.layer_norm_forward(v, w, b)
        assert y.shape == v.shape and torch.equal(y, ops.layer_norm(dense, w, b)) and mean.shape == v.shape[:-1]
        assert torch.equal(ops.dropout(v, 0.3, 9, 2), ops.dropout(dense, 0.3, 9, 2))
        one = torch.full((), 0.25, device=be.device).expand(v.shape)
        a, c = ops.layer_norm_backward(one, v, mean, rstd, w), ops.layer_norm_backward(one.contiguous(), dense, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    ww = torch.stack([w, b], 1)
    assert torch.equal(ops.layer_norm(views[0], ww[:, 0], ww[:, 1]), ops.layer_norm(views[0], w, b))      # strided parameters
    x = torch.randn(7, 33, generator=g).to(be.device)
    assert torch.equal(torch.cat([ops.dropout(x[:3], 0.4, 1, 5), ops.dropout(x[3:], 0.4, 1, 5, row_offset=3)]), ops.dropout(x, 0.4, 1, 5))   # shards


def test_empty_tensors(be):
    w = torch.ones(5, device=be.device)
    x = torch.empty(0, 5, device=be.device)
    y, mean, rstd = ops.layer_norm_forward(x, w, w)
    assert y.shape == (0, 5) and mean.shape == rstd.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 5) and bool((dw == 0).all()) and bool((db == 0).all()) and dw.shape == (5,)
    h, d = ops.layer_norm_dropout(x, w, w, 0.5, 1)
    assert h.shape == d.shape == (0, 5)
    assert ops.dropout(x, 0.5, 1).shape == (0, 5) and ops.dropout(torch.empty(3, 0, device=be.device), 0.5, 1).shape == (3, 0)


def test_gradients_through_autograd(be):
    """The three operators under autograd: equal to their explicit passes, to differences of the 64-bit forward pass, and right where only some inputs want one."""
    g = torch.Generator().manual_seed(8)
    rows, cols, p, seed, step = 9, 21, 0.4, 123, 4
    x0 = torch.randn(rows, cols, generator=g) + 0.3
    x0[x0.abs() < 1e-2] = 0.5             # (differences: nothing close to the ReLU's corner)
    w0, b0 = 1 + 0.2 * torch.randn(cols, generator=g), 0.2 * torch.randn(cols, generator=g)
    up, ud = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
    keep = keep_mask(p, seed, step, np.arange(rows), cols)
    x, w, b = (t.clone().to(be.device).requires_grad_() for t in (x0, w0, b0))
    h, d = ops.layer_norm_dropout(x, w, b, p, seed, step, relu=True)
    grads = torch.autograd.grad([h, d], [x, w, b], [up.to(be.device), ud.to(be.device)])
    hh, dd, mean, rstd = ops.layer_norm_dropout_forward(x.detach(), w.detach(), b.detach(), p, seed, step, relu=True)
    assert torch.equal(h, hh) and torch.equal(d, dd)
    again = ops.layer_norm_dropout_backward(up.to(be.device), ud.to(be.device), x.detach(), mean, rstd, w.detach(), p, seed, step, relu=True)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))

    def value(x, w, b):
        v = x.clamp_min(0.0)
        m = v.mean(1, keepdim=True)
        y = (v - m) * ((v - m).square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b
        return float((y * up.double()).sum() + (drop64(y, p, keep) * ud.double()).sum())
    at = [f64(t) for t in (x0, w0, b0)]
    for i in range(3):
        direction = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + eps * direction, at[i] - eps * direction
        diff = (value(*hi) - value(*lo)) / (2 * eps)
        want = float((f64(grads[i]) * direction).sum())
        scale = float((f64(grads[i]).abs() * direction.abs()).sum())
        assert abs(diff - want) <= 1e-4 * scale          # the difference's own error: eps^2 times third derivatives, 2^-52 |value| / eps
    # one output used, one input wanted
    for leaf in range(3):
        ts = [t.detach().clone().to(be.device).requires_grad_(i == leaf) for i, t in enumerate((x0, w0, b0))]
        h, d = ops.layer_norm_dropout(*ts, p, seed, step, relu=True)
        got, = torch.autograd.grad(d, ts[leaf], ud.to(be.device))
        alone = ops.layer_norm_dropout_backward(None, ud.to(be.device), x.detach(), mean, rstd, w.detach(), p, seed, step, relu=True)[leaf]
        assert torch.equal(got, alone)
    y = ops.layer_norm(x, None, b)                       # an offset alone
    gb, = torch.autograd.grad(y, b, up.to(be.device))
    assert torch.allclose(gb.cpu().double(), up.double().sum(0), rtol=0, atol=float((rows + 8) * U * up.abs().double().sum(0).max()))
    y = ops.dropout(x, p, seed, step)
    gx, = torch.autograd.grad(y, x, up.to(be.device))
    assert torch.equal(gx, ops.dropout(up.to(be.device), p, seed, step))
    ops.dropout(x, p, seed, step).sum().backward()       # an expanded gradient
    assert torch.equal(x.grad.cpu() != 0, keep)
    with torch.no_grad():
        assert not ops.layer_norm(x, w, b).requires_grad


def test_gradients_of_broadcast_and_shared_inputs(be):
    """A row broadcast over a batch, and a gain used by two calls: their gradients are the sums over the uses."""
    g = torch.Generator().manual_seed(12)
    row, w = (torch.randn(24, generator=g).to(be.device).requires_grad_() for _ in range(2))
    up, vp = (torch.randn(5, 24, generator=g).to(be.device) for _ in range(2))
    x = row.expand(5, 24)
    other = torch.randn(5, 24, generator=g).to(be.device)
    y, z = ops.layer_norm(x, w), ops.layer_norm(other, w, relu=True)
    gr, gw = torch.autograd.grad([y, z], [row, w], [up, vp])
    dense = x.detach().contiguous()
    _, m, r = ops.layer_norm_forward(dense, w.detach())
    dx, dw, _ = ops.layer_norm_backward(up, dense, m, r, w.detach())
    _, m2, r2 = ops.layer_norm_forward(other, w.detach(), relu=True)
    _, dw2, _ = ops.layer_norm_backward(vp, other, m2, r2, w.detach(), relu=True)
    assert torch.allclose(gr, dx.sum(0), rtol=1e-6, atol=1e-6) and torch.equal(gw, dw + dw2)      # (the sum over five rows in another order: 4 u of their size)


def test_gradients_cannot_be_differentiated_again(be):
    x = torch.randn(4, 8, device=be.device, requires_grad=True)
    for y in (ops.layer_norm(x, relu=True), ops.dropout(x, 0.5, 1), ops.layer_norm_dropout(x, None, None, 0.5, 1)[1]):
        gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        assert torch.isfinite(gx).all()
        with pytest.raises(RuntimeError, match="differentiate twice"):
            gx.sum().backward()


def test_a_seed_tensor_that_moved_on_is_an_error(be):
    x = torch.randn(4, 8, device=be.device, requires_grad=True)
    state = torch.tensor([5, 0], dtype=torch.int64, device=be.device)
    for f in (lambda: ops.dropout(x, 0.5, state), lambda: ops.layer_norm_dropout(x, None, None, 0.5, state)[1]):
        y = f()
        state[1] += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_refusals(be):
    x = torch.randn(4, 8, device=be.device)
    w = torch.ones(8, device=be.device)
    y, mean, rstd = ops.layer_norm_forward(x, w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.layer_norm(x.double())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.dropout(x.long(), 0.5, 1)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.dropout([1.0], 0.5, 1)
    with pytest.raises(TypeError, match="weight must be float32 or of x's type"):
        ops.layer_norm(x, w.half())
    with pytest.raises(TypeError, match="one type"):
        ops.layer_norm(x.half(), w, w.half())
    with pytest.raises(ValueError, match="at least one dimension"):
        ops.layer_norm(torch.tensor(1.0, device=be.device))
    with pytest.raises(ValueError, match="no elements"):
        ops.layer_norm(torch.empty(3, 0, device=be.device))
    with pytest.raises(ValueError, match=r"bias must have shape \(8,\)"):
        ops.layer_norm(x, w, w[:7])
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="dy must be"):
        ops.layer_norm_backward(y[:3], x, mean, rstd, w)
    with pytest.raises(ValueError, match="dy must be"):
        ops.layer_norm_backward(y.half(), x, mean, rstd, w)
    with pytest.raises(ValueError, match="rstd must be"):
        ops.layer_norm_backward(y, x, mean, rstd[:3], w)
    with pytest.raises(ValueError, match="both None"):
        ops.layer_norm_dropout_backward(None, None, x, mean, rstd, w)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match=r"p must be in \[0, 1\]"):
            ops.dropout(x, p, 1)
    for kw in (dict(seed=-1), dict(seed=1 << 63), dict(seed=1, step=-1), dict(seed=1, step=1 << 32), dict(seed=1, row_offset=-1)):
        with pytest.raises(ValueError):
            ops.dropout(x, 0.5, **kw)
    for state in (torch.zeros(2, device=be.device), torch.zeros(3, dtype=torch.int64, device=be.device), torch.zeros(4, dtype=torch.int64, device=be.device)[::2]):
        with pytest.raises(ValueError, match="seed tensor"):
            ops.dropout(x, 0.5, state)


def test_the_ends_of_the_ranges_of_seed_step_and_row_offset(be):
    """The largest of each, as a number and (seed, step) as a tensor: the masks of the definition; one more is refused."""
    x = torch.randn(3, 11, generator=torch.Generator().manual_seed(1)).to(be.device)
    for seed, step, row0 in (((1 << 63) - 1, 0, 0), ((1 << 63) - 1, (1 << 32) - 1, (1 << 62) - 1), (0, 0, 0)):
        y = ops.dropout(x, 0.5, seed, step, row0)
        keep = keep_mask(0.5, seed, step, np.arange(row0, row0 + 3, dtype=np.uint64), 11)
        assert torch.equal(y.cpu(), torch.where(keep, 2 * x.cpu(), torch.zeros(())))
        assert torch.equal(ops.dropout(x, 0.5, torch.tensor([seed, step], device=be.device), 0, row0), y)
    for kw in (dict(seed=1 << 63), dict(seed=1, step=1 << 32), dict(seed=1, row_offset=1 << 62)):
        with pytest.raises(ValueError, match="must be in"):
            ops.dropout(x, 0.5, **kw)


def test_forward_mode_derivatives_and_batched_tensors_are_refused(be):
    import torch.autograd.forward_ad as fwd
    x, w = torch.randn(4, 8, device=be.device), torch.ones(8, device=be.device)
    with fwd.dual_level():
        for call in (lambda: ops.layer_norm(fwd.make_dual(x, x)), lambda: ops.layer_norm(x, fwd.make_dual(w, w)), lambda: ops.dropout(fwd.make_dual(x, x), 0.5, 1)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: ops.layer_norm(v, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: ops.layer_norm(v, w).sum())(x)


def test_tensors_without_memory_are_refused_or_materialised(be):
    """What has no memory of its own must not be read as an argument that is not there (a weight of ones, the seed 0): torch's zero tensor counts as the zeros it is,
    everything else is refused by name."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x = torch.randn(4, 8, generator=torch.Generator().manual_seed(1)).to(be.device)
    w, state = torch.rand(8, device=be.device) + 0.5, torch.tensor([0, 0], device=be.device)
    y, mean, rstd = ops.layer_norm_forward(x, w)
    zero = lambda *s, **kw: torch._efficientzerotensor(s, device=be.device, **kw)
    assert torch.equal(ops.layer_norm(x, zero(8), w), ops.layer_norm(x, torch.zeros_like(w), w)) and torch.equal(ops.layer_norm(x, w, zero(8)), y)
    assert torch.equal(ops.layer_norm(zero(4, 8), w, w), w.expand(4, 8)) and bool((ops.dropout(zero(4, 8), 0.5, 1) == 0).all())
    assert torch.equal(ops.dropout(x, 0.5, zero(2, dtype=torch.int64)), ops.dropout(x, 0.5, 0))
    for got, want in zip(ops.layer_norm_backward(zero(4, 8), x, zero(4), rstd, w), ops.layer_norm_backward(torch.zeros_like(x), x, torch.zeros_like(mean), rstd, w)):
        assert torch.equal(got, want)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fx, fw, fs, fm = (mode.from_tensor(t) for t in (x, w, state, mean))
    leaf = x.clone().requires_grad_()
    for call in (lambda: ops.layer_norm(fx), lambda: ops.layer_norm(x, fw), lambda: ops.layer_norm(x, None, fw), lambda: ops.dropout(fx, 0.5, 1), lambda: ops.dropout(x, 0.5, fs),
                 lambda: ops.layer_norm_backward(fx, x, mean, rstd), lambda: ops.layer_norm_backward(x, x, fm, rstd), lambda: ops.layer_norm(x, w.to_sparse()),
                 lambda: ops.layer_norm_backward(x.to_sparse(), x, mean, rstd), lambda: torch.func.functionalize(ops.layer_norm)(x),
                 lambda: torch.func.vmap(ops.layer_norm)(x), lambda: torch.func.vmap(lambda v: ops.layer_norm(x, v))(w.expand(3, 8)),
                 lambda: torch.func.vmap(lambda s: ops.dropout(x, 0.5, s))(state.expand(3, 2)), lambda: torch.func.grad(lambda v: ops.layer_norm(v).sum())(x),
                 lambda: torch.autograd.grad(ops.layer_norm(leaf), leaf, x.expand(3, 4, 8), is_grads_batched=True),
                 lambda: torch.autograd.grad(ops.dropout(leaf, 0.5, 1), leaf, x.expand(3, 4, 8), is_grads_batched=True)):
        with pytest.raises(NotImplementedError, match="without memory"):
            call()
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.layer_norm(torch.zeros(2, 2, dtype=torch.complex64, device=be.device))


def test_views_of_the_opposite_sign(be):
    """The imaginary part of a conjugate is a view of memory that holds its elements' negatives: one column of it is evenly spaced rows, read in place."""
    g = torch.Generator().manual_seed(4)
    z = torch.complex(torch.randn(5, 3, generator=g), torch.randn(5, 3, generator=g)).to(be.device).conj()
    v, one = z.imag, torch.complex(torch.zeros(1), torch.tensor([2.0])).to(be.device).conj().imag      # one: [-2]
    assert v.is_neg() and one.is_neg()
    column = torch.tensor([[3.0], [4.0]], device=be.device)
    for t in (v, v[:, 1:2], v[:, 1]):
        plain = t.resolve_neg().clone()
        assert torch.equal(ops.dropout(t, 0.5, 3), ops.dropout(plain, 0.5, 3)) and torch.equal(ops.layer_norm(t, relu=True), ops.layer_norm(plain, relu=True))
        y, mean, rstd = ops.layer_norm_forward(plain)
        assert torch.equal(ops.layer_norm_backward(t, plain, mean, rstd)[0], ops.layer_norm_backward(plain, plain, mean, rstd)[0])
        leaf = plain.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(ops.dropout(leaf, 0.5, 3), leaf, t)[0], ops.dropout(plain, 0.5, 3))
    assert torch.equal(ops.layer_norm(column, None, one), torch.full_like(column, -2.0))       # (a row of one element is its mean)
    y, mean, rstd = ops.layer_norm_forward(column)
    assert torch.equal(ops.layer_norm_backward(column, column, one.expand(2), rstd, one.resolve_neg())[1],
                       ops.layer_norm_backward(column, column, one.resolve_neg().expand(2).contiguous(), rstd, one)[1])


def test_gradients_and_statistics_with_forward_mode_derivatives_are_refused(be):
    import torch.autograd.forward_ad as fwd
    x, w = torch.randn(4, 8, device=be.device), torch.ones(8, device=be.device)
    y, mean, rstd = ops.layer_norm_forward(x, w)
    leaf = x.clone().requires_grad_()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.layer_norm_backward(dual(y), x, mean, rstd, w), lambda: ops.layer_norm_backward(y, x, dual(mean), rstd, w),
                     lambda: ops.layer_norm_backward(y, x, mean, dual(rstd), w), lambda: ops.layer_norm_dropout_backward(y, dual(y), x, mean, rstd, w, 0.5, 1),
                     lambda: torch.autograd.grad(ops.layer_norm(leaf, w), leaf, dual(y)), lambda: torch.autograd.grad(ops.dropout(leaf, 0.5, 1), leaf, dual(y)),
                     lambda: torch.autograd.grad(ops.layer_norm_dropout(leaf, w, w, 0.5, 1)[1], leaf, dual(y))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dropout(torch.ones(2, 2), 0.5, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.layer_norm(torch.ones(2, 2))


def test_the_c_entry_points_refuse_what_they_cannot_do(be):
    import ctypes
    lib = be.lib or engine.get_library()
    x = torch.randn(4, 8, device=be.device)
    out = torch.full((4, 8), 3.0, device=be.device)
    def norm(**kw):
        n = engine._Norm(type=0, w_is_f32=1, rows=4, cols=8, x_stride=8, dy_stride=8, dd_stride=8, x=x.data_ptr(), y=out.data_ptr(), eps=1e-5)
        for k, v in kw.items():
            setattr(n, k, v)
        return n
    drop = engine._Drop(0.5, 1, None, 0, 0)
    assert lib.gnnx_layer_norm_forward(norm(rows=1, cols=1 << 20, x_stride=1 << 20), None, None, 0, None) != 0      # a long row without its workspace
    bad = [norm(type=3), norm(type=-1), norm(rows=-1), norm(cols=0), norm(cols=1 << 30), norm(x_stride=-8), norm(eps=-1.0), norm(y=None), norm(x=None),
           norm(mean=out.data_ptr()), norm(d=out.data_ptr())]
    for n in bad:
        assert lib.gnnx_layer_norm_forward(n, None, None, 0, None) != 0 and len(lib.gnnx_last_error()) > 5
    assert lib.gnnx_layer_norm_forward(None, None, None, 0, None) != 0
    assert lib.gnnx_layer_norm_forward(norm(), drop, None, 0, None) != 0
    assert lib.gnnx_layer_norm_forward(norm(d=out.data_ptr()), engine._Drop(1.5, 1, None, 0, 0), None, 0, None) != 0
    for n, ws in ((norm(dw=out.data_ptr(), dy=x.data_ptr(), mean=out.data_ptr(), rstd=out.data_ptr()), 0), (norm(dx=out.data_ptr()), 0),
                  (norm(dx=out.data_ptr(), dy=x.data_ptr()), 0), (norm(dx=out.data_ptr(), dd=x.data_ptr(), mean=out.data_ptr(), rstd=out.data_ptr()), 0)):
        assert lib.gnnx_layer_norm_backward(n, None, None, ws, None) != 0
    for args in ((3, 4, 8), (0, -1, 8), (0, 4, -1), (0, 4, 1 << 30)):
        assert lib.gnnx_dropout(*args, x.data_ptr(), 8, out.data_ptr(), drop, None) != 0
    assert lib.gnnx_dropout(0, 4, 8, None, 8, out.data_ptr(), drop, None) != 0
    assert lib.gnnx_dropout(0, 4, 8, x.data_ptr(), 8, out.data_ptr(), None, None) != 0
    assert bool((out == 3.0).all())


def test_the_c_entry_points_refuse_outputs_that_share_memory_with_inputs(be):
    """(in place a row's last piece, moved back into the row, could read what another lane has stored; outputs in the gaps between an input's rows are apart from it)"""
    lib = be.lib or engine.get_library()
    rows, cols, pad = 6, 5, 40
    base = torch.randn(rows, cols + pad, generator=torch.Generator().manual_seed(9)).to(be.device)
    other, stats = torch.zeros(2, rows * cols, device=be.device), torch.ones(2, rows, device=be.device)
    at = lambda r, c: base.data_ptr() + 4 * (r * (cols + pad) + c)
    drop = engine._Drop(0.5, 1, None, 0, 0)
    def dropout(y, x=at(0, 0), stride=cols + pad, r=rows):
        return lib.gnnx_dropout(0, r, cols, x, stride, y, drop, None)
    def forward(y, d=None):
        n = engine._Norm(type=0, w_is_f32=1, rows=rows, cols=cols, x_stride=cols + pad, x=at(0, 0), y=y, d=d, eps=1e-5)
        return lib.gnnx_layer_norm_forward(n, drop if d else None, None, 0, None)
    def backward(dx, **kw):
        n = engine._Norm(type=0, w_is_f32=1, rows=rows, cols=cols, x_stride=cols + pad, dy_stride=cols, dd_stride=cols, x=at(0, 0), dy=other[1].data_ptr(), dx=dx,
                         mean=stats[0].data_ptr(), rstd=stats[1].data_ptr())
        for k, v in kw.items():
            setattr(n, k, v)
        return lib.gnnx_layer_norm_backward(n, drop if n.dd else None, None, 0, None)
    before, out = base.clone(), other[0].data_ptr()
    inside = [at(0, 0), at(0, cols - 1), at(0, cols + 11), at(rows - 1, cols - 1), at(0, 0) - 4, at(2, 3), at(rows - 1, 0) - 4 * rows * cols + 4]
    for y in inside:
        for rc in (dropout(y), forward(y), forward(out, y), forward(y, out), backward(y)):
            assert rc != 0 and b"shares memory" in lib.gnnx_last_error()
    assert forward(out, out) != 0 and forward(out, out + 4) != 0
    assert backward(other[1].data_ptr()) != 0 and backward(out, dd=out) != 0 and backward(out, dd=out + 4 * (rows * cols - 1)) != 0
    assert dropout(at(0, 1), stride=0) != 0 and dropout(at(0, 0), stride=cols) != 0
    assert torch.equal(base, before) and bool((other == 0).all())
    # apart: behind the last row, before the first, between two rows that are one output apart
    tail = torch.zeros(rows * cols, device=be.device)
    assert dropout(tail.data_ptr()) == 0 and forward(tail.data_ptr()) == 0 and backward(tail.data_ptr()) == 0
    want = ops.dropout(before[:4, :cols], 0.5, 1)
    assert dropout(at(0, cols), r=4) == 0                                 # 20 elements in the gap of 40 behind the first row
    if be.device != "cpu":
        torch.cuda.synchronize()
    assert torch.equal(base[0, cols:cols + 20].view(4, cols), want) and torch.equal(base[1:], before[1:])


# ---------------------------------------------------------------- the encoders that call them ----------------------------------------------------------------
def _encoder(cls, layers=4, p=0.4, **kw):
    torch.manual_seed(3)
    args = argparse.Namespace(method="base", bias=True, layer_norm=True, dropout_seed=99, **kw)
    m = cls(7, 20, 20, 3, layers, bn=False, dropout=p, args=args)
    for n in m.norms:
        with torch.no_grad():
            n.weight.add_(0.3 * torch.randn(20))
            n.bias.add_(0.3 * torch.randn(20))
    return m


def _encoder64(m, x, adj, uses):
    """The node encoder's forward pass in 64 bits from its parameters; uses: how often its dropout was drawn before (None: evaluation)."""
    P = {k: v.detach().cpu().double().requires_grad_() for k, v in m.named_parameters()}
    convs = ["conv_first"] + ["conv_block.%d" % i for i in range(len(m.conv_block))] + ["conv_last"]
    h, embs = x, []
    for i, c in enumerate(convs):
        if uses is not None and 0 < i < len(convs) - 1:
            step = uses * len(m.conv_block) + i - 1
            keep = keep_mask(0.4, 99, step, np.arange(h.shape[0] * h.shape[1]), h.shape[2]).view(h.shape)
            h = drop64(h, 0.4, keep)
        y = adj @ h @ P[c + ".weight"] + P[c + ".bias"]
        y = y / y.norm(dim=2, keepdim=True).clamp_min(1e-12)
        if i < len(convs) - 1:
            v = torch.relu(y)                            # (its gradient at 0 is 0; clamp_min would pass it on)
            mu = v.mean(2, keepdim=True)
            y = (v - mu) * ((v - mu).square().mean(2, keepdim=True) + 1e-5).rsqrt() * P["norms.%d.weight" % i] + P["norms.%d.bias" % i]
        h = y
        embs.append(y)
    return P, embs


@pytest.mark.parametrize("graph_mode", [False, True])
def test_encoder_training_step_with_layer_norm_and_seeded_dropout(be, graph_mode):
    """The run of all three operators as an encoder makes them: logits and every parameter's gradient of two consecutive training steps against 64 bits, the
    evaluation pass without dropout, and reset_dropout."""
    cls = models.GcnEncoderGraph if graph_mode else models.GcnEncoderNode
    m = _encoder(cls)
    m.to(be.device).train()
    g = torch.Generator().manual_seed(6)
    B, n = 2, 12
    adj = (torch.rand(B, n, n, generator=g) < 0.3).float()
    adj = ((adj + adj.transpose(1, 2)) > 0).float()
    adj[:, 5] = 0
    adj[:, :, 5] = 0                                     # an isolated node: its rows are bias alone
    x = torch.randn(B, n, 7, generator=g)
    first = None
    for uses in (0, 1, None):
        if uses is None:
            m.eval()
        out, _ = m(x.to(be.device), adj.to(be.device))
        P, embs = _encoder64(m, x.double(), adj.double(), uses)
        e = torch.cat([t.max(1)[0] for t in embs], 1) if graph_mode else torch.cat(embs, 2)
        want = e @ P["pred_model.weight"].t() + P["pred_model.bias"]
        # fp32 through four layers of sums of at most 30 terms, each layer norm dividing by a deviation of a few hundredths of the rows' level
        assert (f64(out) - want.detach()).abs().max() <= 2e-4
        up = torch.randn(out.shape, generator=g)
        grads = torch.autograd.grad(out, list(m.parameters()), up.to(be.device))
        want_g = torch.autograd.grad(want, list(P.values()), up.double())
        for (k, _), a, b in zip(m.named_parameters(), grads, want_g):
            assert (f64(a) - b).abs().max() <= 5e-4 * max(1.0, float(b.abs().max())), k
        if uses == 0:
            first = out.detach()
    m.train()
    m.reset_dropout()
    again, _ = m(x.to(be.device), adj.to(be.device))
    assert torch.equal(again, first)


def test_encoder_options_keep_what_was(monkeypatch):
    """Without the options: no new parameters, torch's dropout; with them: the state_dict's keys, the CPU evaluation in torch, bn and layer_norm exclude one another,
    the kernels' job refuses such a state_dict and the explainer sends it to the PyTorch-ROCm route."""
    from gnn_model_explainer_amd.explainer import explain
    plain = models.GcnEncoderNode(7, 20, 20, 3, 4, bn=True, dropout=0.4)
    assert plain.norms is None and not any(k.startswith("norms") for k in plain.state_dict())
    assert all(isinstance(c.dropout_layer, torch.nn.Dropout) for c in plain.conv_block)
    m = _encoder(models.GcnEncoderNode, layers=3)
    assert {k for k in m.state_dict() if k.startswith("norms")} == {"norms.%d.%s" % (i, k) for i in (0, 1) for k in ("weight", "bias")}
    assert all(isinstance(c.dropout_layer, models.CounterDropout) for c in m.conv_block)
    x, adj = torch.randn(1, 6, 7, generator=torch.Generator().manual_seed(1)), torch.ones(1, 6, 6)
    m.eval()
    out, _ = m(x, adj)
    P, embs = _encoder64(m, x.double(), adj.double(), None)
    assert (out.double() - (torch.cat(embs, 2) @ P["pred_model.weight"].t() + P["pred_model.bias"])).abs().max() <= 2e-4
    m.train()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m(x, adj)
    with pytest.raises(ValueError, match="choose one"):
        models.GcnEncoderNode(7, 20, 20, 3, 3, bn=True, args=argparse.Namespace(layer_norm=True))
    args = argparse.Namespace(method="base", mask_act="sigmoid", bn=False)
    assert explain._torch_route_reason(args, m) == "an encoder with layer norm"
    with pytest.raises(NotImplementedError, match="layer norm"):
        engine.model_arrays(m.state_dict())


@pytest.mark.parametrize("layers", [1, 2])
def test_encoders_without_a_middle_layer(be, layers):
    """(an encoder always has its first and last convolution, whatever num_layers says; without concatenation it runs with num_layers = 1 too)"""
    args = argparse.Namespace(method="base", bias=True, layer_norm=True, dropout_seed=9)
    torch.manual_seed(3)
    m = models.GcnEncoderGraph(7, 20, 20, 3, layers, concat=False, bn=False, dropout=0.4, args=args).to(be.device).train()
    assert len(m.norms) == 1
    x, adj = torch.randn(2, 6, 7, device=be.device), torch.ones(2, 6, 6, device=be.device)
    out, _ = m(x, adj)
    h = m.norms[0](m.conv_first(x, adj)[0])
    assert torch.equal(out, m.pred_model(m.conv_last(h, adj)[0].max(dim=1)[0]))


def test_explanations_with_seeded_dropout_are_reproducible(be, tmp_path, monkeypatch):
    """An encoder with layer norm and seeded dropout through Explainer.explain (the PyTorch-ROCm route, dropout active as in the reference: explain.py:135): a target's
    explanation does not depend on what was explained before it nor on torch's generators."""
    import helpers
    from gnn_model_explainer_amd.explainer import explain
    from test_explainer_api import _args as api_args
    monkeypatch.setitem(explain._ENGINE, "device", be.device)
    ck = helpers.load_ckpt("syn1")
    args = api_args(tmp_path, 4, "syn1", layer_norm=True, dropout_seed=7)
    torch.manual_seed(0)
    model = models.GcnEncoderNode(ck["feat"].shape[1], 20, 20, ck["pred"].shape[1], 3, bn=False, dropout=0.3, args=args)
    ex = explain.Explainer(model, ck["adj"][None].astype(np.float64), ck["feat"][None].astype(np.float64), ck["label"][None], ck["pred"][None], None, args,
                           writer=None, print_training=False, graph_mode=False, graph_idx=-1)
    def run(t, junk):
        if junk:
            torch.randn(17, device=be.device)
            model.train()
            model(torch.randn(1, 5, ck["feat"].shape[1], device=be.device), torch.ones(1, 5, 5, device=be.device)) if be.device != "cpu" or be.lib else None
        torch.manual_seed(1000 + t)
        return ex.explain(t)
    a = run(302, False)
    run(309, False)
    b = run(302, True)
    assert np.isfinite(a).all() and np.array_equal(a, b) and (a != 0).any()


def test_an_explanation_leaves_the_count_of_a_training_run_alone(be, tmp_path, monkeypatch):
    import helpers
    from gnn_model_explainer_amd.explainer import explain
    from test_explainer_api import _args as api_args
    monkeypatch.setitem(explain._ENGINE, "device", be.device)
    ck = helpers.load_ckpt("syn1")
    args = api_args(tmp_path, 3, "syn1", layer_norm=True, dropout_seed=7)
    model = models.GcnEncoderNode(ck["feat"].shape[1], 20, 20, ck["pred"].shape[1], 4, bn=False, dropout=0.3, args=args).to(be.device).train()
    x, adj = torch.randn(1, 5, ck["feat"].shape[1], device=be.device), torch.ones(1, 5, 5, device=be.device)
    model(x, adj), model(x, adj)
    ex = explain.Explainer(model, ck["adj"][None].astype(np.float64), ck["feat"][None].astype(np.float64), ck["label"][None], ck["pred"][None], None, args,
                           writer=None, print_training=False, graph_mode=False, graph_idx=-1)
    ex.explain(302)
    assert [c.dropout_layer.uses for c in model.conv_block] == [2, 2]
    def broken(e):
        raise ArithmeticError("no head")
    monkeypatch.setattr(model.pred_model, "forward", broken)
    with pytest.raises(ArithmeticError):
        ex.explain(302)
    assert [c.dropout_layer.uses for c in model.conv_block] == [2, 2]
    assert model.reset_dropout() == [2, 2] and model.reset_dropout([5, 5]) == [0, 0] and model.reset_dropout() == [5, 5]


def test_command_line_run_of_such_an_encoder(be, tmp_path, monkeypatch):
    """The command line from a checkpoint of an encoder with layer norm: --layer-norm rebuilds it, --dropout and --dropout-seed act during the explanation, twice alike."""
    import helpers
    from gnn_model_explainer_amd import explainer_main
    from gnn_model_explainer_amd.explainer import explain
    monkeypatch.setitem(explain._ENGINE, "device", be.device)
    ck = helpers.load_ckpt("syn1")
    torch.manual_seed(2)
    m = models.GcnEncoderNode(ck["feat"].shape[1], 20, 20, ck["pred"].shape[1], 3, bn=False, args=argparse.Namespace(layer_norm=True))
    cg = {"adj": ck["adj"][None].astype(np.float64), "feat": ck["feat"][None].astype(np.float64), "label": ck["label"][None], "pred": ck["pred"][None], "train_idx": []}
    torch.save({"model_state": m.state_dict(), "cg": cg}, tmp_path / "syn1_base_h20_o20.pth.tar")
    def run(*extra):
        torch.manual_seed(5)
        out = explainer_main.main(["--dataset=syn1", "--explain-node=302", "--epochs=3", "--layer-norm", "--ckptdir=%s" % tmp_path, "--logdir=%s" % tmp_path] + list(extra))
        return np.asarray(out)
    plain, a, b, other = run(), run("--dropout=0.4", "--dropout-seed=3"), run("--dropout=0.4", "--dropout-seed=3"), run("--dropout=0.4", "--dropout-seed=4")
    assert np.isfinite(plain).all() and np.array_equal(a, b) and not np.array_equal(a, plain) and not np.array_equal(a, other)


def test_command_line_options():
    from gnn_model_explainer_amd import explainer_main
    a = explainer_main.arg_parse(["--layer-norm", "--dropout", "0.25", "--dropout-seed", "11"])
    assert a.layer_norm is True and a.dropout == 0.25 and a.dropout_seed == 11
    a = explainer_main.arg_parse([])
    assert a.layer_norm is False and a.dropout_seed is None


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("layer_norm", [False, True])
def test_a_recomputed_forward_pass_draws_the_masks_it_drew_first(be, layer_norm, reentrant):
    """torch.utils.checkpoint runs the forward pass again inside the backward pass: with the use given the gradients are those without it, bit for bit; by the count of
    calls it would draw other masks, and is refused."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(16)
    adj = (torch.rand(2, 12, 12, generator=g) < 0.4).float().to(be.device)
    x0, up = torch.randn(2, 12, 7, generator=g).to(be.device), torch.randn(2, 12, 3, generator=g).to(be.device)
    def grads(how):
        torch.manual_seed(3)
        args = argparse.Namespace(method="base", bias=True, layer_norm=layer_norm, dropout_seed=9)
        m = models.GcnEncoderNode(7, 20, 20, 3, 4, bn=False, dropout=0.4, args=args).to(be.device).train()
        x, kw = x0.clone().requires_grad_(), {} if how == "counted" else {"dropout_use": 5}
        f = lambda x, adj: m(x, adj, **kw)[0]
        out = f(x, adj) if how == "plain" else checkpoint(f, x, adj, use_reentrant=reentrant)
        out.backward(up)
        return [out.detach(), x.grad] + [p.grad for p in m.parameters()]
    want, got = grads("plain"), grads("checkpoint")
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and bool((want[1] != 0).any())
    with pytest.raises(RuntimeError, match="dropout_use"):
        grads("counted")


def test_the_use_of_an_encoders_dropout_can_be_given(be):
    """dropout_use=n draws what the n-th counted pass draws and leaves the count alone."""
    m = _encoder(models.GcnEncoderNode).to(be.device).train()
    x, adj = torch.randn(1, 6, 7, generator=torch.Generator().manual_seed(1)).to(be.device), torch.ones(1, 6, 6, device=be.device)
    with torch.no_grad():
        counted = [m(x, adj)[0] for _ in range(3)]
        assert all(torch.equal(m(x, adj, dropout_use=i)[0], counted[i]) for i in (2, 0, 1)) and not torch.equal(counted[0], counted[1])
        assert torch.equal(m(x, adj)[0], m(x, adj, dropout_use=3)[0])
        m.eval()
        assert torch.equal(m(x, adj, dropout_use=3)[0], m(x, adj)[0])
    with pytest.raises(ValueError, match="step"):
        m.train()(x, adj, dropout_use=-1)


def test_a_resumed_training_run_goes_on_with_the_next_masks(be, tmp_path):
    """The count of uses travels with the state_dict; encoders with and without seeded dropout load one another's."""
    x, adj = torch.randn(1, 6, 7, generator=torch.Generator().manual_seed(1)).to(be.device), torch.ones(1, 6, 6, device=be.device)
    m = _encoder(models.GcnEncoderNode).to(be.device).train()
    with torch.no_grad():
        m(x, adj), m(x, adj)
        torch.save(m.state_dict(), tmp_path / "mid_run.pth")
        third = m(x, adj)[0]
        state = torch.load(tmp_path / "mid_run.pth", weights_only=True)
        resumed = _encoder(models.GcnEncoderNode).to(be.device).train()
        assert not resumed.load_state_dict(state).missing_keys
        assert torch.equal(resumed(x, adj)[0], third) and not torch.equal(resumed(x, adj)[0], third)
    # an encoder without seeded dropout: its state_dict loads and leaves the count, and it loads one with a count
    for p in (0.0, 0.4):
        other = models.GcnEncoderNode(7, 20, 20, 3, 4, bn=False, dropout=p, args=argparse.Namespace(method="base", bias=True, layer_norm=True))
        assert not any(k.endswith("uses") for k in other.state_dict())
        other.load_state_dict(state)
        resumed.load_state_dict(other.state_dict())
        assert [c.dropout_layer.uses for c in resumed.conv_block] == [4, 4]
    with pytest.raises(RuntimeError, match="nonsense"):
        resumed.load_state_dict({**state, "conv_block.0.dropout_layer.nonsense": state["conv_first.bias"]})


@pytest.mark.parametrize("layer_norm", [False, True])
@pytest.mark.parametrize("graph_mode", [False, True])
def test_shares_of_a_batch_draw_the_whole_batches_masks(be, graph_mode, layer_norm):
    """Data-parallel ranks: first_graph counts a share's rows from where it lies in the batch."""
    g = torch.Generator().manual_seed(2)
    adj, x = (torch.rand(5, 9, 9, generator=g) < 0.5).float().to(be.device), torch.randn(5, 9, 7, generator=g).to(be.device)
    args = argparse.Namespace(method="base", bias=True, layer_norm=layer_norm, dropout_seed=9)
    torch.manual_seed(3)
    m = (models.GcnEncoderGraph if graph_mode else models.GcnEncoderNode)(7, 20, 20, 3, 4, bn=False, dropout=0.4, args=args).to(be.device).train()
    with torch.no_grad():
        whole = m(x, adj, dropout_use=3)[0]
        # each graph's outputs are those of its own rows; the products over a smaller batch may add up in another order: the bound of the encoder against 64 bits above
        at = 0
        for share in (2, 1, 2):
            part = m(x[at:at + share], adj[at:at + share], dropout_use=3, first_graph=at)[0]
            assert torch.allclose(part, whole[at:at + share], rtol=0, atol=2e-4), at
            if at:
                same = m(x[at:at + share], adj[at:at + share], dropout_use=3)[0]      # the first share's masks: far beyond any rounding
                assert (same - whole[at:at + share]).abs().max() > 1e-2
            at += share


def test_seeded_dropout_in_a_replica_of_data_parallel_is_refused(be):
    """(_replicate_for_data_parallel is what torch.nn.DataParallel makes its copies with: no second device needed)"""
    m = _encoder(models.GcnEncoderNode).to(be.device).train()
    def replica(mod):
        r = mod._replicate_for_data_parallel()
        for k, v in mod._parameters.items():
            setattr(r, k, v)
        for k, v in mod._modules.items():
            r._modules[k] = None if v is None else replica(v)
        return r
    r = replica(m)
    x, adj = torch.randn(1, 6, 7, device=be.device), torch.ones(1, 6, 6, device=be.device)
    for kw in ({}, {"dropout_use": 1}):
        with pytest.raises(RuntimeError, match="DataParallel"):
            r(x, adj, **kw)
    m(x, adj)
    assert torch.isfinite(replica(m.eval())(x, adj)[0]).all()


# ---------------------------------------------------------------- hardware only ----------------------------------------------------------------
@pytest.mark.gpu
def test_captured_training_step_draws_new_masks_at_every_replay():
    dev = "cuda:0"
    g = torch.Generator().manual_seed(4)
    x, dh, dd = (torch.randn(333, 60, generator=g).to(dev) for _ in range(3))
    w, b = torch.rand(60, generator=g).to(dev), torch.rand(60, generator=g).to(dev)
    state = torch.tensor([77, 0], dtype=torch.int64, device=dev)
    def step():
        h, d, mean, rstd = ops.layer_norm_dropout_forward(x, w, b, 0.3, state, 5, relu=True)
        e = ops.dropout(d, 0.2, state, 6)
        return (h, d, e) + ops.layer_norm_dropout_backward(dh, dd, x, mean, rstd, w, 0.3, state, 5, relu=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                   # two graphs: neither shares a workspace with the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
            state[1].add_(10)
        graphs.append((graph, out))
    state[1] = 0
    seen = []
    for i in range(6):
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        now = int(state[1])
        state[1] = now - 10
        eager = step()
        state[1] = now
        assert now == 10 * (i + 1)
        assert all(torch.equal(p, q) for p, q in zip(replayed, eager)), i
        seen.append(replayed[1])
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
def test_captured_autograd_step():
    dev = "cuda:0"
    x = torch.randn(700, 20, generator=torch.Generator().manual_seed(4)).to(dev).requires_grad_()
    w, b = torch.ones(20, device=dev, requires_grad=True), torch.zeros(20, device=dev, requires_grad=True)
    up = torch.randn(700, 20, generator=torch.Generator().manual_seed(5)).to(dev)
    def step():
        h, d = ops.layer_norm_dropout(x, w, b, 0.5, 3, 1, relu=True)
        return torch.autograd.grad([h, d], [x, w, b], [up, up])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        assert all(torch.equal(p, q) for p, q in zip(step(), want))


@pytest.mark.gpu
def test_other_streams_at_once():
    dev = "cuda:0"
    xs = [torch.randn(5000, 257, generator=torch.Generator().manual_seed(i)).to(dev) for i in range(4)]
    w = torch.rand(257, device=dev) + 0.5
    def work(i):
        h, d, mean, rstd = ops.layer_norm_dropout_forward(xs[i], w, w, 0.1, i)
        return (h, d) + ops.layer_norm_dropout_backward(h, d, xs[i], mean, rstd, w, 0.1, i)
    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows whose elements lie beyond 2^31 and 2^32 elements (8.6 GB of bf16): the last rows equal the same rows alone."""
    dev, cols = "cuda:0", 1030
    rows = (1 << 32) // cols + 40
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    x.view(-1)[:1 << 20].normal_()
    tail = torch.randn(64, cols, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    for at in (0, (1 << 31) // cols - 32, rows - 64):
        x[at:at + 64] = tail
    w = (torch.rand(cols, device=dev) + 0.5)
    y = ops.dropout(x, 0.1, 5)
    for at in (0, (1 << 31) // cols - 32, rows - 64):
        assert torch.equal(y[at:at + 64], ops.dropout(tail, 0.1, 5, row_offset=at)), at
    del y
    y, mean, rstd = ops.layer_norm_forward(x, w, w)
    small, m1, r1 = ops.layer_norm_forward(tail, w, w)
    for at in (0, (1 << 31) // cols - 32, rows - 64):
        assert torch.equal(y[at:at + 64], small) and torch.equal(mean[at:at + 64], m1), at
    del y
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd, w)
    dx1 = ops.layer_norm_backward(tail, tail, m1, r1, w)[0]
    for at in (0, (1 << 31) // cols - 32, rows - 64):
        assert torch.equal(dx[at:at + 64], dx1), at


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits():
    dev = "cuda:0"
    x, dy = (torch.randn(20000, 130, generator=torch.Generator().manual_seed(i)).to(dev) for i in range(2))
    w = torch.ones(130, device=dev)
    _, mean, rstd = ops.layer_norm_forward(x, w)
    first = ops.layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.layer_norm_backward(dy, x, mean, rstd, w)))
