"""GPU parity of layer normalisation, dropout and the two fused behind a residual connection
against the fp64 oracle, through the C ABI.

Tolerances, with u = 2^-24 and u_T half a unit of the storage type's last place: every sum a kernel
forms is a tree of at most 64 additions in a row (8 x 4 or 8 x 5 per thread, 5 across the warp, at
most 16 warps), so a mean is off by at most 64 u times the mean of the magnitudes; the variance
doubles that, the few products after it add less than the margin to 128 (forward) and 256 (backward,
where two of those sums and the forward's rounded statistics come together).  One rounding to T ends it.
"""
import numpy as np
import pytest
import torch

from ginn_b200 import binding as B
from oracle import oracle as orc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = [np.float32, np.float16]
# rows: one; below, at and behind the borders of the register variants; unaligned; longer than the
# registers of a CTA; cols: one, fewer than the groups of a CTA, several sweeps of a full grid
SHAPES = [(1, 1), (1, 70), (2, 3), (7, 5), (8, 129), (31, 33), (32, 64), (255, 9), (256, 1300), (257, 6), (384, 2500), (512, 40),
          (520, 40), (1000, 77), (1024, 300), (1032, 19), (2048, 700), (2056, 5), (4096, 160), (5001, 9), (8192, 310),
          (8200, 6), (16384, 4), (16391, 3), (20000, 5)]


def u_of(dt):
    return np.finfo(dt).eps / 2


def bound(got, ref, tol, what):
    got = np.asarray(got, np.float64)
    assert got.shape == np.shape(ref), what
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside; worst {np.nanmax(np.abs(got - ref) / np.maximum(tol, 1e-300)):.2f} x the bound"


def data(rng, rows, cols, dt):
    """Columns with means and scales of their own."""
    x = rng.standard_normal((rows, cols)) * (0.3 + rng.random(cols)) + rng.standard_normal(cols)
    return x.astype(dt)


def check_forward(x, gain, bias, y, mean, rstd, dt, eps=1e-5):
    ref, m, r = orc.layer_norm_forward(x, gain, bias, eps)
    x = x.astype(np.float64)
    top = np.abs(x).max(0)
    xh = (x - m) * r
    g = np.ones(len(x)) if gain is None else np.abs(gain.astype(np.float64))
    b = 0 if bias is None else np.abs(bias.astype(np.float64))[:, None]
    # relative error of rstd: that of var + eps halved, the latter from differences to an inexact mean
    rel = 128 * U * (1 + (top * r) ** 2)
    bound(mean, m, 64 * U * top, "mean")
    bound(rstd, r, rel * r, "rstd")
    bound(y, ref, u_of(dt) * np.abs(ref) + g[:, None] * (128 * U * top * r + rel * np.abs(xh)) + 4 * U * b + 2.0 ** -25, "y")


def check_backward(x, gain, mean, rstd, dy, got, dt, dh=None, old=None, mask=None):
    """got: dict of dres (gradient of x), dx, dgain, dbias."""
    dx, dg, db = orc.layer_norm_backward(x, gain, mean, rstd, dy)
    x, dy = x.astype(np.float64), np.abs(dy.astype(np.float64))
    s = 1 + np.abs(x).max(0) * rstd
    xh = np.abs((x - mean) * rstd)
    g = dy if gain is None else dy * np.abs(gain.astype(np.float64))[:, None]
    inner = 256 * U * rstd * s * (g + g.mean(0) + xh * (g * xh).mean(0) + (g * s).mean(0) * s)
    if dh is not None:
        dx = dx + dh
        inner = inner + U * np.abs(dx)
    old = old or {}
    for name in ("dres", "dx", "dgain", "dbias"):
        if name not in got:
            continue
        ref, tol = {"dres": (dx, inner), "dx": (dx if mask is None else dx * mask, inner if mask is None else inner * mask),
                    "dgain": (dg, 256 * U * (dy * (xh + s)).sum(1)), "dbias": (db, 64 * U * dy.sum(1))}[name]
        if name in old:
            ref = ref + old[name]
            tol = tol + 2 * U * np.abs(ref)
        bound(got[name], ref, tol + u_of(dt) * np.abs(ref) + 2.0 ** -25 + 4 * U * np.abs(ref), name)


def host(t):
    return t.float().cpu().numpy().astype(np.float64) if t.dtype == torch.float32 else B.to_host(t).astype(np.float64)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(gpu, dt, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    x, dy, dx0 = (data(rng, rows, cols, dt) for _ in range(3))
    gain, bias, dg0, db0 = (rng.standard_normal(rows).astype(dt) for _ in range(4))
    X, DY = B.from_host(x), B.from_host(dy)
    G, Bi = B.from_host(gain), B.from_host(bias)
    Y = B.colmajor(rows, cols, X.dtype, fill=7.0)
    M, R = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.layer_norm_forward(X, G, Bi, Y, M, R)
    check_forward(x, gain, bias, host(Y), host(M), host(R), dt)
    for accumulate in (False, True):
        DX, DG, DB = B.from_host(dx0), B.from_host(dg0), B.from_host(db0)
        gpu.layer_norm_backward(X, G, M, R, DY, DX, DG, DB, accumulate=accumulate)
        old = dict(dres=dx0.astype(np.float64), dgain=dg0.astype(np.float64), dbias=db0.astype(np.float64)) if accumulate else None
        check_backward(x, gain, host(M), host(R), dy, dict(dres=host(DX), dgain=host(DG), dbias=host(DB)), dt, old=old)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols,pad,shift", [(384, 50, 8, 0), (384, 50, 3, 0), (1000, 30, 0, 1), (129, 17, 5, 1), (8192, 5, 8, 0), (9000, 5, 1, 1)])
def test_padded_and_shifted_columns(gpu, dt, rows, cols, pad, shift):
    """Leading dimensions above the rows and bases off the 16-byte grid; what lies between the
    columns stays as it was."""
    rng = np.random.default_rng(rows + pad)
    tdt = torch.float32 if dt == np.float32 else torch.float16
    ld = rows + pad

    def place(a):
        buf = torch.full((ld * cols + shift,), 3.0, dtype=tdt, device="cuda")
        t = torch.as_strided(buf, (rows, cols), (1, ld), shift)
        t.copy_(torch.from_numpy(np.ascontiguousarray(a)))
        return t, buf

    x, dy, zero = data(rng, rows, cols, dt), data(rng, rows, cols, dt), np.zeros((rows, cols), dt)
    gain, bias = rng.standard_normal(rows).astype(dt), rng.standard_normal(rows).astype(dt)
    (X, _), (DY, _), (Y, ybuf), (DX, dbuf) = place(x), place(dy), place(zero), place(zero)
    M, R = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.layer_norm_forward(X, B.from_host(gain), B.from_host(bias), Y, M, R)
    check_forward(x, gain, bias, host(Y), host(M), host(R), dt)
    gpu.layer_norm_backward(X, B.from_host(gain), M, R, DY, DX, None, None, accumulate=False)
    check_backward(x, gain, host(M), host(R), dy, dict(dres=host(DX)), dt)
    between = torch.ones(ld * cols + shift, dtype=torch.bool, device="cuda")
    torch.as_strided(between, (rows, cols), (1, ld), shift).fill_(False)
    assert (ybuf[between] == 3).all() and (dbuf[between] == 3).all()


@pytest.mark.parametrize("dt", DT)
def test_without_gain_bias_and_statistics(gpu, dt):
    rng = np.random.default_rng(5)
    x, dy = data(rng, 200, 33, dt), data(rng, 200, 33, dt)
    X, Y = B.from_host(x), B.colmajor(200, 33, B.from_host(x).dtype)
    gpu.layer_norm_forward(X, None, None, Y)
    _, m, r = orc.layer_norm_forward(x)
    check_forward(x, None, None, host(Y), m, r, dt)
    M, R = torch.from_numpy(m).float().cuda(), torch.from_numpy(r).float().cuda()
    DG = torch.zeros(200, dtype=X.dtype, device="cuda")
    gpu.layer_norm_backward(X, None, M, R, B.from_host(dy), None, DG, None)  # the weight gradient alone
    check_backward(x, None, host(M), host(R), dy, dict(dgain=host(DG)), dt)
    gpu.layer_norm_forward(X, None, None, X)  # in place
    check_forward(x, None, None, host(X), m, r, dt)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(1024, 40), (1001, 9), (5000, 9), (9000, 7), (9001, 7), (16384, 3), (70000, 3)])
def test_gradient_over_the_upstream_one(gpu, dt, rows, cols):
    """dx in dy's place, the weight gradients from the dy that was there."""
    rng = np.random.default_rng(rows)
    x, dy, gain = data(rng, rows, cols, dt), data(rng, rows, cols, dt), rng.standard_normal(rows).astype(dt)
    X, G = B.from_host(x), B.from_host(gain)
    Y, M, R = B.colmajor(rows, cols, X.dtype), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.layer_norm_forward(X, G, None, Y, M, R)
    D, DG, DB = B.from_host(dy), torch.empty(rows, dtype=X.dtype, device="cuda"), torch.empty(rows, dtype=X.dtype, device="cuda")
    gpu.layer_norm_backward(X, G, M, R, D, D, DG, DB, accumulate=False)
    check_backward(x, gain, host(M), host(R), dy, dict(dres=host(D), dgain=host(DG), dbias=host(DB)), dt)


@pytest.mark.parametrize("dt", DT)
def test_constant_column_and_large_offset(gpu, dt):
    """A column without variance gives the bias and a finite gradient; a mean a thousand times the
    spread does not cancel the spread away."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((640, 3))
    x[:, 0] = 1.5
    x[:, 1] += 1000 if dt == np.float32 else 30
    x = x.astype(dt)
    X = B.from_host(x)
    Y, M, R = B.colmajor(640, 3, X.dtype), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    gpu.layer_norm_forward(X, None, None, Y, M, R)
    y, m, r = orc.layer_norm_forward(x)
    assert (host(Y)[:, 0] == 0).all()
    # the mean is off by 64 u |mean| at most, which moves y by that times rstd
    bound(host(Y), y, u_of(dt) * np.abs(y) + 2 * 64 * U * np.abs(m) * r * (1 + np.abs(y)) + 256 * U, "y")
    DX = B.colmajor(640, 3, X.dtype)
    gpu.layer_norm_backward(X, None, M, R, B.from_host(rng.standard_normal((640, 3)).astype(dt)), DX, accumulate=False)
    assert np.isfinite(host(DX)).all()


@pytest.mark.parametrize("dt", DT)
def test_no_columns_still_assigns_weight_gradients(gpu, dt):
    tdt = torch.float32 if dt == np.float32 else torch.float16
    X = torch.empty((0, 40), dtype=tdt, device="cuda").t()
    M = torch.empty(0, device="cuda")
    for accumulate, want in ((True, 2.0), (False, 0.0)):
        DG, DB = torch.full((40,), 2.0, dtype=tdt, device="cuda"), torch.full((40,), 2.0, dtype=tdt, device="cuda")
        gpu.layer_norm_backward(X, None, M, M, X, X, DG, DB, accumulate=accumulate)
        assert (DG == want).all() and (DB == want).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.99])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (7, 3, 0), (8, 200, 8), (100, 1000, 0), (101, 77, 3), (104, 77, 4), (1 << 20, 3, 0)])
def test_dropout(gpu, dt, p, rows, cols, pad):
    rng = np.random.default_rng(rows + cols)
    x, res, dx0 = (rng.standard_normal((rows, cols)).astype(dt) for _ in range(3))
    seed, offset = 0x123456789ABCDEF0 + rows, (3 << 32) + 17
    mask = orc.dropout_mask(rows, cols, p, seed, offset)
    X, RS, DX, Y = (B.from_host(a, ld=rows + pad) for a in (x, res, dx0, x))
    x, res, dx0 = (a.astype(np.float64) for a in (x, res, dx0))
    gpu.dropout_forward(X, Y, p, seed, offset)
    bound(host(Y), x * mask, u_of(dt) * np.abs(x * mask) + 4 * U * np.abs(x * mask) + 2.0 ** -25, "y")
    gpu.dropout_forward(X, Y, p, seed, offset, residual=RS)
    bound(host(Y), res + x * mask, u_of(dt) * np.abs(res + x * mask) + 4 * U * (np.abs(x * mask) + np.abs(res)) + 2.0 ** -25, "y + residual")
    gpu.dropout_backward(X, DX, p, seed, offset)
    bound(host(DX), dx0 + x * mask, u_of(dt) * np.abs(dx0 + x * mask) + 4 * U * (np.abs(x * mask) + np.abs(dx0)) + 2.0 ** -25, "dx")
    gpu.dropout_backward(X, X, p, seed, offset, accumulate=False)  # in place
    bound(host(X), x * mask, u_of(dt) * np.abs(x * mask) + 4 * U * np.abs(x * mask) + 2.0 ** -25, "dx in place")


def test_dropout_element_numbers_past_32_bits(gpu):
    """Elements behind number 2^32 take blocks of their own: the last columns of a matrix of 4.4e9
    Half elements against the oracle, formed for those blocks alone."""
    rows, cols = 1 << 21, 2101
    x = torch.ones((cols, rows), dtype=torch.float16, device="cuda").t()
    gpu.dropout_forward(x, x, 0.5, 99, 5)
    n, tail = rows * cols, 4096
    block = np.arange((n - tail) // 8, n // 8, dtype=np.uint64)
    ctr = np.stack([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, 5), np.zeros_like(block)])
    w = orc.philox4x32(ctr, (99, 0))
    numbers = np.stack([h for a in w for h in (a & np.uint64(0xFFFF), a >> np.uint64(16))], 1).reshape(-1)
    got = x[-tail:, -1].cpu().numpy()
    np.testing.assert_array_equal(got, np.where(numbers >= 32768, 2.0, 0.0).astype(np.float16))


def test_dropped_places_may_hold_anything(gpu):
    mask = orc.dropout_mask(64, 64, 0.5, 1, 2)
    x = np.where(mask > 0, 1.0, np.nan).astype(np.float32)
    X = B.from_host(x)
    gpu.dropout_forward(X, X, 0.5, 1, 2)
    np.testing.assert_array_equal(B.to_host(X), mask)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(1, 3), (33, 40), (256, 900), (1001, 60), (1024, 500), (2049, 40), (8192, 170), (8193, 7), (16400, 5)])
def test_residual_norm(gpu, dt, rows, cols):
    rng = np.random.default_rng(rows * 3 + cols)
    x, res, dy, dh, dx0, dr0 = (data(rng, rows, cols, dt) for _ in range(6))
    gain, bias = rng.standard_normal(rows).astype(dt), rng.standard_normal(rows).astype(dt)
    rnd = dict(p=0.25, seed=rows + (1 << 40), offset=cols)
    mask = orc.dropout_mask(rows, cols, **rnd)
    X, RS, DY, DH = (B.from_host(a) for a in (x, res, dy, dh))
    G, Bi = B.from_host(gain), B.from_host(bias)
    H, Y = B.colmajor(rows, cols, X.dtype), B.colmajor(rows, cols, X.dtype)
    M, R = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.residual_norm_forward(X, RS, G, Bi, H, Y, M, R, **rnd)
    h = res.astype(np.float64) + x.astype(np.float64) * mask
    bound(host(H), h, u_of(dt) * np.abs(h) + 4 * U * (np.abs(res) + np.abs(x * mask)), "h")
    check_forward(B.to_host(H), gain, bias, host(Y), host(M), host(R), dt)
    for accumulate in (False, True):
        DX, DR = B.from_host(dx0), B.from_host(dr0)
        DG, DB = torch.full((rows,), 0.5, dtype=X.dtype, device="cuda"), torch.full((rows,), 0.5, dtype=X.dtype, device="cuda")
        gpu.residual_norm_backward(H, G, M, R, DY, DH, DX, DR, DG, DB, accumulate=accumulate, **rnd)
        old = dict(dx=dx0.astype(np.float64), dres=dr0.astype(np.float64), dgain=0.5, dbias=0.5) if accumulate else None
        check_backward(B.to_host(H), gain, host(M), host(R), dy, dict(dx=host(DX), dres=host(DR), dgain=host(DG), dbias=host(DB)), dt,
                       dh=dh.astype(np.float64), old=old, mask=mask)
    # in place: h over the residual, dres over dh; dropout off
    gpu.residual_norm_forward(X, RS, G, Bi, RS, Y, M, R)
    h = res.astype(np.float64) + x
    bound(host(RS), h, u_of(dt) * np.abs(h) + 4 * U * (np.abs(res) + np.abs(x)), "h in place")
    gpu.residual_norm_backward(RS, G, M, R, DY, DH, None, DH, None, None, accumulate=False)
    check_backward(B.to_host(RS), gain, host(M), host(R), dy, dict(dres=host(DH)), dt, dh=dh.astype(np.float64))


def test_results_do_not_depend_on_the_run(gpu):
    """The same call gives the same bits, weight gradients included."""
    rng = np.random.default_rng(8)
    X, DY = (B.from_host(data(rng, 1024, 9000, np.float16)) for _ in range(2))
    M, R = torch.zeros(9000, device="cuda"), torch.ones(9000, device="cuda")
    seen = []
    for _ in range(5):
        DX, DG, DB = B.colmajor(1024, 9000, X.dtype), torch.empty(1024, dtype=X.dtype, device="cuda"), torch.empty(1024, dtype=X.dtype, device="cuda")
        gpu.layer_norm_backward(X, None, M, R, DY, DX, DG, DB, accumulate=False)
        seen.append((DX, DG, DB))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_captured_step_draws_a_new_mask_at_every_replay(gpu):
    """A forward and backward pass in one CUDA graph, with the mask's offset advanced by a device
    counter; two graphs of the same calls run on two streams."""
    rows, cols = 256, 500
    rng = np.random.default_rng(9)
    x, dy = data(rng, rows, cols, np.float32), data(rng, rows, cols, np.float32)
    gain = rng.standard_normal(rows).astype(np.float32)

    class Step:
        def __init__(self):
            self.X, self.DY, self.G = B.from_host(x), B.from_host(dy), B.from_host(gain)
            self.H, self.Y, self.DX = (B.colmajor(rows, cols, torch.float32) for _ in range(3))
            self.M, self.R = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
            self.DG, self.DB = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
            self.step = torch.zeros(1, dtype=torch.int64, device="cuda")

        def __call__(self):
            rnd = dict(p=0.3, seed=4, offset=10, step=self.step)
            gpu.residual_norm_forward(self.X, None, self.G, None, self.H, self.Y, self.M, self.R, **rnd)
            gpu.residual_norm_backward(self.H, self.G, self.M, self.R, self.DY, None, self.DX, None, self.DG, self.DB, accumulate=False, **rnd)
            self.step.add_(1)

    steps, graphs, streams = [Step(), Step()], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in steps:
        s()
        s.step.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s()
        graphs.append(g)
    for replay in range(3):
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        mask = orc.dropout_mask(rows, cols, 0.3, 4, 10 + replay)
        for s in steps:
            h = x * mask
            bound(host(s.H), h, 8 * U * np.abs(h), "h")
            check_forward(B.to_host(s.H), gain, None, host(s.Y), host(s.M), host(s.R), np.float32)
            check_backward(B.to_host(s.H), gain, host(s.M), host(s.R), dy, dict(dx=host(s.DX), dgain=host(s.DG), dbias=host(s.DB)),
                           np.float32, mask=mask)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows", [9000, 40000, 70000])
def test_long_columns_in_place_and_captured(gpu, dt, rows):
    """Columns shared by the CTAs of a cluster and those of two sweeps: y over x, and the backward pass in a graph
    beside an eager one, same bits."""
    rng = np.random.default_rng(rows)
    cols = 90
    x, dy, gain, bias = data(rng, rows, cols, dt), data(rng, rows, cols, dt), rng.standard_normal(rows).astype(dt), rng.standard_normal(rows).astype(dt)
    X, DY, G, Bi = B.from_host(x), B.from_host(dy), B.from_host(gain), B.from_host(bias)
    Y, M, R = B.from_host(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.layer_norm_forward(Y, G, Bi, Y, M, R)
    check_forward(x, gain, bias, host(Y), host(M), host(R), dt)

    def results():
        return B.colmajor(rows, cols, X.dtype), torch.empty(rows, dtype=X.dtype, device="cuda"), torch.empty(rows, dtype=X.dtype, device="cuda")

    eager, captured = results(), results()
    gpu.layer_norm_backward(X, G, M, R, DY, *eager, accumulate=False)
    check_backward(x, gain, host(M), host(R), dy, dict(dres=host(eager[0]), dgain=host(eager[1]), dbias=host(eager[2])), dt)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.layer_norm_backward(X, G, M, R, DY, *captured, accumulate=False)
    other = torch.cuda.Stream()
    again = results()
    for _ in range(3):
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            gpu.layer_norm_backward(X, G, M, R, DY, *again, accumulate=False)
    torch.cuda.synchronize()
    for a, b, c in zip(eager, captured, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_streams_at_once(gpu):
    """Calls on two streams share no scratch."""
    rng = np.random.default_rng(10)
    sets = []
    for i in range(2):
        x, dy = data(rng, 1024, 4000, np.float32), data(rng, 1024, 4000, np.float32)
        sets.append((x, dy, B.from_host(x), B.from_host(dy), torch.empty(1024, device="cuda"), torch.empty(1024, device="cuda"), torch.cuda.Stream()))
    M, R = torch.zeros(4000, device="cuda"), torch.ones(4000, device="cuda")
    torch.cuda.synchronize()
    for _ in range(10):
        for x, dy, X, DY, DG, DB, st in sets:
            with torch.cuda.stream(st):
                gpu.layer_norm_backward(X, None, M, R, DY, None, DG, DB, accumulate=False)
    torch.cuda.synchronize()
    for x, dy, X, DY, DG, DB, st in sets:
        check_backward(x, None, np.zeros(4000), np.ones(4000), dy, dict(dgain=host(DG), dbias=host(DB)), np.float32)
