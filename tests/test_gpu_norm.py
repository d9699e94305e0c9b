"""Group normalisation with an activation and counter-based dropout (fisr_amd/norm.py) against the float64 oracle.

Tolerances.  U = half a step of the tensors' type (2^-24, 2^-11, 2^-8) rounds each output once; everything before it is float32, E = 2^-24.
A thread sums at most CHAIN = 256 values one after the other at the sizes below (chunks of at most 8192 elements + 256 threads' rows, or
tensors of that size), so a mean is off by at most K E max|x| and a sum by K E sum|terms| with K = CHAIN + 32 for the joins; what one
rounding adds to a value v is E |v|.  With X = max|x| of an image:
  mean: K E X;  rstd: relative (K + 2 X rstd) E (the squared deviations' own roundings, each |x - mean| to E X)
  z = (x - mean) rstd gamma + beta: Z = |gamma| rstd K E X + |gamma xh| (K + 2 X rstd + 4) E + E |z|
  y: 1.13 Z (the activations' largest slope) + 8 E |y| (activation) + 2e-7 |z| (its approximations' absolute error) + U |y|
  dz = dy act'(z): |dy| (1.0 Z (their largest curvature) + 1e-6);  sums A, B: sum of these + K E sum |dz|, with |xh| and its error for B
  dx: rstd (|gamma| dz's + (|gamma| A's / M + |xh| |gamma| B's / M summed over the group) + 8 E of each term) + U |dx|, and what xh's error
  times S2 gives."""
import numpy as np
import pytest

import fisr_norm_oracle as no

pytestmark = pytest.mark.gpu
E, K = 2.0 ** -24, 288
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}      # a step of the smallest numbers: float16 has subnormals in range


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from fisr_amd import norm
    return torch, norm


def _type(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def _to(torch, a, t):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to("cuda:0", _type(torch, t))


def _np(t):
    return t.detach().double().cpu().numpy()


def _inputs(torch, n, h, w, c, t, seed, shift=0.5):
    """x, dy (as the type holds them, in float64 too), gamma, beta."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, h, w, c)) * (0.5 + r.random(c)) + shift + r.standard_normal(c)
    dy = r.standard_normal((n, h, w, c))
    x, dy = (_to(torch, v, t) for v in (x, dy))
    gamma, beta = (_to(torch, v, "f32") for v in (1 + 0.2 * r.standard_normal(c), 0.2 * r.standard_normal(c)))
    return x, dy, gamma, beta


def _bounds(x, groups, gamma, beta, eps, act, fac, half, tiny):
    """(y, mean, rstd, their bounds, z's bound, xh's bound) by the docstring's arithmetic."""
    y, mean, rstd, z, xh = no.forward(x, groups, gamma, beta, eps, act, fac)
    c = x.shape[3]
    X = np.abs(x).max(axis=(1, 2, 3))[:, None]
    emean = K * E * X + 0 * mean
    erstd = (K + 2 * X * rstd) * E
    exh = no.per_channel(rstd * emean, c) + np.abs(xh) * (no.per_channel(erstd, c) + 4 * E)
    ez = np.abs(gamma) * exh + E * np.abs(z)
    ey = fac * (1.13 * ez + 8 * E * np.abs(act_abs(z, act)) + 2e-7 * np.abs(z)) + half * np.abs(y) + tiny
    return y, mean, rstd, ey, emean + E * np.abs(mean), (erstd + E) * rstd, ez, exh


def act_abs(z, act):
    return np.abs(no.act(z, act))


def _within(got, want, bound, what):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(bound, bad.shape)[bad][:4])


SHAPES = [
    # (n, h, w, c, groups)
    (1, 1, 1, 1, 1), (1, 1, 1, 8, 1), (2, 1, 1, 64, 8), (3, 1, 2, 2, 2), (1, 1, 7, 6, 3), (2, 3, 3, 512, 32), (4, 6, 6, 256, 32), (1, 5, 9, 29, 29),
    (2, 13, 11, 29, 1), (2, 17, 9, 36, 4), (1, 24, 24, 64, 64), (3, 12, 12, 512, 1), (2, 19, 23, 40, 5), (2, 9, 7, 12, 2), (1, 3, 2, 600, 4),
    (1, 2, 3, 4104, 8), (2, 2, 2, 2060, 4), (1, 1, 3, 1027, 13), (37, 3, 5, 16, 16), (2, 96, 96, 64, 8), (1, 130, 70, 8, 2), (1, 191, 67, 3, 1),
    (5, 31, 33, 24, 8), (300, 2, 2, 8, 4), (2, 40, 30, 521, 521), (1, 96, 40, 1042, 521), (3, 70, 60, 1027, 13), (2, 60, 50, 2056, 4), (1, 210, 200, 72, 8),
    (2, 130, 150, 96, 32),
]
KINDS = [("f32", "none", 0.0), ("f32", "silu", 0.25), ("f16", "gelu", 0.0), ("f16", "relu", 0.1), ("bf16", "silu", 0.0), ("bf16", "gelu", 0.5), ("f32", "relu", 0.0),
         ("f32", "gelu", 0.1)]


@pytest.mark.parametrize("t,act,p", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_group_norm_and_gradients_vs_oracle(env, shape, t, act, p):
    torch, norm = env
    n, h, w, c, groups = shape
    x, dy, gamma, beta = _inputs(torch, n, h, w, c, t, n * 1000 + h * 10 + c)
    x64, dy64, g64, b64 = map(_np, (x, dy, gamma, beta))
    seed, offset = 0xFEDCBA9876543210, (1 << 40) + 77
    drop = norm.Dropout(p, seed, offset) if p else None
    fac = no.drop_factor(x64.shape, p, seed, offset) if p else np.ones_like(x64)
    y64, mean, rstd, ey, emean, erstd, ez, exh = _bounds(x64, groups, g64, b64, 1e-5, act, fac, HALF[t], TINY[t])
    y, stats = norm.group_norm(x, groups, gamma, beta, act=act, dropout=drop)
    got = _np(stats)
    _within(got[0], mean, emean, "mean")
    _within(got[1], rstd, erstd, "rstd")
    _within(_np(y), y64, ey, "y")
    # ---- gradients (relu: no gradient comes in where rounding decides the sign of z)
    if act == "relu":
        dy64 = np.where(np.abs(no.forward(x64, groups, g64, b64, 1e-5, act)[3]) <= ez, 0.0, dy64)
        dy = _to(torch, dy64, t)
    m = h * w * (c // groups)
    dx64, dg64, db64 = no.backward(dy64, x64, groups, g64, b64, 1e-5, act, fac)
    z, xh = no.forward(x64, groups, g64, b64, 1e-5, act)[3:5]
    dz = np.abs(dy64 * fac * no.act_grad(z, act))
    curve = 0.0 if act in ("none", "relu") else 1.0
    edz = np.abs(dy64) * fac * (curve * ez + 1e-6)
    ta, tb = edz + K * E * dz, (edz + K * E * dz) * np.abs(xh) + dz * exh            # errors of the terms of A, B, with the sums' own
    grp = lambda v: no.per_channel((v.sum(axis=(1, 2)) * np.abs(g64)).reshape(n, groups, -1).sum(2) / m, c)  # noqa: E731
    rs = no.per_channel(rstd, c)
    s2 = grp(dz * np.abs(xh))
    edx = rs * (np.abs(g64) * (edz + 8 * E * dz) + grp(ta) + np.abs(xh) * grp(tb) + exh * s2 + 8 * E * (grp(dz) + np.abs(xh) * s2)) + HALF[t] * np.abs(dx64) + TINY[t]
    edx = edx + no.per_channel(erstd, c) / rs * (np.abs(dx64) + rs * (np.abs(g64) * dz + grp(dz) + np.abs(xh) * s2))
    dx, dg, db = norm.group_norm_backward(dy, x, stats, groups, gamma, beta, act=act, dropout=drop)
    _within(_np(db), db64, ta.sum(axis=(0, 1, 2)) + E * np.abs(db64), "dbeta")
    _within(_np(dg), dg64, tb.sum(axis=(0, 1, 2)) + E * np.abs(dg64), "dgamma")
    _within(_np(dx), dx64, edx, "dx")


@pytest.mark.parametrize("t,act,p", KINDS[:3])
@pytest.mark.parametrize("shape", [(2, 9, 11, 1031, 1), (1, 40, 25, 2062, 2), (2, 50, 40, 1031, 1)], ids=lambda s: "x".join(map(str, s)))
def test_groups_of_more_channels_than_a_join_has_threads(env, shape, t, act, p):
    test_group_norm_and_gradients_vs_oracle(env, shape, t, act, p)


def test_mean_far_from_the_values_spread(env):
    """Values around 4096 with a spread of 1: a sum of squares about zero would lose all of it.  The bound of the docstring holds with
    X rstd = 4100."""
    torch, norm = env
    x, _, gamma, beta = _inputs(torch, 2, 40, 36, 32, "f32", 5, shift=4096.0)
    x[:, 0, 0] = 0.0                                       # the first pixel is far from all others
    x64, g64, b64 = map(_np, (x, gamma, beta))
    y64, mean, rstd, ey, emean, erstd, _, _ = _bounds(x64, 4, g64, b64, 1e-5, "none", 1.0, E, 0.0)
    y, stats = norm.group_norm(x, 4, gamma, beta)
    _within(_np(stats)[1], rstd, erstd, "rstd")
    _within(_np(y), y64, ey, "y")


def test_without_parameters_and_accumulated(env):
    torch, norm = env
    x, dy, _, _ = _inputs(torch, 2, 9, 7, 24, "f32", 8)
    one, zero = torch.ones(24, device="cuda:0"), torch.zeros(24, device="cuda:0")
    y, st = norm.group_norm(x, 3, act="silu")
    y1, st1 = norm.group_norm(x, 3, one, zero, act="silu")
    assert torch.equal(y, y1) and torch.equal(st, st1)
    a = norm.group_norm_backward(dy, x, st, 3, act="silu")
    b = norm.group_norm_backward(dy, x, st, 3, one, zero, act="silu")
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    dg, db = torch.full((24,), 2.0, device="cuda:0"), torch.full((24,), -3.0, device="cuda:0")
    norm.group_norm_backward(dy, x, st, 3, act="silu", dgamma=dg, dbeta=db, accumulate=True)
    assert torch.allclose(dg, a[1] + 2.0, rtol=0, atol=float(4 * E * (a[1].abs().max() + 2))) and torch.allclose(db, a[2] - 3.0, rtol=0, atol=float(4 * E * (a[2].abs().max() + 3)))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c,lo,hi", [(24, 0, 8), (24, 8, 24), (40, 4, 20), (40, 1, 13), (13, 2, 12)])
def test_channel_ranges_of_wider_buffers(env, t, c, lo, hi):
    """Strided pixels, bases that fit no vector load: the dense call's results, and nothing written beside the range."""
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 2, 11, 13, c, t, 4)
    k = hi - lo
    g, b = gamma[:k].clone(), beta[:k].clone()
    xs, dys = x[..., lo:hi], dy[..., lo:hi]
    drop = norm.Dropout(0.3, 5, 6)
    y0, st0 = norm.group_norm(xs.contiguous(), 2, g, b, act="gelu", dropout=drop)
    out = torch.full_like(x, 7.0)
    y1, st1 = norm.group_norm(xs, 2, g, b, act="gelu", dropout=drop, out=out[..., lo:hi])
    tol = 3 * HALF[t]                                       # another vector width sums in another order
    assert torch.allclose(st0, st1, rtol=K * E, atol=K * E)
    assert torch.allclose(y0.double(), y1.double(), rtol=tol, atol=1e-4)
    assert (out[..., :lo] == 7).all() and (out[..., hi:] == 7).all()
    a = norm.group_norm_backward(dys.contiguous(), xs.contiguous(), st0, 2, g, b, act="gelu", dropout=drop)
    dxo = torch.full_like(x, 7.0)
    d = norm.group_norm_backward(dys, xs, st0, 2, g, b, act="gelu", dropout=drop, dx=dxo[..., lo:hi])
    assert torch.allclose(a[0].double(), d[0].double(), rtol=tol, atol=1e-3) and torch.allclose(a[1], d[1], rtol=1e-4, atol=1e-4) and torch.allclose(a[2], d[2], rtol=1e-4, atol=1e-4)
    assert (dxo[..., :lo] == 7).all() and (dxo[..., hi:] == 7).all()


@pytest.mark.parametrize("shape", [(3, 33, 31, 32), (1, 90, 80, 64)])           # one launch, two
def test_in_place(env, shape):
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, *shape, "bf16", 11)
    y, st = norm.group_norm(x, 4, gamma, beta, act="silu")
    dx, _, _ = norm.group_norm_backward(dy, x, st, 4, gamma, beta, act="silu")
    xi, di = x.clone(), dy.clone()
    yi, sti = norm.group_norm(xi, 4, gamma, beta, act="silu", out=xi)
    assert yi.data_ptr() == xi.data_ptr() and torch.equal(yi, y) and torch.equal(sti, st)
    norm.group_norm_backward(di, x, st, 4, gamma, beta, act="silu", dx=di)
    assert torch.equal(di, dx)
    xx = x.clone()
    norm.group_norm_backward(dy, xx, st, 4, gamma, beta, act="silu", dx=xx)
    assert torch.equal(xx, dx)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_group(env, act, bad):
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 2, 20, 20, 16, "f32", 12)
    y0, st0 = norm.group_norm(x, 4, gamma, beta, act=act)
    d0 = norm.group_norm_backward(dy, x, st0, 4, gamma, beta, act=act)
    x2 = x.clone()
    x2[1, 3, 4, 5] = bad                                    # image 1, group 1
    y, st = norm.group_norm(x2, 4, gamma, beta, act=act)
    assert torch.isnan(y[1, :, :, 4:8]).all() and torch.isnan(st[1, 1, 1])
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[1, :, :, 4:8] = False
    assert torch.equal(y[keep], y0[keep])
    d = norm.group_norm_backward(dy, x2, st, 4, gamma, beta, act=act)
    assert torch.equal(d[0][keep], d0[0][keep]) and torch.isnan(d[1][4:8]).all()
    others = torch.tensor([k for k in range(16) if not 4 <= k < 8], device="cuda:0")
    assert torch.equal(d[1][others], d0[1][others])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count", [1, 7, 8, 9, 64, 1000, 4095, 73728, 1000003])
@pytest.mark.parametrize("p", [0.0, 1e-3, 0.1, 0.5, 0.999, 1.0])
def test_dropout_vs_oracle(env, t, count, p):
    torch, norm = env
    r = np.random.default_rng(count)
    x, res = (_to(torch, r.standard_normal(count), t) for _ in range(2))
    seed, offset = (1 << 63) + 12345, 999999999999
    fac = no.drop_factor((count,), p, seed, offset)
    drop = norm.Dropout(p, seed, offset)
    got = _np(norm.dropout(x, drop))
    want = _np(x) * fac
    assert np.array_equal(got == 0, (want == 0))
    _within(got, want, (HALF[t] + 2 * E) * np.abs(want) + TINY[t], "dropout")
    want = want + _np(res)
    got = _np(norm.dropout(x, drop, residual=res))
    _within(got, want, HALF[t] * np.abs(want) + 3 * E * (np.abs(want) + np.abs(_np(x) * fac)) + TINY[t], "with residual")
    # the gradient has the same mask
    assert torch.equal(norm.dropout_backward(x, drop), norm.dropout(x, drop))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_dropout_in_place_and_unaligned(env, t):
    torch, norm = env
    buf, rbuf = (torch.randn(5003, device="cuda:0").to(_type(torch, t)) for _ in range(2))
    drop = norm.Dropout(0.4, 3, 4)
    for off in (0, 1, 3, 8):
        x, res = buf[off:off + 4999 - off], rbuf[off:off + 4999 - off]
        want = norm.dropout(x.clone(), drop, residual=res.clone())
        assert torch.equal(norm.dropout(x, drop, residual=res), want)
        wide = torch.full((5003,), 7.0, device="cuda:0", dtype=x.dtype)
        v = wide[off:off + 4999 - off]
        v.copy_(x)
        norm.dropout(v, drop, residual=res, out=v)
        assert torch.equal(v, want) and (wide[:off] == 7).all() and (wide[4999:] == 7).all()


def test_dropped_values_are_zero_whatever_they_were(env):
    torch, norm = env
    x = torch.full((4096,), float("nan"), device="cuda:0")
    x[::2] = float("inf")
    drop = norm.Dropout(0.5, 21, 22)
    kept = torch.from_numpy(no.drop_factor((4096,), 0.5, 21, 22) > 0).cuda()
    y = norm.dropout(x, drop, residual=torch.ones_like(x))
    assert (y[~kept] == 1).all() and not torch.isfinite(y[kept]).any()
    # ... and in the fused form: what the mask drops of the gradient is not read
    xx, dy, gamma, beta = _inputs(torch, 1, 16, 16, 16, "f32", 1)
    _, st = norm.group_norm(xx, 2, gamma, beta, act="silu", dropout=drop)
    d0 = norm.group_norm_backward(dy, xx, st, 2, gamma, beta, act="silu", dropout=drop)
    dy2 = torch.where(kept.view(dy.shape), dy, torch.full_like(dy, float("nan")))
    d1 = norm.group_norm_backward(dy2, xx, st, 2, gamma, beta, act="silu", dropout=drop)
    assert all(torch.equal(a, b) for a, b in zip(d0, d1))


def test_fused_dropout_is_the_dropout_operator(env):
    torch, norm = env
    for c, t in ((32, "f32"), (36, "f16"), (29, "bf16"), (6, "f32")):
        x, dy, gamma, beta = _inputs(torch, 2, 9, 10, c, t, 31)
        drop = norm.Dropout(0.2, 8, 9)
        y, _ = norm.group_norm(x, 1, gamma, beta, act="none", dropout=drop)
        mask = norm.dropout(torch.ones_like(x), drop)
        assert torch.equal(y == 0, mask == 0), c


def test_same_bits_every_time_and_on_streams(env):
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 4, 61, 47, 64, "f32", 17)
    drop = norm.Dropout(0.1, 8, 9)

    def once():
        y, st = norm.group_norm(x, 8, gamma, beta, act="silu", dropout=drop)
        return (y, st) + norm.group_norm_backward(dy, x, st, 8, gamma, beta, act="silu", dropout=drop)

    want = once()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in side:                                      # two at once, each with a workspace of its own
            with torch.cuda.stream(s):
                got.append(once())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_captured_and_replayed(env):
    """A block's forward and backward in one graph: with the counter advanced before each replay, every replay equals the eager calls with
    that number; eager work of the same inputs runs in between."""
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 2, 30, 26, 64, "bf16", 23)
    counter = torch.zeros(1, dtype=torch.int64, device="cuda:0")

    def once(drop, drop2):
        y, st = norm.group_norm(x, 8, gamma, beta, act="silu", dropout=drop)
        z = norm.dropout(y, drop2, residual=x)
        g = norm.dropout_backward(dy, drop2)
        return (y, st, z, g) + norm.group_norm_backward(g, x, st, 8, gamma, beta, act="silu", dropout=drop)

    pair = norm.Dropout(0.1, 5, 100, counter), norm.Dropout(0.3, 5, 1 << 33, counter)
    once(*pair)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(*pair)
    seen = []
    for k in (0, 1, 2, 7, 1 << 35):
        counter.fill_(k)
        graph.replay()
        want = once(norm.Dropout(0.1, 5, 100 + k), norm.Dropout(0.3, 5, (1 << 33) + k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        seen.append(out[0].clone())
    assert not torch.equal(seen[0], seen[1])


def test_gradients_against_differences(env):
    """The loss sum(y * r) along random directions.  Central differences with h = 2^-6: the third derivative of the loss along a unit-size
    direction is below 50 here (h^2 / 6 * 50 = 2e-3); outputs are off by at most 2e-6 each, 4000 of them at random: 2e-6 * 63 / h = 8e-3."""
    torch, norm = env
    n, h, w, c = 2, 10, 10, 20
    x, r, gamma, beta = _inputs(torch, n, h, w, c, "f32", 41)
    drop = norm.Dropout(0.25, 1, 2)
    _, st = norm.group_norm(x, 4, gamma, beta, act="gelu", dropout=drop)
    grads = norm.group_norm_backward(r, x, st, 4, gamma, beta, act="gelu", dropout=drop)
    loss = lambda *a: float((norm.group_norm(a[0], 4, a[1], a[2], act="gelu", dropout=drop)[0].double() * r.double()).sum())  # noqa: E731
    gen = torch.Generator(device="cuda:0").manual_seed(5)
    leaves, step = [x, gamma, beta], 2.0 ** -6
    for k in range(3):
        v = torch.randn(leaves[k].shape, device="cuda:0", generator=gen)
        v /= v.norm()
        hi, lo = ([q + s * step * v if j == k else q for j, q in enumerate(leaves)] for s in (1, -1))
        num = (loss(*hi) - loss(*lo)) / (2 * step)
        assert abs(num - float((grads[k].double() * v.double()).sum())) < 1e-2, k


def test_offsets_past_32_bits(env):
    """More than 2^32 elements: the last ones' mask and normalisation are theirs (a 32-bit index would take the first ones')."""
    torch, norm = env
    count = (1 << 32) + (1 << 20) + 24
    x = torch.ones(count, dtype=torch.bfloat16, device="cuda:0")
    norm.dropout(x, norm.Dropout(0.5, 77, 78), out=x)
    for first in (0, (1 << 31) - 512, (1 << 32) - 512, count - 1024):
        want = no.drop_factor((1024,), 0.5, 77, 78, first)
        assert np.array_equal(_np(x[first:first + 1024]), want), first
    del x
    n, h, w, c = 3, 4731, 4733, 64                          # 4.3e9 elements, half a type's step of bf16 around 1
    x = torch.empty(n, h, w, c, dtype=torch.bfloat16, device="cuda:0")
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    block = torch.randn(1, 1, w, c, device="cuda:0", generator=gen)
    for i in range(n):
        x[i] = (block * (i + 1) + i).to(torch.bfloat16)     # every row of an image alike: its statistics are the row's
    assert x.numel() > 1 << 32
    drop = norm.Dropout(0.25, 5, 6)
    y, st = norm.group_norm(x, 4, act="none", dropout=drop, out=x)
    for i in range(n):
        row = (block * (i + 1) + i).to(torch.bfloat16).double().cpu().numpy()
        mean, rstd = no.stats(row, 4, 1e-5)
        # sums of 1.4e9 values: threads' chains of 700 batches, K E -> 1e-4 relative at the most
        assert np.abs(_np(st[0, i]) - mean[0]).max() < 1e-4 * (i + 1) and np.abs(_np(st[1, i]) / rstd[0] - 1).max() < 1e-4
        first = (i * h * w + (h - 1) * w) * c               # the image's last row
        want = (row - no.per_channel(mean, c)) * no.per_channel(rstd, c) * no.drop_factor(row.shape, 0.25, 5, 6, first)
        got = _np(y[i, h - 1])
        assert np.abs(got - want[0, 0]).max() < 2.0 ** -8 * 6 + 1e-3, i
        assert np.array_equal(got == 0, want[0, 0] == 0)


def test_c_entries_refuse_host_memory_beside_device_tensors(env):
    """Whole calls on device tensors with one parameter, parameter gradient or counter in host memory: refused by name, outputs untouched."""
    import ctypes
    from fisr_amd import lib
    torch, _ = env
    L = lib.lib()
    n, h, w, c, g = 2, 5, 6, 16, 4
    x, dy, gamma, beta = _inputs(torch, n, h, w, c, "f32", 3)
    y, st = torch.full_like(x, 7.0), torch.full((2, n, g), 7.0, device="cuda:0")
    dg, db = torch.full_like(gamma, 7.0), torch.full_like(gamma, 7.0)
    need = L.fisr_train_groupnorm_workspace_bytes(n, h, w, c, g, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda:0")
    host = torch.ones(64)
    stream = torch.cuda.current_stream().cuda_stream
    dev = dict(gamma=gamma, beta=beta, dgamma=dg, dbeta=db, mean_rstd=st)
    for name in (*dev, "d_counter"):
        p = {k: (host if k == name else v).data_ptr() for k, v in dev.items()}
        drop = ctypes.byref(lib.DropoutDesc(0.5, 1, 2, host.data_ptr() if name == "d_counter" else None))
        if name not in ("dgamma", "dbeta"):
            assert L.fisr_train_groupnorm(x.data_ptr(), c, p["gamma"], p["beta"], y.data_ptr(), c, p["mean_rstd"], n, h, w, c, g, 1e-5, 0, drop, 0, ws.data_ptr(),
                                          need, stream) == -1
            assert f"{name} is not memory of a GPU" in L.fisr_last_error(None).decode()
        assert L.fisr_train_groupnorm_bwd(x.data_ptr(), c, dy.data_ptr(), c, p["gamma"], p["beta"], p["mean_rstd"], y.data_ptr(), c, p["dgamma"], p["dbeta"], 0, n,
                                          h, w, c, g, 0, drop, 0, ws.data_ptr(), need, stream) == -1
        assert f"{name} is not memory of a GPU" in L.fisr_last_error(None).decode()
    assert L.fisr_train_dropout(x.data_ptr(), None, y.data_ptr(), x.numel(), drop, 0, stream) == -1
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in (y, st, dg, db))


def test_given_outputs_count_as_changed_in_place(env):
    """A graph of autograd that kept a tensor which a call then writes raises in its backward pass instead of using the new values; tensors
    that are only read do not count, nor do tensors of inference mode, which have no count."""
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 2, 4, 5, 16, "f32", 9)
    drop = norm.Dropout(0.5, 1, 2)
    _, st = norm.group_norm(x, 4, gamma, beta)

    def backward(t, **kw):
        norm.group_norm_backward(dy, x, st, 4, gamma, beta, **{"dx": torch.empty_like(x), "dgamma": torch.empty_like(gamma), "dbeta": torch.empty_like(beta), **kw})

    calls = [(x, lambda t: norm.dropout(t, drop, out=t)), (x, lambda t: norm.group_norm(t, 4, gamma, beta, out=t)), (x, lambda t: backward(t, dx=t)),
             (gamma, lambda t: backward(t, dgamma=t)), (beta, lambda t: backward(t, dbeta=t)), (x, lambda t: norm.dropout_backward(dy, drop, out=t))]
    for like, call in calls:
        w = torch.ones_like(like, requires_grad=True)
        t = w * 2
        loss = (t * t).sum()
        call(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    w = torch.ones_like(x, requires_grad=True)
    t = w * 2
    loss = (t * t).sum()
    y, _ = norm.group_norm(t, 4, gamma, beta)
    assert not y.requires_grad and not norm.dropout(t, drop, residual=t).requires_grad
    loss.backward()
    assert torch.equal(w.grad, torch.full_like(w, 8.0))
    with torch.inference_mode():
        t = x * 2
        want, _ = norm.group_norm(t, 4, gamma, beta)
        assert torch.equal(norm.group_norm(t, 4, gamma, beta, out=t)[0], want)


def test_c_entries_refuse_outputs_across_other_operands(env):
    """What a call writes is apart from all else that it goes to, but where the very same tensor is allowed and beside other channels of the same
    pixels.  Refused calls launch nothing."""
    import ctypes
    from fisr_amd import lib
    torch, norm = env
    L = lib.lib()
    n, h, w, c, g = 2, 40, 50, 64, 4
    need = L.fisr_train_groupnorm_workspace_bytes(n, h, w, c, g, 1)
    count = n * h * w * c
    buf = torch.full((16 * count,), 7.0, device="cuda:0")
    f = {"x": 0, "dy": 2 * count, "y": 4 * count, "gamma": 8 * count, "beta": 8 * count + c, "dgamma": 8 * count + 2 * c, "dbeta": 8 * count + 3 * c,
         "st": 8 * count + 4 * c, "counter": 8 * count + 5 * c, "ws": 9 * count}
    assert 16 < need <= 4 * 7 * count
    buf[f["counter"]:f["counter"] + 2] = 0
    stream = torch.cuda.current_stream().cuda_stream

    def call(backward, cs=None, **at):
        p = {k: buf.data_ptr() + 4 * v for k, v in {**f, **at}.items()}
        cs = {"x": c, "dy": c, "y": c, **(cs or {})}
        drop = ctypes.byref(lib.DropoutDesc(0.5, 1, 2, p["counter"]))
        if backward:
            rc = L.fisr_train_groupnorm_bwd(p["x"], cs["x"], p["dy"], cs["dy"], p["gamma"], p["beta"], p["st"], p["y"], cs["y"], p["dgamma"], p["dbeta"], 0, n, h, w, c,
                                            g, 0, drop, 0, p["ws"], need, stream)
        else:
            rc = L.fisr_train_groupnorm(p["x"], cs["x"], p["gamma"], p["beta"], p["y"], cs["y"], p["st"], n, h, w, c, g, 1e-5, 0, drop, 0, p["ws"], need, stream)
        return rc, L.fisr_last_error(None).decode()

    small = 2 * c                                           # pixels 2 c apart: room for another tensor's channels
    for backward, what, kw in [
            (False, "y overlaps x", dict(y=4)), (False, "y overlaps x", dict(y=count - 4)), (False, "y overlaps gamma", dict(gamma=4 * count + 8)),
            (False, "y overlaps beta", dict(beta=5 * count - 4)), (False, "mean_rstd overlaps x", dict(st=8)), (False, "mean_rstd overlaps gamma", dict(st=8 * count)),
            (False, "d_counter", dict(counter=4 * count)), (False, "the workspace overlaps x", dict(ws=count - 4)), (False, "the workspace overlaps y", dict(ws=4 * count)),
            (False, "y overlaps x", dict(y=c - 4, cs=dict(x=small, y=small))), (False, "y overlaps x", dict(y=0, cs=dict(x=small))),
            (True, "dx overlaps x", dict(y=4)), (True, "dx overlaps dy", dict(y=2 * count + 4)), (True, "dgamma overlaps gamma", dict(dgamma=8 * count)),
            (True, "dgamma overlaps dbeta", dict(dbeta=8 * count + 2 * c)), (True, "dgamma overlaps dbeta", dict(dbeta=8 * count + c + 4)),
            (True, "mean_rstd", dict(dgamma=8 * count + 4 * c)), (True, "dgamma overlaps x", dict(dgamma=4)), (True, "the workspace overlaps dx", dict(ws=5 * count - 4)),
            (True, "overlaps the workspace", dict(ws=8 * count - 4))]:
        rc, said = call(backward, **kw)
        assert rc == -1 and what in said, (what, kw, rc, said)
    d = ctypes.byref(lib.DropoutDesc(0.5, 1, 2, None))
    at = buf.data_ptr()
    for res, y, what in ((None, 4, "y overlaps x"), (8 * count, 8 * count - 4, "y overlaps residual"), (8 * count, 4 * (count - 1), "y overlaps x")):
        assert L.fisr_train_dropout(at, None if res is None else at + res, at + y, count, d, 0, stream) == -1 and what in L.fisr_last_error(None).decode()
    torch.cuda.synchronize()
    untouched = buf.clone()
    untouched[f["counter"]:f["counter"] + 2] = 7.0
    assert (untouched == 7).all()
    # allowed: in place, other channels of the same pixels, neighbours without a gap
    for backward, kw in [(False, dict(y=0)), (False, dict(y=c, cs=dict(x=small, y=small))), (False, dict(y=count)), (True, dict(y=0)), (True, dict(y=2 * count)),
                         (True, dict(y=3 * count)), (True, dict(dy=c, cs=dict(x=small, dy=small)))]:
        rc, said = call(backward, **kw)
        assert rc == 0, (kw, said)
    torch.cuda.synchronize()
    x, dy, gamma, beta = _inputs(torch, 1, 4, 4, 16, "f32", 1)
    _, st = norm.group_norm(x, 4, gamma, beta)
    with pytest.raises(lib.FisrError, match="dgamma overlaps gamma"):
        norm.group_norm_backward(dy, x, st, 4, gamma, beta, dgamma=gamma)


def test_the_most_groups_with_wide_joins(env):
    """n * groups = 2^22, the limit, in groups of more channels than a join of 256 threads is meant for: a launch of 1024 threads a group would be
    2^32, one more than a grid holds.  One pixel an image, all images alike but the last.  A group is 4097 values: bounds as above with K for 4096 values in
    float64 joins of single values (no chain of float32 sums: E each), so y is off by a few E before it is rounded."""
    torch, norm = env
    torch.cuda.empty_cache()
    n, c, groups = 1 << 20, 16388, 4
    if torch.cuda.mem_get_info()[0] < 185 << 30:
        pytest.skip("needs 185 GB of device memory")
    r = np.random.default_rng(1)
    rows = r.standard_normal((2, c)) * (0.5 + r.random(c)) + 0.5
    rows = _to(torch, rows, "bf16")
    x = rows[0].expand(n, 1, 1, c).contiguous()
    x[-1, 0, 0] = rows[1]
    _, st = norm.group_norm(x, groups, out=x)
    for i, row in ((0, 0), (1, 0), (n // 2, 0), (n - 2, 0), (n - 1, 1)):
        want, mean, rstd, _, _ = no.forward(_np(rows[row]).reshape(1, 1, 1, c), groups, 1.0, 0.0, 1e-5, "none")
        assert np.abs(_np(st[0, i]) - mean[0]).max() <= 4 * E and np.abs(_np(st[1, i]) / rstd[0] - 1).max() <= 8 * E
        _within(_np(x[i, 0, 0]), want[0, 0, 0], 2.0 ** -8 * np.abs(want[0, 0, 0]) + 16 * E * (1 + np.abs(want[0, 0, 0])), i)
    assert (st[:, :-1] == st[:, :1]).all()
    del x, st
    torch.cuda.empty_cache()


def test_an_unaligned_call_leaves_the_aligned_ones_as_they_were(env):
    """3 x 3 pixels of 1024 float16 channels in one group: one launch and no workspace where vectors of 16 bytes are possible, several launches from an
    address that allows none.  After such a call the aligned one still allocates y and the statistics alone."""
    torch, norm = env
    x, _, gamma, beta = _inputs(torch, 2, 3, 3, 1024, "f16", 6)
    odd = torch.empty(x.numel() + 8, dtype=x.dtype, device="cuda:0")[1:1 + x.numel()].view(x.shape)
    odd.copy_(x)

    def allocations(t):
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        kept = norm.group_norm(t, 1, gamma, beta)
        return torch.cuda.memory_stats()["allocation.all.allocated"] - before, kept

    allocations(x)
    allocations(odd)
    assert allocations(odd)[0] == 3 and allocations(x)[0] == 2


# ---- what full-size calls take: float64 on the GPU, an image at a time, with the bounds of the first docstring ----
def _act64(torch, z, act):
    """act'(z) and the bound on its curvature."""
    if act == "silu":
        sg = torch.sigmoid(z)
        return sg * (1 + z * (1 - sg)), 1.0
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327, 1.0
    return torch.ones_like(z), 0.0


def _check_backward(torch, x, dy, mask, stats, got, groups, gamma, beta, act, t, k, slices=1):
    """dx, dgamma, dbeta of group_norm_backward(dy, x, stats ...); mask: what multiplies dy.  k: a thread's chain and the joins (K of the first
    docstring).  Images are worked on in `slices` ranges of pixels."""
    dx, dg, db = got
    n, c = x.shape[0], x.shape[3]
    p, d = x[0].numel() // c, c // groups
    g, b = gamma.double(), beta.double()
    bounds = list(range(0, p, (p + slices - 1) // slices)) + [p]
    parts = [slice(lo, hi) for lo, hi in zip(bounds, bounds[1:])]
    sums = torch.zeros(4, c, dtype=torch.float64, device=x.device)              # dgamma, its bound, dbeta, its bound
    chan = lambda v: v.repeat_interleave(d)  # noqa: E731
    for i in range(n):
        xi, dyi, mi, dxi = (v[i].view(p, c) for v in (x, dy, mask, dx))
        far = max(float(xi[q].abs().max()) for q in parts)
        mean = sum(xi[q].double().sum(0) for q in parts).view(groups, d).sum(1) / (p * d)
        var = sum(((xi[q].double() - chan(mean)) ** 2).sum(0) for q in parts).view(groups, d).sum(1) / (p * d)
        rstd = 1 / torch.sqrt(var + 1e-5)
        emean, erstd = torch.full_like(mean, k * E * far), (k + 2 * far * rstd) * E
        assert ((stats[0, i].double() - mean).abs() <= emean + E * mean.abs()).all() and ((stats[1, i].double() - rstd).abs() <= (erstd + E) * rstd).all()
        mean, rstd, emean, erstd = map(chan, (mean, rstd, emean, erstd))

        def terms(q):
            xh = (xi[q].double() - mean) * rstd
            exh = rstd * emean + xh.abs() * (erstd + 4 * E)
            z = xh * g + b
            ez = g.abs() * exh + E * z.abs()
            slope, curve = _act64(torch, z, act)
            dyq = dyi[q].double() * mi[q].double()
            dz = dyq * slope
            edz = dyq.abs() * (curve * ez + 1e-6)
            ta = edz + k * E * dz.abs()
            return xh, exh, dz, edz, ta, ta * xh.abs() + dz.abs() * exh

        acc = torch.zeros(6, c, dtype=torch.float64, device=x.device)           # sums of dz, dz xh, their terms' bounds, |dz|, |dz xh|
        for q in parts:
            xh, exh, dz, edz, ta, tb = terms(q)
            acc += torch.stack([v.sum(0) for v in (dz, dz * xh, ta, tb, dz.abs(), (dz * xh).abs())])
            del xh, exh, dz, edz, ta, tb
        sums += torch.stack((acc[1], acc[3], acc[0], acc[2]))
        grp = lambda v, w: chan((v * w).view(groups, d).sum(1) / (p * d))  # noqa: E731
        s1, s2 = grp(acc[0], g), grp(acc[1], g)
        ga, gb, m1, m2 = (grp(v, g.abs()) for v in acc[2:])
        for q in parts:
            xh, exh, dz, edz, _, _ = terms(q)
            want = rstd * (dz * g - s1 - xh * s2)
            bound = rstd * (g.abs() * (edz + 8 * E * dz.abs()) + ga + xh.abs() * gb + exh * m2 + 8 * E * (m1 + xh.abs() * m2)) + HALF[t] * want.abs() + TINY[t]
            bound += erstd * (want.abs() + rstd * (g.abs() * dz.abs() + m1 + xh.abs() * m2))
            off = (dxi[q].double() - want).abs() - bound
            assert float(off.max()) <= 0, (i, q, float(off.max()))
            del xh, exh, dz, edz, want, bound, off
    assert ((dg.double() - sums[0]).abs() <= sums[1] + E * sums[0].abs()).all()
    assert ((db.double() - sums[2]).abs() <= sums[3] + E * sums[2].abs()).all()


def _large(torch, n, h, w, c, t, seed):
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda:0")  # noqa: E731
    x, dy = (torch.empty(n, h, w, c, dtype=_type(torch, t), device="cuda:0") for _ in range(2))
    scale, shift = 0.5 + normal(c).abs().clamp(max=1), 0.5 + normal(c)
    for i in range(n):
        x[i] = (normal(h, w, c) * scale + shift).to(x.dtype)
        dy[i] = normal(h, w, c).to(x.dtype)
    return x, dy, 1 + 0.2 * normal(c), 0.2 * normal(c)


@pytest.mark.parametrize("t,n,h,w,c,groups,act,p", [
    ("bf16", 4, 544, 992, 64, 8, "silu", 0.1),               # 552 MB of x and dy: reads past the caches, pieces by size
    ("f32", 2, 544, 992, 64, 16, "gelu", 0.25),              # the same in float32, where a generator block is two threads' work
    ("f16", 1, 544, 992, 128, 32, "gelu", 0.0),              # 276 MB, one image: the join between the launches
    ("f32", 32, 116, 116, 64, 8, "none", 0.1),               # 220 MB: pieces by size, through the caches
    ("bf16", 5, 400, 300, 72, 9, "silu", 0.1),               # 173 MB: 1536 pieces
])
def test_large_backward(env, t, n, h, w, c, groups, act, p):
    """Chains: at most 132 values a thread, 256 a join."""
    torch, norm = env
    x, dy, gamma, beta = _large(torch, n, h, w, c, t, 7)
    drop = norm.Dropout(p, 91, 1 << 35)
    mask = norm.dropout(torch.ones(x.shape, device="cuda:0"), drop)
    _, st = norm.group_norm(x, groups, gamma, beta, act=act, dropout=drop)
    got = norm.group_norm_backward(dy, x, st, groups, gamma, beta, act=act, dropout=drop)
    _check_backward(torch, x, dy, mask, st, got, groups, gamma, beta, act, t, K + 132)


def test_backward_past_32_bits(env):
    """4.3e9 elements, dx in dy's place.  A thread's chain in the sums is 131762 pixels of a chunk / 32 rows = 4118; K follows it."""
    torch, norm = env
    torch.cuda.empty_cache()
    n, h, w, c, groups = 3, 4731, 4733, 64, 4
    x, dy, gamma, beta = _large(torch, n, h, w, c, "bf16", 8)
    assert x.numel() > 1 << 32
    drop = norm.Dropout(0.25, 5, 6)
    mask = norm.dropout(torch.ones_like(x), drop)             # 4 / 3 in bfloat16: 1.3359, a factor of its own
    for first in (0, (1 << 32) - 512, x.numel() - 1024):
        want = no.drop_factor((1024,), 0.25, 5, 6, first)
        assert np.array_equal(_np(mask.view(-1)[first:first + 1024]) > 0, want > 0)
    _, st = norm.group_norm(x, groups, gamma, beta, act="silu", dropout=drop)
    dx = dy.clone()
    got = norm.group_norm_backward(dx, x, st, groups, gamma, beta, act="silu", dropout=drop, dx=dx)
    mask.clamp_(max=1.0)
    dy_scaled = 65536 / (65536 - 16384)
    _check_backward(torch, x, dy, _Times(mask, dy_scaled), st, got, groups, gamma, beta, "silu", "bf16", 4118 + K, slices=8)
    del x, dy, mask, dx, got
    torch.cuda.empty_cache()


class _Times:
    """A mask of ones and zeros times a factor that its type does not hold."""

    def __init__(self, mask, factor):
        self.mask, self.factor = mask, factor

    def __getitem__(self, i):
        return _Times(self.mask[i], self.factor)

    def view(self, *shape):
        return _Times(self.mask.view(*shape), self.factor)

    def double(self):
        return self.mask.double() * self.factor


@pytest.mark.parametrize("t,count", [("f32", 22000003), ("f16", 44000005), ("bf16", 44000000)])
def test_large_dropout_with_residual(env, t, count):
    """More than 160 MB of reads, which go past the caches; the tail of the odd counts too."""
    torch, norm = env
    gen = torch.Generator(device="cuda:0").manual_seed(4)
    x, res = (torch.randn(count, generator=gen, device="cuda:0").to(_type(torch, t)) for _ in range(2))
    fac = torch.from_numpy(no.drop_factor((count,), 0.3, 61, 62)).cuda()
    got = norm.dropout(x, norm.Dropout(0.3, 61, 62), residual=res)
    kept = x.double() * fac
    want = kept + res.double()
    assert ((got.double() - want).abs() <= HALF[t] * want.abs() + 3 * E * (want.abs() + kept.abs()) + TINY[t]).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_pixels_far_apart(env, t):
    """Channels of a buffer whose pixels are 3 M elements apart: a thread's offsets would pass 32 bits in the one-launch form, and in float32 in the
    two-launch form too.  Against the dense call, as in test_channel_ranges_of_wider_buffers; a float32 mean goes by K E."""
    torch, norm = env
    x, dy, gamma, beta = _inputs(torch, 2, 2, 3, 24, t, 14)
    wide, dwide, ywide, gwide = (torch.full((2, 2, 3, 3 << 20), 7.0, dtype=x.dtype, device="cuda:0") for _ in range(4))
    lo, hi = (3 << 20) - 40, (3 << 20) - 16
    wide[..., lo:hi], dwide[..., lo:hi] = x, dy
    drop = norm.Dropout(0.3, 5, 6)
    y0, st0 = norm.group_norm(x, 2, gamma, beta, act="gelu", dropout=drop)
    d0 = norm.group_norm_backward(dy, x, st0, 2, gamma, beta, act="gelu", dropout=drop)
    tol = 3 * HALF[t]
    y1, st1 = norm.group_norm(wide[..., lo:hi], 2, gamma, beta, act="gelu", dropout=drop, out=ywide[..., lo:hi])
    d1 = norm.group_norm_backward(dwide[..., lo:hi], wide[..., lo:hi], st1, 2, gamma, beta, act="gelu", dropout=drop, dx=gwide[..., lo:hi])
    assert torch.allclose(st0, st1, rtol=K * E, atol=K * E) and torch.allclose(y0.double(), y1.double(), rtol=tol, atol=1e-4)
    assert torch.allclose(d0[0].double(), d1[0].double(), rtol=tol, atol=1e-3)
    assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-4) for a, b in zip(d0[1:], d1[1:]))
    for v in (ywide, gwide):
        assert (v[..., :lo] == 7).all() and (v[..., hi:] == 7).all()
