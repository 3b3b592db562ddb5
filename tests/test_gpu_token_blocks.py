"""A token model's block (xdna_train.tokens: layer norm, linear layer, decay attention) against plain
64-bit implementations on the CPU, at the sizes, lengths and strides where they can go wrong.

Tolerances, per element.  u = 2^-24 (half an fp32 ulp at 1), b = 2^-8 (half a bf16 ulp at 1, the one
rounding of a bf16 result); each function's docstring derives its own:
* layer norm: norm_reference;  * linear layer: linear_reference;  * decay attention: walk.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def T(hip):
    from xdna_train import tokens
    return tokens


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rounding(dtype):
    return B if dtype == BF16 else U


def close(got, ref, tol, what):
    got = got.detach().cpu().to(F64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got == ref) | ((got - ref).abs() <= tol))
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4], tol[bad][:4] if torch.is_tensor(tol) else tol)


def padded(t, extra, offset=0):
    """t's values in a larger allocation of NaN: rows `extra` elements apart, `offset` elements in."""
    rows, n = t.shape
    buf = torch.full((rows * (n + extra) + offset + 8,), math.nan, dtype=t.dtype, device="xdna")
    v = torch.as_strided(buf, (rows, n), (n + extra, 1), offset)
    v.copy_(t)
    return v


def same(a, b):
    """equal bits (the tests' values hold no NaN)"""
    return torch.equal(a.detach().cpu(), b.detach().cpu())


# ---- layer norm --------------------------------------------------------------------------------

def norm_reference(x, w, b, dy, ds, eps, dtype, ptype):
    """{name: (value, tolerance)} for the stored rows x.

    A row's sum goes through at most 40 terms a thread, 6 steps in a wave and 16 waves: 64 u of the sum of
    magnitudes.  That is the mean's error; the deviations' squares add up within 66 u, and a mean that is off
    by e adds (e / deviation)^2 to the variance; a square root and a reciprocal within 3 u: the inverse
    deviation is off by 40 u of itself and half of that square.  h is off by (64 u mean|x| + u |x - m|) / deviation and
    the inverse's error.  The gradients' sums over rows go through at most 128 terms in any order."""
    x, w, b, dy, ds = (None if t is None else t.to(F64) for t in (x, w, b, dy, ds))
    r, p = rounding(dtype), rounding(ptype)
    one = torch.ones(x.shape[1], dtype=F64)
    wv, bv = one if w is None else w, 0 * one if b is None else b
    m = x.mean(1, keepdim=True)
    d = x - m
    inv = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    h = d * inv
    em = 64 * U * x.abs().mean(1, keepdim=True)
    ei = 40 * U + (em * inv) ** 2 / 2
    eh = inv * (em + U * d.abs()) + (ei + 2 * U) * h.abs()
    y = h * wv + bv
    ey = eh * wv.abs() + 4 * U * ((h * wv).abs() + bv.abs()) + r * y.abs()
    out = {"y": (y, ey)}
    if dy is not None:
        g = dy * wv
        mg, mh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
        emg = 66 * U * g.abs().mean(1, keepdim=True)
        emh = 67 * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * eh).mean(1, keepdim=True)
        core = g - mg - h * mh
        dx = inv * core
        edx = inv * (4 * U * (g.abs() + mg.abs() + (h * mh).abs()) + emg + eh * mh.abs() + (h.abs() + eh) * emh) + (ei + 2 * U) * dx.abs()
        if ds is not None:
            dx = dx + ds
            edx = edx + 2 * U * (dx.abs() + ds.abs())
        out["dx"] = (dx, edx + r * dx.abs())
        dw, db = (dy * h).sum(0), dy.sum(0)
        out["dw"] = (dw, (dy.abs() * eh).sum(0) + 130 * U * (dy * h).abs().sum(0) + p * dw.abs())
        out["db"] = (db, 130 * U * dy.abs().sum(0) + p * db.abs())
    return {k: (v, e + 1e-30) for k, (v, e) in out.items()}


NORM = [  # rows, width
    (1, 1), (1, 2), (3, 7), (2, 8), (5, 9), (1, 511), (4, 512), (9, 513), (33, 515), (7, 1000), (3, 1024), (6, 1025), (700, 1160), (2, 2047), (5, 2048),
    (3, 2049), (2, 4096), (3, 4099), (2, 8192), (2, 8193), (2, 16384), (2, 16385), (3, 20011), (4200, 64), (9000, 24),
]


@pytest.mark.parametrize("types", [(BF16, BF16), (BF16, F32), (F32, F32)], ids=["bf16", "bf16-f32", "f32"])
@pytest.mark.parametrize("add", [False, True], ids=["norm", "add"])
@pytest.mark.parametrize("R,D", NORM)
def test_layer_norm(T, R, D, add, types):
    print("layer norm", R, D, add, types, flush=True)
    dtype, ptype = types
    g = gen(R * 7 + D)
    x = (torch.randn(R, D, generator=g) + torch.randn(R, 1, generator=g)).to(dtype)
    r = torch.randn(R, D, generator=g).to(dtype) if add else None
    w, b = (1 + 0.2 * torch.randn(D, generator=g)).to(ptype), torch.randn(D, generator=g).to(ptype)
    dy, ds = torch.randn(R, D, generator=g).to(dtype), torch.randn(R, D, generator=g).to(dtype) if add else None
    leaves = [t.to("xdna").requires_grad_() for t in (x, r, w, b) if t is not None]
    if add:
        y, s = T.add_layer_norm(*leaves)
        stored = (x.float() + r.float()).to(dtype)
        assert same(s, stored)
        grads = torch.autograd.grad([y, s], leaves, [dy.to("xdna"), ds.to("xdna")])
        assert same(grads[0], grads[1])
        grads = grads[1:]
    else:
        y, stored = T.layer_norm(*leaves), x
        grads = torch.autograd.grad(y, leaves, dy.to("xdna"))
    ref = norm_reference(stored, w, b, dy, ds, 1e-5, dtype, ptype)
    for got, name in zip((y, *grads), ("y", "dx", "dw", "db")):
        close(got, *ref[name], name)
    with torch.no_grad():  # without a gradient: the same bits
        again = T.add_layer_norm(*leaves) if add else (T.layer_norm(*leaves),)
    assert same(again[0], y)
    if add:  # the fused form is the norm of the stored sum
        assert same(T.layer_norm(s.detach(), *[t.detach() for t in leaves[2:]]), y)


@pytest.mark.parametrize("D", [5, 515, 520, 3001])
def test_layer_norm_strides_and_absent_parameters(T, D):
    print("layer norm strides", D, flush=True)
    g = gen(D)
    x, r, dy = (torch.randn(11, D, generator=g).to(BF16) for _ in range(3))
    w = torch.randn(D, generator=g)
    xx, rx, dyx = padded(x, 3, 1).requires_grad_(), padded(r, 5, 3).requires_grad_(), padded(dy, 1, 5)
    y, s = T.add_layer_norm(xx, rx)
    ref = norm_reference((x.float() + r.float()).to(BF16), None, None, dy, None, 1e-5, BF16, BF16)
    close(y, *ref["y"], "without parameters")
    (dx,) = torch.autograd.grad(y, [xx], dyx, retain_graph=True)
    close(dx, *ref["dx"], "dx of the norm alone")
    dr, = torch.autograd.grad(s, [rx], dyx)
    assert same(dr, dy)  # the sum alone has no norm's gradient
    wx = w.to("xdna").requires_grad_()
    y = T.layer_norm(xx.detach(), wx, eps=1e-3)
    ref = norm_reference(x, w, None, dy, None, 1e-3, BF16, F32)
    close(y, *ref["y"], "weight alone")
    close(torch.autograd.grad(y, [wx], dyx)[0], *ref["dw"], "dw without dx")
    y3 = T.layer_norm(xx.detach().view(1, 11, D), wx.detach(), eps=1e-3)
    assert y3.shape == (1, 11, D) and same(y3[0], y)
    t = torch.randn(D, 11, generator=g).to(BF16)
    assert same(T.layer_norm(t.to("xdna").t()), T.layer_norm(t.t().contiguous().to("xdna")))


def test_layer_norm_of_no_rows_and_broadcast_gradients(T):
    w, b = torch.ones(9, device="xdna").requires_grad_(), torch.zeros(9, device="xdna").requires_grad_()
    x = torch.zeros(0, 9, device="xdna").requires_grad_()
    y = T.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 9, device="xdna"))
    assert y.shape == (0, 9) and grads[0].shape == (0, 9) and not grads[1].cpu().any() and not grads[2].cpu().any()
    x = torch.randn(4, 9, generator=gen(3))
    xx = x.to("xdna").requires_grad_()
    (dx, dw) = torch.autograd.grad(T.layer_norm(xx, w, b).sum(), [xx, w])  # a gradient of stride 0
    ref = norm_reference(x, torch.ones(9), torch.zeros(9), torch.ones(4, 9), None, 1e-5, F32, F32)
    close(dx, *ref["dx"], "dx")
    close(dw, *ref["dw"], "dw")


def test_layer_norm_of_special_rows(T):
    """A constant row is exact zeros (and the bias); a row of an infinity or NaN is NaN and touches no other;
    a row of large values with a small spread keeps it (two passes)."""
    x = torch.zeros(6, 64)
    x[0] = 3.0
    x[1] = torch.randn(64, generator=gen(1))
    x[1, 5] = math.inf
    x[2] = math.nan
    x[3] = 4096 + torch.randn(64, generator=gen(2))
    x[4] = torch.randn(64, generator=gen(3))
    x[5] = 1e-30 * torch.randn(64, generator=gen(4))
    y = T.layer_norm(x.to("xdna"), None, torch.full((64,), 0.5, device="xdna")).cpu()
    assert (y[0] == 0.5).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    ref = norm_reference(x[3:], None, torch.full((64,), 0.5), None, None, 1e-5, F32, F32)["y"]
    close(y[3:], *ref, "rows beside them")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [7, 64, 515, 1000, 1160, 2047, 3000, 10000, 20011])
def test_layer_norm_of_constant_rows(T, D, dtype):
    """A constant row is zeros before the bias, whatever 1 / width rounds to, and gives the weight no gradient.  The mean is
    off by n = 66 u of itself at most before it is corrected by the deviations' own mean, which is as exact of them: what is left
    is (66 u)^2 of the row's value, over sqrt(eps)."""
    print("layer norm of constant rows", D, dtype, flush=True)
    at = torch.tensor([3.0, 1000.0, 1e6, -0.1, 1000.1, 0.0])[:, None].to(dtype)
    x, dy = at.expand(6, D).contiguous(), torch.ones(6, D).to(dtype)
    lv = [t.to("xdna").requires_grad_() for t in (x, torch.ones(D, dtype=dtype))]
    y = T.layer_norm(*lv, torch.full((D,), 0.5, dtype=dtype, device="xdna"))
    left = (66 * U) ** 2 * at.to(F64).abs() / math.sqrt(1e-5)
    close(y, torch.full((6, D), 0.5, dtype=F64), (left + rounding(dtype)).expand(6, D), "y")
    dx, dw = torch.autograd.grad(y, lv, dy.to("xdna"))
    close(dw, torch.zeros(D, dtype=F64), float(left.sum()) + 1e-30, "dw")
    # dx = inv (1 - mean(1) - h mean(h)): the mean of ones is within 66 u of one
    close(dx, torch.zeros(6, D, dtype=F64), ((66 * U + left * left) / math.sqrt(1e-5)).expand(6, D), "dx")


@pytest.mark.parametrize("at,spread", [(1000.0, 0.01), (-1e4, 1.0), (1e6, 30.0)])
@pytest.mark.parametrize("D", [7, 515, 1000, 2047, 3000, 10000, 20011])
def test_layer_norm_of_rows_far_from_zero(T, D, at, spread):
    """fp32 rows whose spread is small against their mean.  x - mean is exact (within a factor of two); the correction leaves
    it off by e = 66 u (mean |x - m| + 66 u |m|).  The squares' mean less the correction's square is off by 68 u of both, and
    e adds its square.  The gradient takes the mean as it is kept, rounded: half an ulp, 2 u of it, more."""
    print("layer norm far from zero", D, at, spread, flush=True)
    g = gen(D)
    x = (at + spread * torch.randn(4, D, generator=g)).to(F32)
    dy = torch.randn(4, D, generator=g)
    lv = [t.to("xdna").requires_grad_() for t in (x, torch.ones(D))]
    y = T.layer_norm(*lv)
    dx, dw = torch.autograd.grad(y, lv, dy.to("xdna"))
    m, dy = x.to(F64).mean(1, keepdim=True), dy.to(F64)
    d = x.to(F64) - m
    inv = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    h = d * inv
    first = 66 * U * m.abs()
    e = 66 * U * (d.abs().mean(1, keepdim=True) + first)
    ei = 40 * U + 68 * U * (first * inv) ** 2 + (e * inv) ** 2
    close(y, h, inv * (e + U * d.abs()) + (ei + 4 * U) * h.abs() + 1e-30, "y")
    eh = inv * (e + 2 * U * m.abs() + U * d.abs()) + (ei + 2 * U) * h.abs()
    mg, mh = dy.mean(1, keepdim=True), (dy * h).mean(1, keepdim=True)
    emg, emh = 66 * U * dy.abs().mean(1, keepdim=True), 67 * U * (dy * h).abs().mean(1, keepdim=True) + (dy.abs() * eh).mean(1, keepdim=True)
    want = inv * (dy - mg - h * mh)
    close(dx, want, inv * (4 * U * (dy.abs() + mg.abs() + (h * mh).abs()) + emg + eh * mh.abs() + (h.abs() + eh) * emh) + (ei + 4 * U) * want.abs(), "dx")
    close(dw, (dy * h).sum(0), (dy.abs() * eh).sum(0) + 6 * U * (dy * h).abs().sum(0) + 1e-30, "dw")


@pytest.mark.parametrize("add", [False, True], ids=["norm", "add"])
@pytest.mark.parametrize("D", [(1 << 22) + 5, 1 << 24])
def test_layer_norm_of_the_longest_rows(T, D, add):
    """Squares and gradients that are alike: a thread's plain sum of 4096 or 16384 of them would round most additions the same
    way.  The tolerance is that of every other row (norm_reference)."""
    print("layer norm of the longest rows", D, add, flush=True)
    g = gen(D)
    x = torch.where(torch.rand(1, D, generator=g) < 0.5, 0.7, -0.7)
    r, dy = torch.full((1, D), 0.125), torch.full((1, D), 0.7)
    leaves = [t.to("xdna").requires_grad_() for t in ((x, r) if add else (x,))]
    y, stored = (T.add_layer_norm(*leaves).norm, x + r) if add else (T.layer_norm(*leaves), x)
    (dx,) = torch.autograd.grad(y, leaves[:1], dy.to("xdna"))
    ref = norm_reference(stored, None, None, dy, None, 1e-5, F32, F32)
    close(y, *ref["y"], "y")
    close(dx, *ref["dx"], "dx")


MANY = [  # rows, width: more rows than the backward's launch has places for, in each of its forms
    (9001, 1160), (4200, 2047), (600, 2049), (1100, 4099), (1030, 8192), (520, 16384), (130, 16400),
]


@pytest.mark.parametrize("types,add", [((BF16, BF16), True), ((BF16, F32), False), ((F32, F32), True)], ids=["bf16-add", "bf16-f32-norm", "f32-add"])
@pytest.mark.parametrize("R,D", MANY)
def test_layer_norm_of_several_rows_a_place(T, R, D, types, add):
    """A wave or workgroup that takes one row after another: rows loaded ahead, sums in LDS in turn, the parameters' sums
    over rows."""
    test_layer_norm(T, R, D, add, types)


@pytest.mark.parametrize("R,D", [(263001, 64), (65537 + 400, 2050), (65537 + 400, 9000), (65537 + 400, 16392)])
def test_layer_norm_of_more_rows_than_a_launch(T, R, D):
    """Rows past the grid's bound: those of the second turn have the bits of a small call."""
    print("layer norm of many rows", R, D, flush=True)
    part = torch.randn(331, D, generator=gen(D)).to(BF16).to("xdna")
    with torch.no_grad():
        y = T.layer_norm(part.repeat(R // 331 + 1, 1)[:R])
        one = T.layer_norm(part).cpu()
    for r0 in (0, R // 331 // 2 * 331, (R // 331 - 1) * 331):
        assert same(y[r0:r0 + 331], one), r0


def test_layer_norm_gradient_against_differences(T):
    g = gen(11)
    x, w, dy = torch.randn(3, 40, generator=g), 1 + 0.1 * torch.randn(40, generator=g), torch.randn(3, 40, generator=g)

    def f(x, w):
        d = x.to(F64) - x.to(F64).mean(1, keepdim=True)
        return (d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * w.to(F64) * dy.to(F64)).sum()

    xx, wx = x.to("xdna").requires_grad_(), w.to("xdna").requires_grad_()
    dx, dw = (t.cpu().to(F64) for t in torch.autograd.grad(T.layer_norm(xx, wx), [xx, wx], dy.to("xdna")))
    for i in range(5):
        vx, vw = torch.randn(3, 40, generator=g).to(F64), torch.randn(40, generator=g).to(F64)
        e = 1e-5
        slope = (f(x.to(F64) + e * vx, w.to(F64) + e * vw) - f(x.to(F64) - e * vx, w.to(F64) - e * vw)) / (2 * e)
        assert abs(slope - ((dx * vx).sum() + (dw * vw).sum())) <= 1e-4 * (1 + abs(slope))


# ---- linear layer --------------------------------------------------------------------------------

def act64(act, g):
    if act == "none":
        return g, torch.ones_like(g)
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).to(F64)


def linear_reference(x, w, b, r, dy, act):
    """{name: (value, tolerance)}.  A fp32 sum of n products is off by (n + 8) u of the sum of magnitudes;
    act' is at most 1.13 and act'' at most 0.8 in size; the slope is kept within 2^-12 of itself (fp16
    times 2^15: 2^-40 where that is subnormal), and for relu it is another one where the sum's sign is in doubt."""
    x, w, b, r, dy = (None if t is None else t.to(F64) for t in (x, w, b, r, dy))
    K, (M, N) = x.shape[1], (x.shape[0], w.shape[0])
    v, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        v, mag = v + b, mag + b.abs()
    ev = (K + 8) * U * mag
    y, s = act64(act, v)
    ey = 1.13 * ev + (0 if act == "none" else 16 * U * (y.abs() + v.abs()))
    if r is not None:
        y = y + r
        ey = ey + U * (y.abs() + r.abs())
    out = {"y": (y, ey + B * y.abs())}
    if dy is not None:
        if act == "none":
            es = 0 * s
        else:
            es = (torch.where(v.abs() <= 2 * ev, 1.0, 0.0) if act == "relu" else 0.8 * ev + 32 * U * (1 + v.abs())) + 2.0 ** -12 * s.abs() + 2.0 ** -40
        p = dy * s
        ep = dy.abs() * es + 2 * U * p.abs()
        stored = ep + (0 if act == "none" else B) * p.abs()
        dx, dw, db = p @ w, p.t() @ x, p.sum(0)
        out["dx"] = (dx, (stored + (N + 8) * U * p.abs()) @ w.abs() + B * dx.abs())
        out["dw"] = (dw, (stored + (M + 8) * U * p.abs()).t() @ x.abs() + B * dw.abs())
        out["db"] = (db, (ep + (M + 8) * U * p.abs()).sum(0) + B * db.abs())
    return {k: (t, e + 1e-30) for k, (t, e) in out.items()}


LINEAR = [  # rows, K, N
    (1, 1, 1), (1, 64, 32), (1, 2048, 300), (1, 4096, 64), (2, 7, 5), (4, 3000, 100), (5, 72, 100), (16, 256, 128), (17, 130, 63), (33, 8, 65),
    (64, 64, 64), (65, 65, 129), (130, 512, 384), (333, 1000, 217), (200, 4000, 65), (70, 3, 4), (100, 5000, 3),
]


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear(T, M, K, N, act):
    print("linear", M, K, N, act, flush=True)
    g = gen(M + K + N)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    b = torch.randn(N, generator=g).to(BF16) if (M + N) % 3 else None
    r = torch.randn(M, N, generator=g).to(BF16) if M % 2 else None
    dy = torch.randn(M, N, generator=g).to(BF16)
    given = {"x": x, "w": w, "b": b, "r": r}
    lv = {n: t.to("xdna").requires_grad_() for n, t in given.items() if t is not None}
    y = T.linear(lv["x"], lv["w"], lv.get("b"), act, lv.get("r"))
    ref = linear_reference(x, w, b, r, dy, act)
    close(y, *ref["y"], "y")
    grads = dict(zip(lv, torch.autograd.grad(y, list(lv.values()), dy.to("xdna"))))
    close(grads["x"], *ref["dx"], "dx")
    close(grads["w"], *ref["dw"], "dw")
    if b is not None:
        close(grads["b"], *ref["db"], "db")
    if r is not None:
        assert same(grads["r"], dy)
    with torch.no_grad():
        assert same(T.linear(lv["x"], lv["w"], lv.get("b"), act, lv.get("r")), y)


@pytest.mark.parametrize("M,K,N,act", [(4096, 264, 4096, "relu"), (4100, 512, 4096, "silu"), (2048, 1024, 2056, "none"), (600, 8192, 512, "gelu"),
                                       (8200, 128, 3080, "gelu")])
def test_linear_large(T, M, K, N, act):
    """The 256 x 256 tiles, k in splits, gradients on the GEMM: rows of the result checked at random."""
    print("linear large", M, K, N, act, flush=True)
    g = gen(M)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    b, r, dy = torch.randn(N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16)
    lv = [t.to("xdna").requires_grad_() for t in (x, w, b)]
    y = T.linear(*lv, act, r.to("xdna"))
    dx, dw, db = torch.autograd.grad(y, lv, dy.to("xdna"))
    ref = linear_reference(x, w, b, r, dy, act)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        close(got, *ref[name], name)


@pytest.mark.parametrize("M,K,N,act", [(8192, 72, 3001, "relu"), (8200, 64, 3002, "silu"), (8192, 136, 4093, "relu"), (8193, 64, 4093, "gelu"), (8192, 64, 3002, "relu"),
                                       (8192, 72, 3001, "none"), (8192, 64, 4099, "gelu")])
def test_linear_large_of_odd_units(T, M, K, N, act):
    """256 x 256 tiles whose units are no whole vectors: outputs, slopes and ReLU's rows of bits at odd places, parts of
    vectors at the rows' ends, bias and residual at any alignment."""
    print("linear large, odd units", M, K, N, act, flush=True)
    tiles = -(-M // 256) * -(-N // 256)
    assert tiles >= 256 and 100 * tiles >= 65 * 256 * -(-tiles // 256) and K % 8 == 0
    g = gen(M + N)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    b, r, dy = torch.randn(N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16)
    bx = padded(b[None], 0, 3)[0]
    lv = [x.to("xdna").requires_grad_(), w.to("xdna").requires_grad_(), bx.requires_grad_()]
    ref = linear_reference(x, w, b, r, dy, act)
    y = T.linear(*lv, act, padded(r, 4, 5))
    for got, name in zip((y, *torch.autograd.grad(y, lv, padded(dy, 1, 1))), ("y", "dx", "dw", "db")):
        close(got, *ref[name], name)
    with torch.no_grad():
        assert same(T.linear(*lv, act, padded(r, 0, 1)), y)


@pytest.mark.parametrize("M,K,N,off,how", [(8191, 520, 1032, 0, 2), (5056, 1024, 448, 0, 2), (5056, 1024, 448, 8, 2), (5056, 1024, 448, 1, 0),
                                           (2500, 2048, 2048, 0, 1), (6001, 768, 1536, 0, 2), (6001, 1024, 1536, 0, 2)])
def test_linear_gradients_in_one_launch_of_large_tiles(T, hip, M, K, N, off, how):
    """Both products' 256 x 256 tiles together, whole or with either's k in splits; operands that are slices (``off``),
    of which those off the 16-byte grid go elsewhere."""
    print("linear large gradients", M, K, N, off, flush=True)
    g = gen(M + off)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    dy = torch.randn(M, N, generator=g).to(BF16)
    cut = lambda t: torch.nn.functional.pad(t, (off, 8)).to("xdna")[:, off:off + t.shape[1]] if off else t.to("xdna")  # noqa: E731
    lv = [cut(x).detach().requires_grad_(), cut(w).detach().requires_grad_()]
    d = cut(dy)
    assert (hip.xdna_linear_grads_pick(d.data_ptr(), d.stride(0), lv[0].data_ptr(), lv[0].stride(0), lv[1].data_ptr(), lv[1].stride(0), M, K, N) == 2) == (how == 2)
    dx, dw = torch.autograd.grad(T.linear(*lv), lv, d)
    ref = linear_reference(x, w, None, None, dy, "none")
    close(dx, *ref["dx"], "dx")
    close(dw, *ref["dw"], "dw")
    again = torch.autograd.grad(T.linear(*lv), lv, d)
    assert same(again[0], dx) and same(again[1], dw)


@pytest.mark.parametrize("M,K,N", [(3, 40, 24), (70, 129, 65), (700, 264, 512)])
def test_linear_strides_and_parts_of_the_gradient(T, M, K, N):
    print("linear strides", M, K, N, flush=True)
    g = gen(M)
    x, w, r, dy = (torch.randn(*s, generator=g).to(BF16) for s in ((M, K), (N, K), (M, N), (M, N)))
    b = torch.randn(2 * N, generator=g).to(BF16).to("xdna")[::2]
    ref = linear_reference(x, w, b.cpu(), r, dy, "gelu")
    xx, wx, rx, dyx = padded(x, 3, 1), padded(w, 5, 3), padded(r, 1, 1), padded(dy, 7, 5)
    for wanted in ((0,), (1,), (2,), (0, 1), (1, 2), (3,), (0, 1, 2, 3)):
        lv = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((xx, wx, b, rx))]
        y = T.linear(lv[0], lv[1], lv[2], "gelu", lv[3])
        close(y, *ref["y"], "y")
        for i, got in zip(wanted, torch.autograd.grad(y, [lv[i] for i in wanted], dyx)):
            if i == 3:
                assert same(got, dy)
            else:
                close(got, *ref[("dx", "dw", "db")[i]], i)
    y3 = T.linear(xx.unsqueeze(0), wx, b, "gelu", rx.unsqueeze(0))
    assert y3.shape == (1, M, N) and same(y3[0], y)
    assert same(T.linear(x.t().contiguous().to("xdna").t(), wx, b, "gelu", rx), y)
    one = torch.ones(1, N, device="xdna", dtype=BF16).expand(M, N)  # stride 0
    lv = [xx.detach().requires_grad_(), wx.detach()]
    ref = linear_reference(x, w, None, torch.ones(M, N).to(BF16), torch.ones(M, N).to(BF16), "silu")
    y = T.linear(*lv, None, "silu", one)
    close(y, *ref["y"], "broadcast residual")
    close(torch.autograd.grad(y, [lv[0]], one)[0], *ref["dx"], "broadcast gradient")


def test_linear_without_rows(T):
    x, w, b = torch.zeros(0, 8, device="xdna", dtype=BF16), torch.ones(5, 8, device="xdna", dtype=BF16), torch.ones(5, device="xdna", dtype=BF16)
    lv = [t.requires_grad_() for t in (x, w, b)]
    for act in ("none", "silu"):
        y = T.linear(*lv, act)
        dx, dw, db = torch.autograd.grad(y, lv, torch.zeros(0, 5, device="xdna", dtype=BF16))
        assert y.shape == (0, 5) and dx.shape == (0, 8) and not dw.cpu().any() and not db.cpu().any()


def test_linear_slopes_keep_the_lower_tail(T):
    """A unit far in an activation's tail still has a gradient: the kept slope's relative error is 2^-12 down
    to 1.9e-9."""
    M, K = 32, 16
    for act, at in (("silu", -12.0), ("gelu", -5.0), ("silu", -19.0)):
        x = torch.zeros(M, K)
        x[:, 0] = at
        x[:, 1] = 1.0
        w, dy = torch.zeros(1, K), torch.ones(M, 1)
        w[0, 0] = 1.0
        lv = [t.to(BF16).to("xdna").requires_grad_() for t in (x, w)]
        dx, dw = torch.autograd.grad(T.linear(*lv, None, act), lv, dy.to(BF16).to("xdna"))
        s = float(act64(act, torch.tensor(at, dtype=F64))[1])
        assert abs(float(dx[0, 0]) - s) <= (2 * B + 2.0 ** -10) * abs(s), (act, at, float(dx[0, 0]), s)
        assert abs(float(dw[0, 1]) - M * s) <= (2 * B + 2.0 ** -10) * abs(M * s)


@pytest.mark.parametrize("M,K,N", [(3, 8, 24), (70, 129, 65), (700, 264, 512), (8192, 72, 3001)])
def test_linear_relu_selects_its_gradient(T, M, K, N):
    """As torch.relu's: a unit that is off has gradient 0 whatever comes in, infinities and NaN too, and a unit whose sum is
    NaN passes it.  Whole numbers: every sum is exact, the results are the reference's roundings."""
    print("linear relu selects", M, K, N, flush=True)
    g = gen(M)
    x, w = torch.zeros(M, K), torch.zeros(N, K)
    x[:, 0], w[:, 0] = torch.where(torch.rand(M, generator=g) < 0.5, 1.0, -1.0), 1.0
    x[0, 0], x[1, 0], x[M - 1, 0] = 1.0, -1.0, math.nan
    on = ~(x[:, :1] <= 0)
    dy = torch.randint(-8, 9, (M, N), generator=g).float()
    p = torch.where(on, dy, 0.0)
    bad = torch.tensor([math.inf, -math.inf, math.nan])[torch.randint(0, 3, (M, N), generator=g)]
    dy = torch.where(~on & (torch.rand(M, N, generator=g) < 0.5), bad, dy)
    assert not dy.isfinite().all()
    lv = [t.to(BF16).to("xdna").requires_grad_() for t in (x, w, torch.zeros(N))]
    y = T.linear(*lv, "relu")
    assert (y[:-1].cpu() == on[:-1]).all() and y[-1].cpu().isnan().all()
    dx, dw, db = (t.cpu() for t in torch.autograd.grad(y, lv, dy.to(BF16).to("xdna")))
    assert torch.equal(db, p.sum(0).to(BF16))
    assert torch.equal(dx, (p @ w).to(BF16))
    assert not dw[:, 1:].any() and dw[:, 0].isnan().all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,N", [(2, 1, 700), (4, 5, 453)])
def test_linear_bias_gradient_that_cancels(T, M, K, N, act):
    """Few rows whose terms of d_bias nearly cancel: what is left shows the kept slopes' rounding, half a step of fp16: 2^-11 of a
    slope.  Beside it the sum's error times act'' (at most 0.8), the activation's own arithmetic (32 u) and the sums over rows."""
    print("linear bias gradient that cancels", M, K, N, act, flush=True)
    g = gen(M * K * N)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(BF16)
    b = torch.randn(N, generator=g).to(BF16)
    v = x.to(F64) @ w.to(F64).t() + b.to(F64)
    ev = (K + 8) * U * (x.to(F64).abs() @ w.to(F64).abs().t() + b.to(F64).abs())
    s = act64(act, v)[1]
    dy = torch.ones(M, N)
    dy[-1] = -(s[:-1].sum(0) / s[-1]).clamp(-8, 8)  # the last row takes the others' terms away
    dy = dy.to(BF16)
    bx = b.to("xdna").requires_grad_()
    (db,) = torch.autograd.grad(T.linear(x.to("xdna"), w.to("xdna"), bx, act), [bx], dy.to("xdna"))
    p = dy.to(F64) * s
    ep = dy.to(F64).abs() * (0.8 * ev + 32 * U * (1 + v.abs()) + 2.0 ** -11 * s.abs() + 2.0 ** -40) + 2 * U * p.abs()
    want = p.sum(0)
    close(db, want, (ep + (M + 8) * U * p.abs()).sum(0) + B * want.abs(), "db")


def test_linear_gradient_against_differences(T):
    g = gen(5)
    x, w, b, dy = (torch.randn(*s, generator=g).to(BF16) for s in ((6, 24), (10, 24), (10,), (6, 10)))
    w = (w.float() / 5).to(BF16)
    for act in ("silu", "gelu"):
        def f(x, w, b):
            return (act64(act, x @ w.t() + b)[0] * dy.to(F64)).sum()

        lv = [t.to("xdna").requires_grad_() for t in (x, w, b)]
        grads = [t.cpu().to(F64) for t in torch.autograd.grad(T.linear(*lv, act), lv, dy.to("xdna"))]
        base = [t.to(F64) for t in (x, w, b)]
        for _ in range(5):
            vs = [torch.randn(t.shape, generator=g).to(F64) for t in base]
            e = 1e-5
            slope = (f(*[t + e * v for t, v in zip(base, vs)]) - f(*[t - e * v for t, v in zip(base, vs)])) / (2 * e)
            mine = sum((d * v).sum() for d, v in zip(grads, vs))
            mag = sum((d * v).abs().sum() for d, v in zip(grads, vs))
            assert abs(slope - mine) <= 2 * B * mag, (act, slope, mine)


# ---- decay attention -------------------------------------------------------------------------------

CHUNK = 64


def walk(q, k, v, g, s0, lead, p, qs, ks):
    """One head's walk in 64 bits: ((outputs, tolerance), (last state, tolerance)) without the outputs' own
    rounding.  Weights are exp of a product: (2 |exponent| + 4) u, under 200 u of the largest that counts.  fp32 sums
    over n tokens, 128 of a head and the carries: (n + 640) u of the sum of magnitudes.  The weighted scores of a
    chunk and the state before it, as operands, are rounded to bf16 (b each); the state's own sum has its
    weighted v in two bf16: 2^-16."""
    n, u = q.shape[0], (q.shape[0] + 640) * U
    at = torch.arange(n, dtype=F64)
    apart = at[:, None] - at
    weight = torch.where(apart >= 0, torch.exp(apart * g), 0.0) if g > -math.inf else (apart == 0).to(F64)
    power = (lambda e: torch.exp(e * g)) if g > -math.inf else (lambda e: (e == 0).to(F64))
    P = (q @ k.t()) * weight * p
    mag = (q.abs() @ k.abs().t()) * weight * abs(p)
    inner = (at[:, None] // CHUNK) == (at // CHUNK)
    out = P @ v
    tol = u * (mag @ v.abs()) + B * ((P * inner).abs() @ v.abs()) + 2.0 ** -16 * (mag @ v.abs())
    first = power(at + lead)[:, None]
    out = out + qs * first * (q @ s0)
    tol = tol + u * abs(qs) * first * (q.abs() @ s0.abs())
    # the states before the chunks, for what their rounding costs
    s, c0 = s0, 0
    for c0 in range(0, n, CHUNK):
        m = min(CHUNK, n - c0)
        local = power(torch.arange(m, dtype=F64) + lead)[:, None]
        tol[c0:c0 + m] += B * abs(qs) * local * (q[c0:c0 + m].abs() @ s.abs())
        w = power(m - lead - torch.arange(m, dtype=F64))[:, None] * ks
        s = power(torch.tensor(float(m), dtype=F64)) * s + (k[c0:c0 + m] * w).t() @ v[c0:c0 + m]
    w = power(n - lead - at)[:, None] * abs(ks)
    es = (u + 2.0 ** -16) * ((k.abs() * w).t() @ v.abs() + power(torch.tensor(float(n), dtype=F64)) * s0.abs())
    return (out, tol), (s, es)


def decay_reference(q, k, v, g, s0, lengths, scale, dout=None, ds=None):
    """{name: (value, tolerance)} of every output and gradient."""
    q, k, v, g = (t.to(F64) for t in (q, k, v, g))
    Bn, Tn, H, dk = q.shape
    G, dv = k.shape[2], v.shape[3]
    zeros = lambda *s: (torch.zeros(*s, dtype=F64), torch.zeros(*s, dtype=F64))  # noqa: E731
    out, last = zeros(Bn, Tn, H, dv), zeros(Bn, H, dk, dv)
    dq, dkk, dvv, d0 = zeros(Bn, Tn, H, dk), zeros(Bn, Tn, G, dk), zeros(Bn, Tn, G, dv), zeros(Bn, H, dk, dv)
    for b in range(Bn):
        n = Tn if lengths is None else max(0, min(Tn, int(lengths[b])))
        for h in range(H):
            j = h // (H // G)
            qh, kh, vh = q[b, :n, h], k[b, :n, j], v[b, :n, j]
            s = torch.zeros(dk, dv, dtype=F64) if s0 is None else s0[b, h].to(F64)
            o, e = walk(qh, kh, vh, g[h], s, 1, scale, scale, 1.0)
            for at in (0, 1):
                out[at][b, :n, h], last[at][b, h] = o[at], e[at]
            if dout is None:
                continue
            do = dout[b, :n, h].to(F64)
            r = torch.zeros(dk, dv, dtype=F64) if ds is None else ds[b, h].to(F64)
            o, _ = walk(do, vh, kh, g[h], s.t(), 1, scale, scale, 1.0)
            rev = lambda t: t.flip(0)  # noqa: E731
            ov, e0 = walk(rev(kh), rev(qh), rev(do), g[h], r, 0, scale, 1.0, scale)
            ok, _ = walk(rev(vh), rev(do), rev(qh), g[h], r.t(), 0, scale, 1.0, scale)
            for at in (0, 1):
                dq[at][b, :n, h] = o[at]
                dvv[at][b, :n, j] += rev(ov[at])
                dkk[at][b, :n, j] += rev(ok[at])
                d0[at][b, h] = e0[at]
    ref = {"out": out, "state": last}
    if dout is not None:
        ref |= {"dq": dq, "dk": dkk, "dv": dvv, "dstate": d0}
    return {n: (t, e + (B * t.abs() if "state" not in n else 2 * U * t.abs()) + 1e-30) for n, (t, e) in ref.items()}


def decay_values(Bn, Tn, H, G, dk, dv, seed, state=True):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    v = {"q": r(Bn, Tn, H, dk).to(BF16), "k": r(Bn, Tn, G, dk).to(BF16), "v": r(Bn, Tn, G, dv).to(BF16),
         "g": -torch.exp2(-0.5 - 8.0 * torch.arange(H) / H), "dout": r(Bn, Tn, H, dv).to(BF16)}
    v["state"], v["dstate"] = (2 * r(Bn, H, dk, dv), r(Bn, H, dk, dv)) if state else (None, None)
    return v


def run_decay(T, v, lengths=None, scale=None, grads=True):
    """Outputs and gradients by name."""
    names = [n for n in ("q", "k", "v", "state") if v[n] is not None]
    lv = {n: (v[n] if v[n].device.type == "xdna" else v[n].to("xdna")).detach().requires_grad_(grads) for n in names}
    r = T.decay_attention(lv["q"], lv["k"], lv["v"], v["g"].to("xdna"), lv.get("state"), None if lengths is None else lengths.to("xdna"), scale)
    got = {"out": r.out, "state": r.state}
    if grads:
        ends = [(r.out, v["dout"])] + ([(r.state, v["dstate"])] if v["dstate"] is not None else [])
        d = torch.autograd.grad([e for e, _ in ends], list(lv.values()), [x.to("xdna") for _, x in ends])
        got |= {"d" + n: t for n, t in zip(names, d)}
    return got


def check_decay(got, ref):
    for n, t in got.items():
        close(t, *ref[n], n)


DECAY = [  # batch, tokens, heads, kv heads, dk, dv
    (1, 1, 1, 1, 1, 1), (1, 2, 1, 1, 8, 8), (2, 5, 2, 1, 16, 16), (1, 16, 1, 1, 64, 64), (1, 31, 2, 2, 64, 64), (2, 32, 1, 1, 33, 65), (1, 33, 3, 1, 64, 128),
    (1, 64, 1, 1, 128, 64), (1, 100, 2, 1, 7, 3), (1, 65, 1, 1, 64, 8), (1, 95, 1, 1, 32, 64), (1, 97, 2, 1, 128, 32), (1, 127, 2, 2, 128, 128), (2, 128, 1, 1, 100, 72), (1, 129, 2, 2, 48, 80), (1, 256, 1, 1, 128, 128),
    (1, 300, 4, 2, 64, 64), (2, 391, 2, 1, 72, 127), (1, 777, 6, 2, 48, 80),
]


@pytest.mark.parametrize("state", [True, False], ids=["state", "new"])
@pytest.mark.parametrize("size", DECAY)
def test_decay_attention(T, size, state):
    print("decay", size, state, flush=True)
    v = decay_values(*size, seed=sum(size), state=state)
    scale = 0.37 if size[1] % 2 else None
    got = run_decay(T, v, scale=scale)
    check_decay(got, decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, scale or size[4] ** -0.5, v["dout"], v["dstate"]))
    again = run_decay(T, v, scale=scale)
    assert all(same(got[n], again[n]) for n in got), "equal inputs, different bits"


@pytest.mark.parametrize("size", [(7, 300, 2, 1, 64, 64), (6, 200, 3, 3, 40, 100), (7, 700, 1, 1, 128, 128)])
@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=["int64", "int32"])
def test_decay_attention_of_ragged_batches(T, size, kind):
    """Lengths of zero, one, a chunk and its neighbours, past the tensor and below zero; what lies behind a
    sequence's end is NaN."""
    print("decay ragged", size, kind, flush=True)
    Bn, Tn = size[:2]
    lengths = torch.tensor([0, 1, 64, 129, Tn - 1, Tn + 5, -3][:Bn], dtype=kind)
    v = decay_values(*size, seed=5)
    ref = decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], lengths, 0.2, v["dout"], v["dstate"])
    for b in range(Bn):
        n = max(0, min(Tn, int(lengths[b])))
        for name in ("q", "k", "v", "dout"):
            v[name][b, n:] = math.nan
    got = run_decay(T, v, lengths, 0.2)
    check_decay(got, ref)
    for name in ("out", "dq", "dk", "dv"):
        for b in range(Bn):
            assert not got[name][b, max(0, min(Tn, int(lengths[b]))):].cpu().any(), (name, b)


def segments(hip, size, backward):
    """Segments of a sequence, from the workspace that holds all but one of their states."""
    Bn, Tn, H, G, dk, dv = size
    state = 4 * Bn * H * dk * dv
    if not backward:
        return 1 + hip.xdna_decay_workspace_bytes(Bn, Tn, H, dk, dv) // state
    shared = 4 * Bn * Tn * H * (dk + dv) if G < H else 0
    return 1 + (hip.xdna_decay_bwd_workspace_bytes(Bn, Tn, H, G, dk, dv) - shared) // (2 * state)


SEGMENTED = [  # size, segments of the forward's and the backward's sequences: whole, few (read one by one) or many (summed first)
    ((1, 1500, 1, 1, 64, 64), "many", "many"), ((2, 1100, 20, 20, 128, 128), "few", "whole"), ((1, 1300, 20, 20, 72, 72), "many", "few"),
    ((1, 2500, 30, 15, 16, 128), "many", "many"), ((2, 2000, 9, 3, 128, 24), "many", "many"), ((3, 777, 6, 2, 48, 80), "many", "whole"),
    ((1, 1000, 22, 11, 16, 128), "many", "few"),
]


@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("size,forward,backward", SEGMENTED)
def test_decay_attention_in_segments(T, hip, size, forward, backward, ragged):
    n = [segments(hip, size, b) for b in (False, True)]
    print("decay segments", size, ragged, n, flush=True)
    assert [("whole" if x == 1 else "few" if x < 5 else "many") for x in n] == [forward, backward], n
    v = decay_values(*size, seed=7)
    lengths = torch.tensor([300, size[1] - 1, 65][: size[0]]) if ragged else None
    got = run_decay(T, v, lengths)
    check_decay(got, decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], lengths, size[4] ** -0.5, v["dout"], v["dstate"]))


@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("size", [(1, 1500, 2, 1, 33, 65), (2, 1300, 5, 5, 100, 71), (1, 1100, 6, 3, 127, 5), (2, 900, 3, 3, 6, 126), (1, 2000, 14, 14, 90, 66)])
def test_decay_attention_of_odd_heads_in_segments(T, hip, size, ragged):
    """Rows that are no whole vectors, shorter than one, or whose last block of columns is."""
    n = [segments(hip, size, b) for b in (False, True)]
    print("decay odd segments", size, ragged, n, flush=True)
    assert max(n) > 1, n
    v = decay_values(*size, seed=17)
    lengths = torch.tensor([700, 65][: size[0]]) if ragged else None
    ref = decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], lengths, size[4] ** -0.5, v["dout"], v["dstate"])
    for b in range(size[0] if ragged else 0):
        for name in ("q", "k", "v", "dout"):
            v[name][b, int(lengths[b]):] = math.nan
    check_decay(run_decay(T, v, lengths), ref)


def test_decay_attention_of_many_heads_in_one_walk(T):
    """As many workgroups as the chip takes: no segments, several chunks each."""
    size = (1, 400, 260, 260, 9, 70)
    v = decay_values(*size, seed=8)
    check_decay(run_decay(T, v), decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, size[4] ** -0.5, v["dout"], v["dstate"]))


def test_decay_attention_of_a_large_batch(T):
    """2000 sequences, more rounds of workgroups than the chip holds at once: the bits of its parts' calls."""
    Bn, Tn, H, dk, dv = 2000, 100, 4, 48, 44
    g = gen(4)
    part = {n: torch.randn(100, Tn, H, d, generator=g).to(BF16).to("xdna") for n, d in (("q", dk), ("k", dk), ("v", dv), ("dout", dv))}
    log_decay = torch.tensor([-0.5, -0.1, -0.02, -0.004], device="xdna")

    def run(v):
        lv = [v[n].requires_grad_() for n in ("q", "k", "v")]
        r = T.decay_attention(*lv, log_decay)
        return [r.out.detach(), r.state.detach(), *torch.autograd.grad(r.out, lv, v["dout"])]

    one = [t.cpu() for t in run({n: t.clone() for n, t in part.items()})]
    whole = run({n: t.repeat(Bn // 100, 1, 1, 1) for n, t in part.items()})
    for i, (a, b) in enumerate(zip(whole, one)):
        for j in (0, 1, 10, Bn // 100 - 1):
            assert same(a[100 * j:100 * j + 100], b), (i, j)


def test_decay_attention_at_the_ends_of_the_decays(T):
    """Nothing forgotten (0), everything (-inf), and decays that underflow within a chunk."""
    v = decay_values(2, 200, 4, 4, 16, 24, seed=9)
    v["g"] = torch.tensor([0.0, -math.inf, -30.0, -3.0])
    check_decay(run_decay(T, v), decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, 0.25, v["dout"], v["dstate"]))
    got = T.decay_attention(*[v[n].to("xdna") for n in ("q", "k", "v", "g")], scale=-0.25)
    close(got.out, *decay_reference(v["q"], v["k"], v["v"], v["g"], None, None, -0.25)["out"], "negative scale")
    got = T.decay_attention(*[v[n].to("xdna") for n in ("q", "k", "v", "g")], scale=0.0)
    assert not got.out.cpu().any()


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_decay_attention_of_a_token_that_is_not_finite(T, name, bad):
    """Its own and all later outputs are not finite; of the earlier ones at most 63 are not, and the others keep their bits.  So do
    the other heads and sequences."""
    size = (2, 300, 3, 3, 32, 40)
    v = decay_values(*size, seed=3)
    v["g"] = torch.tensor([-0.01, -0.1, -0.02])
    call = lambda: T.decay_attention(*[v[n].to("xdna") for n in ("q", "k", "v", "g", "state")]).out.cpu()  # noqa: E731
    clean = call()
    v[name][1, 200, 1] = bad
    got = call()
    assert not got[1, 200:, 1].isfinite().any()
    got[1, 137:, 1] = clean[1, 137:, 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_decay_gradients_of_a_token_that_is_not_finite(T, name, bad):
    """k and v go forwards (out and dq of their own and the later tokens), q and out's gradient backwards (dk and dv of their
    own and the earlier ones, and the first state's): those are not finite, and of the tokens on the other side at most 63.  What
    a token's own row alone enters is bad there alone, and everything else keeps its bits."""
    size, s = (2, 300, 3, 3, 32, 40), 170
    v = decay_values(*size, seed=3)
    v["g"] = torch.tensor([-0.01, -0.1, -0.02])
    call = lambda: {n: t.detach().cpu() for n, t in run_decay(T, v).items()}  # noqa: E731
    clean = call()
    v[name][1, s, 1] = bad
    got = call()
    forwards, backwards = (slice(s, None), slice(s - 63, None)), (slice(None, s + 1), slice(None, s + 64))
    own = (slice(s, s + 1), slice(s, s + 1))
    reach = {"q": {"out": own, "dk": backwards, "dv": backwards}, "k": {"out": forwards, "dq": forwards, "dv": own},
             "v": {"out": forwards, "dq": forwards, "dk": own}, "dout": {"dq": own, "dk": backwards, "dv": backwards}}[name]
    for n, (must, may) in reach.items():
        assert not got[n][1, must, 1].isfinite().any(), n
        got[n][1, may, 1] = clean[n][1, may, 1]
    for n in (["state"] if name in "kv" else ["dstate"]):
        assert not got[n][1, 1].isfinite().any(), n
        got[n][1, 1] = clean[n][1, 1]
    for n in got:
        assert torch.equal(got[n], clean[n]), n


@pytest.mark.parametrize("size", [(1, 2, 3, 3, 64, 64), (2, 5, 3, 1, 128, 128), (1, 64, 3, 3, 33, 70), (1, 1000, 3, 3, 128, 64)])
def test_decay_attention_keeps_states_in_24_bits(T, size):
    """The weighted v of the state's sum has 24 bits.  Each sequence has one token that counts, so that every element of the
    state is one product: exp(g n) is off by (2 |g n| + 2) u, its product with v by u, the three parts' sum by 4 u, and what
    carries it to the end by 2 u a chunk: 16 u with |g n| at most 1 and two chunks.  (Parts of 16 bits would be off by up to 128
    u, over 16 u in half of the elements.)  The gradient's sum for the state is the same walk."""
    print("decay state's bits", size, flush=True)
    Bn, Tn, H, G, dk, dv = size
    v = decay_values(*size, seed=40)
    v["g"] = -torch.tensor([0.05, 0.3, 0.9])
    counts = max(0, Tn - 2)  # the forward's: a token before the last
    far = torch.arange(Tn) != counts
    kk, state = v["k"].clone(), torch.zeros(Bn, H, dk, dv)
    kk[:, far] = 0.0
    leaf = state.to("xdna").requires_grad_()
    r = T.decay_attention(v["q"].to("xdna"), kk.to("xdna"), v["v"].to("xdna"), v["g"].to("xdna"), leaf, scale=1.0)
    heads = lambda t: t.to(F64).repeat_interleave(H // t.shape[1], 1)  # noqa: E731
    a = torch.exp(v["g"].to(F64) * (Tn - 1 - counts))[:, None, None]
    want = a * heads(kk[:, counts])[..., :, None] * heads(v["v"][:, counts])[..., None, :]
    close(r.state, want, 16 * U * want.abs() + 1e-30, "state")
    dout = v["dout"].clone()
    dout[:, 1:] = 0.0  # the backward's: the first token, decayed once
    (d,) = torch.autograd.grad(r.out, [leaf], dout.to("xdna"))
    want = torch.exp(v["g"].to(F64))[:, None, None] * v["q"][:, 0].to(F64)[..., :, None] * dout[:, 0].to(F64)[..., None, :]
    close(d, want, 16 * U * want.abs() + 1e-30, "dstate")


@pytest.mark.parametrize("size", [(1, 1, 2, 2, 32, 32), (3, 2, 4, 4, 128, 128), (2, 4, 2, 1, 32, 32), (1, 20, 2, 2, 7, 3), (3, 22, 1, 1, 32, 64), (1, 40, 2, 2, 100, 72),
                                  (2, 64, 3, 3, 128, 128)])
def test_decay_attention_keeps_scores_in_16_bits(T, size):
    """A chunk alone, without a state before it: nothing but the weighted scores is rounded before the result, and they have
    two bf16: 2^-18 of each.  (One rounding to 8 bits, b, put sequences of a few tokens 1.8 times as far off as the result's own.)"""
    print("decay score's bits", size, flush=True)
    Bn, Tn, H, G, dk, dv = size
    v = decay_values(*size, seed=50, state=False)
    got = run_decay(T, v, scale=0.4)
    want = {n: (torch.zeros(v[m].shape, dtype=F64), torch.zeros(v[m].shape, dtype=F64)) for n, m in (("out", "dout"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    zero, rev, u = torch.zeros(dk, dv, dtype=F64), lambda t: t.flip(0), (Tn + 640) * U + 2.0 ** -18
    for b in range(Bn):
        for h in range(H):
            j = h // (H // G)
            qh, kh, vh, do = (v[n][b, :, i].to(F64) for n, i in (("q", h), ("k", j), ("v", j), ("dout", h)))
            for n, (x, y, z), s, i, turn in (("out", (qh, kh, vh), zero, h, False), ("dq", (do, vh, kh), zero.t(), h, False), ("dv", (kh, qh, do), zero, j, True),
                                             ("dk", (vh, do, qh), zero.t(), j, True)):
                x, y, z = (rev(t) if turn else t for t in (x, y, z))
                (o, _), _ = walk(x, y, z, v["g"][h].to(F64), s, 0 if turn else 1, 0.4, 0.4, 1.0)
                (mag, _), _ = walk(x.abs(), y.abs(), z.abs(), v["g"][h].to(F64), s, 0 if turn else 1, 0.4, 0.4, 1.0)
                want[n][0][b, :, i] += rev(o) if turn else o
                want[n][1][b, :, i] += u * (rev(mag) if turn else mag)
    for n, (o, e) in want.items():
        close(got[n], o, e + B * o.abs() + 1e-30, n)


def test_decay_attention_of_slices_and_broadcast_heads(T):
    Bn, Tn, H, G, dk, dv = 2, 150, 4, 2, 24, 40
    v = decay_values(Bn, Tn, H, G, dk, dv, seed=10)
    ref = decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, dk ** -0.5, v["dout"], v["dstate"])
    qkv = torch.cat([v["q"].flatten(2), v["k"].flatten(2), v["v"].flatten(2)], 2).to("xdna")
    parts = torch.split(qkv, [H * dk, G * dk, G * dv], 2)
    cut = dict(v, q=parts[0].view(Bn, Tn, H, dk), k=parts[1].view(Bn, Tn, G, dk), v=parts[2].view(Bn, Tn, G, dv))
    check_decay(run_decay(T, cut), ref)
    heads_first = dict(v, **{n: v[n].transpose(1, 2).contiguous().to("xdna").transpose(1, 2) for n in ("q", "k", "v", "dout")})
    heads_first["dout"] = heads_first["dout"].to("xdna")
    check_decay(run_decay(T, heads_first), ref)
    size_first = dict(v, q=v["q"].permute(3, 0, 1, 2).contiguous().to("xdna").permute(1, 2, 3, 0))  # a copy is made
    check_decay(run_decay(T, size_first), ref)
    # one head of k and v for all, as a broadcast: the gradient of the one is the sum
    one_k, one_v = v["k"][:, :, :1], v["v"][:, :, :1]
    kx, vx = one_k.to("xdna").requires_grad_(), one_v.to("xdna").requires_grad_()
    r = T.decay_attention(v["q"].to("xdna"), kx.expand(-1, -1, H, -1), vx.expand(-1, -1, H, -1), v["g"].to("xdna"))
    ref = decay_reference(v["q"], one_k, one_v, v["g"], None, None, dk ** -0.5, v["dout"])
    close(r.out, *ref["out"], "broadcast")
    dkx, dvx = torch.autograd.grad(r.out, [kx, vx], v["dout"].to("xdna"))
    for got, (t, e), single in ((dkx, ref["dk"], v["k"]), (dvx, ref["dv"], v["v"])):
        close(got, t, 2 * e, "sum of rounded gradients")  # (a head's gradient, rounded, is off by b of terms that e holds b of)


def test_decay_attention_continues_where_it_left_off(T):
    """A sequence in two parts, then token by token, against the whole."""
    Bn, Tn, H, G, dk, dv = 2, 260, 4, 2, 40, 48
    v = decay_values(Bn, Tn, H, G, dk, dv, seed=12)
    d = {n: t.to("xdna") for n, t in v.items()}
    ref = decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, 0.3)
    first = T.decay_attention(d["q"][:, :100], d["k"][:, :100], d["v"][:, :100], d["g"], d["state"], scale=0.3)
    second = T.decay_attention(d["q"][:, 100:200], d["k"][:, 100:200], d["v"][:, 100:200], d["g"], first.state, scale=0.3)
    outs, state = [first.out, second.out], second.state.clone()
    for t in range(200, Tn):
        outs.append(T.decay_attention_step(d["q"][:, t], d["k"][:, t], d["v"][:, t], d["g"], state, scale=0.3)[:, None])
    (o, eo), (s, es) = ref["out"], ref["state"]
    # (where the whole has chunks the parts have others: both within the tolerance of their own)
    q, k, w = (v[n].to(F64) for n in ("q", "k", "v"))
    at = torch.arange(Tn, dtype=F64)
    apart = (at[:, None] - at).clamp(min=0)
    for h in range(H):
        weight = torch.where(at[:, None] >= at, torch.exp(apart * v["g"][h].to(F64)), 0.0)
        for b in range(Bn):
            mag = ((q[b, :, h].abs() @ k[b, :, h // 2].abs().t()) * weight) @ w[b, :, h // 2].abs()
            mag += torch.exp((at + 1) * v["g"][h].to(F64))[:, None] * (q[b, :, h].abs() @ v["state"][b, h].to(F64).abs())
            eo[b, :, h] = 2 * B * 0.3 * mag + B * o[b, :, h].abs()
    close(torch.cat([x.cpu() for x in outs], 1), o, eo, "parts")
    close(state, s, es, "state")


@pytest.mark.parametrize("Bn,H,G,dk,dv", [(1, 1, 1, 1, 1), (1, 8, 8, 64, 64), (3, 4, 2, 33, 5), (5, 2, 1, 128, 128), (2, 3, 3, 31, 127), (4, 2, 2, 100, 36)])
def test_decay_step(T, Bn, H, G, dk, dv):
    print("decay step", Bn, H, G, dk, dv, flush=True)
    v = decay_values(Bn, 1, H, G, dk, dv, seed=Bn + dk)
    d = {n: t.to("xdna") for n, t in v.items()}
    state = d["state"].clone()
    version = state._version
    out = T.decay_attention_step(d["q"][:, 0], d["k"][:, 0], d["v"][:, 0], d["g"], state)
    assert state._version > version
    s = v["state"].to(F64) * torch.exp(v["g"].to(F64))[:, None, None]
    kh, vh = (v[n][:, 0].to(F64).repeat_interleave(H // G, 1) for n in ("k", "v"))
    add = kh[..., None] * vh[..., None, :]
    close(state, s + add, 8 * U * (s.abs() + add.abs()) + 1e-30, "state")
    o = dk ** -0.5 * (v["q"][:, 0].to(F64)[..., None] * (s + add)).sum(2)
    mag = dk ** -0.5 * (v["q"][:, 0].to(F64).abs()[..., None] * (s.abs() + add.abs())).sum(2)
    close(out, o, (dk + 16) * U * mag + B * o.abs() + 1e-30, "out")


@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=["int64", "int32"])
def test_decay_step_of_a_pool(T, kind):
    """Slots in any order; empty places, slots past the pool and slots named twice touch no state."""
    Bn, H, dk, dv, pool = 300, 2, 16, 20, 320
    v = decay_values(Bn, 1, H, H, dk, dv, seed=3)
    q, k, w = (v[n][:, 0].to("xdna") for n in ("q", "k", "v"))
    states = torch.randn(pool, H, dk, dv, generator=gen(4))
    slots = torch.randperm(pool, generator=gen(5))[:Bn].to(kind)
    slots[3], slots[50], slots[120], slots[299] = -1, pool, slots[7], slots[298]
    slots[298] = slots[0]
    pool_x = states.to("xdna")
    out = T.decay_attention_step(q, k, w, v["g"].to("xdna"), pool_x, slots.to("xdna")).cpu()
    seen, expect = set(), states.clone()
    for b in range(Bn):
        s = int(slots[b])
        if s < 0:
            assert not out[b].any()
        elif s >= pool or s in seen:
            assert torch.isnan(out[b]).all(), b
        else:
            one = states[s:s + 1].to("xdna")
            alone = T.decay_attention_step(q[b:b + 1], k[b:b + 1], w[b:b + 1], v["g"].to("xdna"), one)
            assert same(alone[0], out[b])
            expect[s] = one[0].cpu()
        seen.add(s)
    assert same(pool_x, expect)


def test_decay_attention_without_tokens_or_sequences(T):
    g, s = torch.tensor([-0.5, -0.1], device="xdna"), torch.randn(3, 2, 4, 5, device="xdna").requires_grad_()
    q, k, w = (torch.zeros(3, 0, 2, n, device="xdna", dtype=BF16).requires_grad_() for n in (4, 4, 5))
    r = T.decay_attention(q, k, w, g, s)
    assert r.out.shape == (3, 0, 2, 5) and same(r.state, s)
    (ds, dq) = torch.autograd.grad([r.out, r.state], [s, q], [torch.zeros_like(r.out), torch.ones_like(r.state)])
    assert (ds.cpu() == 1).all() and dq.shape == q.shape
    assert not T.decay_attention(q.detach(), k.detach(), w.detach(), g).state.cpu().any()
    none = T.decay_attention(*(t.detach()[:0] for t in (q, k, w)), g)
    assert none.out.shape == (0, 0, 2, 5) and none.state.shape == (0, 2, 4, 5)
    step = T.decay_attention_step(*(torch.zeros(0, 2, n, device="xdna", dtype=BF16) for n in (4, 4, 5)), g, torch.zeros(0, 2, 4, 5, device="xdna"))
    assert step.shape == (0, 2, 5)


def test_decay_gradients_of_one_result_alone(T):
    v = decay_values(1, 150, 2, 2, 24, 32, seed=21)
    lv = [v[n].to("xdna").requires_grad_() for n in ("q", "k", "v", "state")]
    r = T.decay_attention(*lv[:3], v["g"].to("xdna"), lv[3])
    grads = torch.autograd.grad(r.state, lv, v["dstate"].to("xdna"))
    ref = decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, 24 ** -0.5, 0 * v["dout"], v["dstate"])
    for got, n in zip(grads, ("dq", "dk", "dv", "dstate")):
        close(got, *ref[n], n)
    frozen = T.decay_attention(lv[0], lv[1].detach(), lv[2].detach(), v["g"].to("xdna"), lv[3].detach())
    (dq,) = torch.autograd.grad(frozen.out, [lv[0]], v["dout"].to("xdna"))
    close(dq, *decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, 24 ** -0.5, v["dout"])["dq"], "dq alone")


def test_decay_gradient_against_differences(T):
    v = decay_values(1, 140, 1, 1, 12, 10, seed=22)
    got = run_decay(T, v)
    base = {n: v[n].to(F64) for n in ("q", "k", "v", "state")}

    def f(x):  # token by token
        s, total, a = x["state"][0, 0], 0.0, math.exp(float(v["g"][0]))
        for t in range(140):
            s = a * s + x["k"][0, t, 0][:, None] * x["v"][0, t, 0]
            total = total + 12 ** -0.5 * ((x["q"][0, t, 0] @ s) * v["dout"][0, t, 0].to(F64)).sum()
        return float(total + (s * v["dstate"][0, 0].to(F64)).sum())

    g = gen(23)
    for _ in range(4):
        vs = {n: torch.randn(t.shape, generator=g).to(F64) for n, t in base.items()}
        e = 1e-4
        slope = (f({n: t + e * vs[n] for n, t in base.items()}) - f({n: t - e * vs[n] for n, t in base.items()})) / (2 * e)
        terms = [(got["d" + n].detach().cpu().to(F64) * vs[n]) for n in base]
        assert abs(slope - sum(t.sum() for t in terms)) <= 4 * B * sum(t.abs().sum() for t in terms)


def test_decay_attention_past_32_bits(T):
    """Offsets of q, k, v and of the states past 2^31 elements."""
    H, dk, dv, far = 1, 16, 16, (1 << 31) + 64
    v = decay_values(1, 2, H, H, dk, dv, seed=31)
    buf = torch.zeros(far + 1024, dtype=BF16, device="xdna")
    cut = dict(v)
    for i, n in enumerate(("q", "k", "v")):
        t = torch.as_strided(buf, (1, 2, 1, 16), (far, far, 16, 1), 256 * i)
        t.copy_(v[n])
        cut[n] = t
    check_decay(run_decay(T, cut), decay_reference(v["q"], v["k"], v["v"], v["g"], v["state"], None, 0.25, v["dout"], v["dstate"]))
    del buf, cut, t
    pool = torch.zeros((1 << 23) + 3, 1, 16, 16, dtype=F32, device="xdna")
    pool[-1] = v["state"][0].to("xdna")
    slots = torch.tensor([(1 << 23) + 2], device="xdna")
    out = T.decay_attention_step(*(v[n][:, 0].to("xdna") for n in ("q", "k", "v", )), v["g"].to("xdna"), pool, slots)
    one = v["state"].to("xdna").clone()
    assert same(out, T.decay_attention_step(*(v[n][:, 0].to("xdna") for n in ("q", "k", "v")), v["g"].to("xdna"), one))
    assert same(pool[-1], one[0])


# ---- together --------------------------------------------------------------------------------------

def block_weights(width, heads, head, seed):
    g = gen(seed)
    r = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(BF16)  # noqa: E731
    return {"n1": (1 + 0.1 * torch.randn(width, generator=g)).to(BF16), "b1": torch.zeros(width, dtype=BF16), "qkv": r(3 * heads * head, width),
            "bq": torch.zeros(3 * heads * head, dtype=BF16), "o": r(width, heads * head), "n2": torch.ones(width, dtype=BF16), "b2": torch.zeros(width, dtype=BF16),
            "w_in": r(4 * width, width), "w_out": r(width, 2 * width)}


def block(T, p, x, g, heads, head, state=None, lengths=None):
    """norm -> projection -> attention -> projection and residual -> norm -> feed-forward, and the block's residual in
    the next norm's sum."""
    Bn, Tn, _ = x.shape
    q, k, v = T.linear(T.layer_norm(x, p["n1"], p["b1"]), p["qkv"], p["bq"]).view(Bn, Tn, 3, heads, head).unbind(2)
    a = T.decay_attention(q, k, v, g, state, lengths)
    x = T.linear(a.out.reshape(Bn, Tn, heads * head), p["o"], residual=x)
    m = T.gated_mlp(T.layer_norm(x, p["n2"], p["b2"]), p["w_in"], p["w_out"])
    return T.add_layer_norm(m, x, p["n1"], p["b1"]), a.state


def block32(p, x, g, heads, head, acts=False):
    """The same in plain fp32 operations on the CPU, token by token, differentiable."""
    Bn, Tn, _ = x.shape
    norm = lambda t, w, b: (t - t.mean(-1, keepdim=True)) / torch.sqrt(t.var(-1, correction=0, keepdim=True) + 1e-5) * w + b  # noqa: E731
    q, k, v = (norm(x, p["n1"], p["b1"]) @ p["qkv"].t() + p["bq"]).view(Bn, Tn, 3, heads, head).unbind(2)
    s, outs = torch.zeros(Bn, heads, head, head), []
    for t in range(Tn):
        s = s * torch.exp(g)[:, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append(head ** -0.5 * (q[:, t, :, :, None] * s).sum(2))
    x = torch.stack(outs, 1).reshape(Bn, Tn, heads * head) @ p["o"].t() + x
    gu = norm(x, p["n2"], p["b2"]) @ p["w_in"].t()
    f = gu.shape[-1] // 2
    x = (torch.nn.functional.silu(gu[..., :f]) * gu[..., f:]) @ p["w_out"].t() + x
    return norm(x, p["n1"], p["b1"]), x, s


def test_a_block_of_them_together(T):
    """Forward and gradients of a whole block against fp32, in the 2-norm: each of the chain's 8 roundings to bf16 is
    under b of its tensor's norm and no step of the block enlarges a relative error by more than 4."""
    Bn, Tn, width, heads, head = 2, 150, 64, 4, 16
    p = block_weights(width, heads, head, 1)
    x = torch.randn(Bn, Tn, width, generator=gen(2)).to(BF16)
    g = -torch.exp2(-1.0 - torch.arange(heads).float())
    dy = torch.randn(Bn, Tn, width, generator=gen(3)).to(BF16)
    lv = {n: t.to("xdna").requires_grad_() for n, t in p.items()}
    xx = x.to("xdna").requires_grad_()
    (y, s), state = block(T, lv, xx, g.to("xdna"), heads, head)
    grads = torch.autograd.grad([y, s], [xx, *lv.values()], [dy.to("xdna"), dy.to("xdna")])
    ref = {n: t.float().requires_grad_() for n, t in p.items()}
    xr = x.float().requires_grad_()
    yr, sr, stater = block32(ref, xr, g, heads, head)
    want = torch.autograd.grad([yr, sr], [xr, *ref.values()], [dy.float(), dy.float()])
    for got, w, n in [(y, yr, "y"), (s, sr, "sum"), (state, stater, "state")] + list(zip(grads, want, ["x", *p])):
        off = (got.detach().cpu().float() - w.detach()).norm() / w.detach().norm()
        assert off <= 8 * 4 * B, (n, float(off))


def test_decoding_token_by_token_is_the_prompt(T):
    """The block's steps from the prompt's state against the prompt itself: the norms, projections and the
    feed-forward of a token are the same rows, the attention's states the same numbers up to their rounding."""
    Bn, Tn, width, heads, head = 3, 40, 64, 4, 16
    p = {n: t.to("xdna") for n, t in block_weights(width, heads, head, 4).items()}
    x = torch.randn(Bn, Tn, width, generator=gen(5)).to(BF16).to("xdna")
    g = -torch.exp2(-1.0 - torch.arange(heads).float()).to("xdna")
    with torch.no_grad():
        (y, _), state = block(T, p, x, g, heads, head)
        (_, _), s = block(T, p, x[:, :30], g, heads, head)
        s = s.clone()
        for t in range(30, Tn):
            xt = x[:, t]
            q, k, v = T.linear(T.layer_norm(xt, p["n1"], p["b1"]), p["qkv"], p["bq"]).view(Bn, 3, heads, head).unbind(1)
            a = T.decay_attention_step(q, k, v, g, s)
            xt = T.linear(a.reshape(Bn, heads * head), p["o"], residual=xt)
            r = T.add_layer_norm(T.gated_mlp(T.layer_norm(xt, p["n2"], p["b2"]), p["w_in"], p["w_out"]), xt, p["n1"], p["b1"])
            off = (r.norm.cpu().float() - y[:, t].cpu().float()).norm() / y[:, t].cpu().float().norm()
            assert off <= 8 * 4 * B, (t, float(off))
    off = (s - state).cpu().norm() / state.cpu().norm()
    assert off <= 4 * 4 * B, float(off)


def test_captured_block_replays_like_the_eager_one(T):
    """Forward, backward and a decoding step of a block as a graph, replayed with eager work between: the same bits
    each time."""
    Bn, Tn, width, heads, head = 2, 300, 64, 2, 32
    p = {n: t.to("xdna").requires_grad_() for n, t in block_weights(width, heads, head, 6).items()}
    x = torch.randn(Bn, Tn, width, generator=gen(7)).to(BF16).to("xdna")
    dy = torch.randn(Bn, Tn, width, generator=gen(8)).to(BF16).to("xdna")
    g = torch.tensor([-0.3, -0.01], device="xdna")
    lengths = torch.tensor([300, 171], device="xdna")
    pool = torch.zeros(4, heads, head, head, device="xdna")
    slots = torch.tensor([2, 0], device="xdna")

    def step():
        (y, s), state = block(T, p, x, g, heads, head, None, lengths)
        grads = torch.autograd.grad([y, s], list(p.values()), [dy, dy])
        with torch.no_grad():
            pool[:2].copy_(state.detach())
            qs = x[:, :3].reshape(Bn, 3, heads, head)
            o = T.decay_attention_step(qs[:, 0], qs[:, 1], qs[:, 2], g, pool, slots)
        return [y.detach(), s.detach(), o, *grads]

    eager = [t.cpu() for t in step()]
    pool_after = pool.cpu()
    for _ in range(2):
        step()
    graph = torch.xdna.Graph()
    with torch.xdna.graph(graph):
        out = step()
    for i in range(4):
        pool[2:].zero_()
        graph.replay()
        torch.xdna.synchronize()
        for j, (a, b) in enumerate(zip(out, eager)):
            assert same(a, b), (i, j)
        if i == 0:
            assert pool.shape == pool_after.shape
        between = [t.cpu() for t in step()] if i % 2 else None  # eager work between the replays
        del between
    graph.reset()


@pytest.mark.parametrize("leaves", ["alone", "shared"])
def test_captured_blocks_follow_their_inputs(T, leaves):
    """Two graphs of forward and backward, replayed in turn on inputs rewritten between the replays: the bits of eager
    runs on those inputs.  ``shared``: an eager graph of the same leaves lives while the two are captured, and its own
    backward runs after them."""
    width, heads, head = 64, 2, 32
    p = {n: t.to("xdna").requires_grad_() for n, t in block_weights(width, heads, head, 6).items()}
    g = torch.tensor([-0.3, -0.01], device="xdna")
    sizes = [(2, 300), (1, 1300)]
    host = [[torch.randn(Bn, Tn, width, generator=gen(20 + 4 * i + j)).to(BF16) for j in range(4)] for i, (Bn, Tn) in enumerate(sizes)]
    x = [h[0].to("xdna") for h in host]
    dy = [h[1].to("xdna") for h in host]

    def forward(i):
        (y, s), _ = block(T, p, x[i], g, heads, head, None, None)
        return y, s

    def step(i):
        y, s = forward(i)
        for t in p.values():
            t.grad = None
        torch.autograd.backward([y, s], [dy[i], dy[i]])
        return [y.detach(), s.detach(), *(t.grad for t in p.values())]

    def write(i, j):
        x[i].copy_(host[i][2 * j])
        dy[i].copy_(host[i][2 * j + 1])

    eager = {}
    for i in range(2):
        for j in range(2):
            write(i, j)
            eager[i, j] = [t.cpu() for t in step(i)]
    write(0, 0)
    live = forward(0) if leaves == "shared" else None
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.xdna.Graph())
        with torch.xdna.graph(graphs[i]):
            outs.append(step(i))
    if live is not None:
        of_live = torch.autograd.grad(live, list(p.values()), [dy[0], dy[0]])
        for a, b in zip(of_live, eager[0, 0][2:]):
            assert same(a, b)
    for i, j in [(0, 1), (1, 1), (0, 0), (1, 0), (1, 1), (0, 1)]:
        write(i, j)
        torch.xdna.synchronize()
        graphs[i].replay()
        torch.xdna.synchronize()
        for n, (a, b) in enumerate(zip(outs[i], eager[i, j])):
            assert same(a, b), (i, j, n)
    for gr in graphs:
        gr.reset()


def test_one_tensor_in_several_places(T):
    """A tensor that a call has twice or three times gets the sum of what separate ones get."""
    x, w = torch.randn(40, 64, generator=gen(1)).to(BF16), (torch.randn(64, 64, generator=gen(2)) / 8).to(BF16)
    dy = torch.randn(40, 64, generator=gen(3)).to(BF16).to("xdna")

    def grads(call, n, shape):
        one = x.view(shape).to("xdna").requires_grad_()
        several = [x.view(shape).to("xdna").requires_grad_() for _ in range(n)]
        y1, y = call(*[one] * n), call(*several)
        assert same(y1, y)
        g = torch.autograd.grad(y, several, dy.view(y.shape))
        return torch.autograd.grad(y1, one, dy.view(y1.shape))[0], [t.cpu().double() for t in g]

    log_decay = torch.tensor([-0.1, -0.5], device="xdna")
    for call, n, shape in [(lambda a, b: T.add_layer_norm(a, b).norm, 2, (40, 64)), (lambda a, b: T.linear(a, w.to("xdna"), None, "silu", b), 2, (40, 64)),
                           (lambda a, b, c: T.decay_attention(a, b, c, log_decay).out, 3, (2, 20, 2, 32))]:
        got, parts = grads(call, n, shape)
        size = sum(p.abs() for p in parts)
        assert ((got.cpu().double() - sum(parts)).abs() <= (n - 1) * B * size).all()  # (a rounding of each sum of two)


def test_a_result_written_before_its_backward_raises(T):
    x, r = (torch.randn(5, 16, generator=gen(i)).to("xdna").requires_grad_() for i in (1, 2))
    out = T.add_layer_norm(x, r)
    with torch.no_grad():
        out.sum.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.norm.sum().backward()
    q = torch.randn(1, 9, 1, 8, generator=gen(3)).to(BF16).to("xdna").requires_grad_()
    g, state = torch.tensor([-0.1], device="xdna"), torch.zeros(1, 1, 8, 8, device="xdna")
    a = T.decay_attention(q, q, q, g, state)
    with torch.no_grad():
        T.decay_attention_step(*[q[:, 0].detach()] * 3, g, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.out.sum().backward()


def test_captured_attention_follows_lengths_and_slots(T):
    """Lengths and slots are device data of a replay: rewritten between replays, they give the eager results."""
    v = {n: t.to("xdna") for n, t in decay_values(3, 200, 2, 2, 16, 24, seed=6).items()}
    lengths, slots = torch.tensor([200, 3, 64], device="xdna"), torch.tensor([0, 1, 2], device="xdna")
    pool = torch.zeros(4, 2, 16, 24, device="xdna")

    def run():
        a = T.decay_attention(v["q"], v["k"], v["v"], v["g"], v["state"], lengths)
        pool.zero_()
        pool[:3].copy_(a.state)
        return a.out, a.state, T.decay_attention_step(v["q"][:, 0], v["k"][:, 0], v["v"][:, 0], v["g"], pool, slots), pool.clone()

    run()
    graph = torch.xdna.Graph()
    with torch.xdna.graph(graph):
        out = run()
    for n, s in [([0, 200, 65], [3, 2, 0]), ([7, 128, 500], [-1, 0, 1]), ([200, 3, 64], [2, 1, 0]), ([63, 1, -2], [3, 1, 2])]:
        lengths.copy_(torch.tensor(n))
        slots.copy_(torch.tensor(s))
        torch.xdna.synchronize()
        graph.replay()
        torch.xdna.synchronize()
        got = [t.cpu() for t in out]
        for i, (a, b) in enumerate(zip(got, run())):
            assert same(a, b), (n, s, i)
    graph.reset()


def test_captured_steps_leave_the_pool_like_eager_ones(T):
    """A decoding step as a graph, after a prompt whose states it goes on with: the pool behind each replay has the bits of as
    many eager steps, in the slots that are named and in the others."""
    Bn, heads, head = 3, 2, 32
    v = {n: t.to("xdna") for n, t in decay_values(Bn, 200, heads, heads, head, head, seed=41).items()}
    start = torch.randn(5, heads, head, head, generator=gen(42))
    pool, slots = start.to("xdna"), torch.tensor([4, 0, 2], device="xdna")
    qkv = [v[n][:, 0].clone() for n in ("q", "k", "v")]

    def step():
        return T.decay_attention_step(*qkv, v["g"], pool, slots)

    def begin():
        pool.copy_(start)
        pool[:2].copy_(T.decay_attention(v["q"], v["k"], v["v"], v["g"], v["state"]).state[:2])

    with torch.no_grad():
        begin()
        eager = []
        for i in range(4):
            for t, n in zip(qkv, ("q", "k", "v")):
                t.copy_(v[n][:, i])
            eager.append((step().cpu(), pool.cpu()))
        graph = torch.xdna.Graph()
        with torch.xdna.graph(graph):
            out = step()
        for _ in range(2):
            begin()
            for i in range(4):
                for t, n in zip(qkv, ("q", "k", "v")):
                    t.copy_(v[n][:, i])
                torch.xdna.synchronize()
                graph.replay()
                torch.xdna.synchronize()
                assert same(out, eager[i][0]) and same(pool, eager[i][1]), i
                assert same(pool[1], eager[0][1][1]) and same(pool[3], start[3])
    graph.reset()


def test_refusals_on_the_device(T):
    x, w = torch.randn(3, 8, device="xdna"), torch.ones(8, device="xdna")
    for call, why in [
        (lambda: T.layer_norm(x.half(), w.half()), "float32 or bfloat16"), (lambda: T.layer_norm(x, w[:4]), "weight and bias"),
        (lambda: T.layer_norm(x, w, w.bfloat16()), "weight and bias"), (lambda: T.layer_norm(x.bfloat16(), w, w.bfloat16()), "one type"),
        (lambda: T.layer_norm(x, eps=-1.0), "eps"), (lambda: T.layer_norm(x, eps=math.inf), "eps"), (lambda: T.layer_norm(x, eps=1e39), "eps"),
        (lambda: T.layer_norm(x.cpu()), "xdna"), (lambda: T.add_layer_norm(x, x[:2]), "residual"), (lambda: T.add_layer_norm(x, x.bfloat16()), "residual"),
        (lambda: T.layer_norm(x, w.cpu()), "weight and bias"), (lambda: T.layer_norm(torch.zeros((), device="xdna")), "width"),
        (lambda: T.linear(x, x), "bfloat16"), (lambda: T.linear(x.bfloat16(), x[:, :4].bfloat16()), "weight"),
        (lambda: T.linear(x.bfloat16(), x.bfloat16(), w), "bias"), (lambda: T.linear(x.bfloat16(), x.bfloat16(), w.bfloat16()), "bias"),
        (lambda: T.linear(x.bfloat16(), x.bfloat16(), residual=x.bfloat16()), "residual"), (lambda: T.linear(x.bfloat16(), x.bfloat16(), activation="tanh"), "one of"),
    ]:
        with pytest.raises((RuntimeError, ValueError), match=why):
            call()
    q, k, v = (torch.zeros(2, 5, h, n, device="xdna", dtype=BF16) for h, n in ((4, 8), (2, 8), (2, 6)))
    g, s = torch.zeros(4, device="xdna"), torch.zeros(2, 4, 8, 6, device="xdna")
    wide = torch.zeros(2, 5, 4, 129, device="xdna", dtype=BF16)
    A, S = T.decay_attention, T.decay_attention_step
    q1, k1, v1 = q[:, 0], k[:, 0], v[:, 0]
    leaf = q.clone().requires_grad_()
    for call, why in [
        (lambda: A(q.float(), k, v, g), "bfloat16"), (lambda: A(q, k, v[:, :4], g), "tokens"), (lambda: A(q, k[..., :4], v, g), "heads of"),
        (lambda: A(q[:, :, :3], k, v, g[:3]), "divisor"), (lambda: A(q, k, v[:, :, :1], g), "divisor"), (lambda: A(wide, wide, wide, g), "1 to 128"),
        (lambda: A(q, k, v, g[:2]), "log_decay"), (lambda: A(q, k, v, g.bfloat16()), "log_decay"), (lambda: A(q, k, v, g.clone().requires_grad_()), "constant"),
        (lambda: A(q, k, v, g, s[:1]), "state"), (lambda: A(q, k, v, g, s.bfloat16()), "state"), (lambda: A(q, k, v, g, lengths=torch.zeros(3, device="xdna", dtype=torch.long)), "lengths"),
        (lambda: A(q, k, v, g, lengths=torch.zeros(2, device="xdna")), "int64 or int32"), (lambda: A(q, k, v, g, scale=math.inf), "scale"),
        (lambda: A(q, k, v, g, scale=math.nan), "scale"), (lambda: A(q1, k1, v1, g), "batch, tokens"), (lambda: S(q, k, v, g, s), "batch, heads"),
        (lambda: S(q1, k1, v1, g, s[:1]), "without slots"), (lambda: S(q1, k1, v1, g, s.transpose(0, 1)), "contiguous"),
        (lambda: S(q1, k1, v1, g, s.bfloat16()), "float32"), (lambda: S(q1, k1, v1, g, s, torch.zeros(3, device="xdna", dtype=torch.long)), "slots"),
        (lambda: S(q1, k1, v1, g, s, torch.zeros(2, device="xdna")), "int64 or int32"), (lambda: S(leaf[:, 0], k1, v1, g, s), "no gradient"),
        (lambda: S(q1, k1, v1, g, s.clone().requires_grad_()), "no gradient"),
    ]:
        with pytest.raises((RuntimeError, ValueError), match=why):
            call()
    r = A(leaf, k, v, g)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(r.out.sum(), [leaf], create_graph=True)


def test_work_on_another_stream_is_refused(T):
    """The device's allocator orders its blocks on one stream: a call on a stream beside it raises, and writes nothing."""
    x, w = torch.randn(40, 64, device="xdna").bfloat16(), torch.ones(64, 64, device="xdna", dtype=BF16)
    q, g = torch.zeros(2, 5, 2, 8, device="xdna", dtype=BF16), torch.zeros(2, device="xdna")
    state = torch.ones(2, 2, 8, 8, device="xdna")
    before = T.linear(x, w)
    torch.xdna.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for call in (lambda: T.layer_norm(x), lambda: T.add_layer_norm(x, x), lambda: T.linear(x, w), lambda: T.decay_attention(q, q, q, g, state),
                     lambda: T.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], g, state)):
            with pytest.raises(RuntimeError, match="default one is not supported"):
                call()
    torch.cuda.synchronize()
    assert same(T.linear(x, w), before) and (state.cpu() == 1).all()


def test_forward_mode_is_refused(T):
    import torch.autograd.forward_ad as fw

    x = torch.randn(3, 8, device="xdna").bfloat16()
    q = torch.zeros(1, 3, 2, 8, device="xdna", dtype=BF16)
    g, s = torch.zeros(2, device="xdna"), torch.zeros(1, 2, 8, 8, device="xdna")
    with fw.dual_level():
        d, dq = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(q, torch.ones_like(q))
        for call in (lambda: T.layer_norm(d), lambda: T.add_layer_norm(x, d), lambda: T.linear(x, d), lambda: T.linear(x, x, residual=fw.make_dual(x[:, :3].contiguous(), x[:, :3].contiguous())),
                     lambda: T.decay_attention(q, dq, q, g), lambda: T.decay_attention_step(dq[:, 0], q[:, 0], q[:, 0], g, s)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
