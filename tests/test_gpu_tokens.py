"""Token-model operators (xdna_train.tokens) against plain 64-bit implementations on the CPU,
at the sizes, masks and strides where they can go wrong.

Tolerances, per element.  u = 2^-24 (half an fp32 ulp at 1), b = 2^-8 (half a bf16 ulp at 1, the
one rounding of a bf16 result):
* lookups: bit-exact (one fp32 product, one rounding);
* embedding gradient: n u sum |scale dy| for a row of n tokens (any order of fp32 sums), plus
  the result's rounding;
* log probabilities: (64 + 8 |value|) u: the sum over the vocabulary goes through 32 terms a
  thread and under 32 more levels, each hardware exp is within 2 u and its argument, a
  difference times a constant, within 2 u of itself; entropy: 4 times that on 1 + H + |ln s|;
* gradients of rows: (64 + 4 |ln q|) u on every term's magnitude (exp turns the two roundings of
  its argument into |ln q| u each), plus the result's rounding;
* gated products: see gated_reference, which carries each rounding's bound through the products.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TINY = 1e-37  # the hardware exp flushes results below the normal range


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
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    bad = ~same & ~((got - ref).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4],
                           (tol[bad][:4] if torch.is_tensor(tol) and tol.shape == ref.shape else tol))


def padded(t, extra, offset=0):
    """t's values in a larger allocation: rows `extra` elements apart, `offset` elements in."""
    rows, n = t.shape
    buf = torch.full((rows * (n + extra) + offset + 8,), 7.0, dtype=t.dtype, device="xdna")
    v = torch.as_strided(buf, (rows, n), (n + extra, 1), offset)
    v.copy_(t)
    return v


# ---- embedding --------------------------------------------------------------------------------

EMBED = [  # tokens, vocabulary, width
    (1, 1, 1), (1, 5, 8), (3, 2, 7), (31, 9, 33), (32, 300, 64), (33, 1, 40), (65, 70000, 17), (257, 511, 512),
    (300, 512, 520), (1000, 513, 129), (8191, 40, 24), (8192, 1024, 8), (8193, 1000, 16), (20000, 300000, 9), (17000, 3, 72),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,V,D", EMBED)
def test_embedding(T, n, V, D, dtype):
    print("embedding", n, V, D, dtype, flush=True)
    g = gen(n + V + D)
    scale = 1.0 if D % 2 else math.sqrt(D)
    w = torch.randn(V, D, generator=g).to(dtype)
    ids = (torch.rand(n, generator=g, dtype=F64) ** 3 * V).long().clamp_(max=V - 1)  # crowded low ids
    dy = torch.randn(n, D, generator=g).to(dtype)
    wx = w.to("xdna").requires_grad_()
    y = T.embed(ids.to("xdna"), wx, scale=scale)
    assert torch.equal(y.detach().cpu(), (w[ids].float() * torch.tensor(scale, dtype=F32)).to(dtype))
    y.backward(dy.to("xdna"))
    ref = torch.zeros(V, D, dtype=F64).index_add_(0, ids, dy.to(F64)) * scale
    mag = torch.zeros(V, D, dtype=F64).index_add_(0, ids, dy.to(F64).abs()) * scale
    count = torch.bincount(ids, minlength=V).to(F64)[:, None]
    close(wx.grad, ref, (count + 2) * U * mag + rounding(dtype) * ref.abs(), "embedding gradient")
    again = torch.autograd.grad(T.embed(ids.to("xdna"), wx, scale=scale), [wx], dy.to("xdna"))[0]
    assert torch.equal(again.cpu(), wx.grad.cpu()), "equal inputs, different bits"


@pytest.mark.parametrize("n", [200, 9000])
def test_embedding_padding_outside_ids_strides_and_int32(T, n):
    print("embedding edges", n, flush=True)
    V, D, pad = 50, 37, 7
    g = gen(n)
    ids = torch.randint(-3, V + 3, (n,), generator=g)
    ids[::5] = pad
    w, dy = torch.randn(V, D, generator=g).bfloat16(), torch.randn(n, D, generator=g).bfloat16()
    wx = padded(w, 3, 1).requires_grad_()
    y = T.embed(ids.int().to("xdna"), wx, scale=0.5, padding_idx=pad - V)
    inside = (ids >= 0) & (ids < V)
    got = y.detach().cpu()
    assert torch.equal(got[inside], (w[ids[inside]].float() * 0.5).bfloat16())
    assert torch.isnan(got[~inside].float()).all()
    dyx = padded(dy, 11, 3)
    (dw,) = torch.autograd.grad(y, [wx], dyx)
    keep = inside & (ids != pad)
    ref = torch.zeros(V, D, dtype=F64).index_add_(0, ids[keep], dy[keep].to(F64)) * 0.5
    mag = torch.zeros(V, D, dtype=F64).index_add_(0, ids[keep], dy[keep].to(F64).abs())
    close(dw, ref, n * U * mag + B * ref.abs(), "gradient with padding")
    assert not dw[pad].cpu().any()


def test_embedding_without_tokens_and_of_any_shape(T):
    w = torch.randn(6, 5, generator=gen(0)).to("xdna").requires_grad_()
    y = T.embed(torch.zeros(0, 3, dtype=torch.long, device="xdna"), w)
    assert y.shape == (0, 3, 5)
    (dw,) = torch.autograd.grad(y, [w], torch.zeros(0, 3, 5, device="xdna"))
    assert not dw.cpu().any() and dw.shape == w.shape
    ids = torch.tensor([[0, 5], [2, 2]], device="xdna")
    assert torch.equal(T.embed(ids, w).detach().cpu(), w.detach().cpu()[ids.cpu()])
    broadcast = torch.ones(1, 1, 5, device="xdna").expand(2, 2, 5)  # a gradient of stride 0
    (dw,) = torch.autograd.grad(T.embed(ids, w), [w], broadcast)
    assert dw.cpu()[:, 0].tolist() == [1, 0, 2, 0, 0, 1]


# ---- gated feed-forward -----------------------------------------------------------------------

def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).to(F64)


def gated_reference(x, w, wo, dy, act, fused):
    """Values and bounds: {name: (value, tolerance)}.  Each stored bf16 value is off by b of itself,
    each fp32 sum of n products by (n + 8) u of the sum of magnitudes; act' is at most 1.13 and act''
    at most 0.8 in size (relu: a rounded gate keeps its sign).  fused: dh is not stored."""
    x, w, wo, dy = (t.to(F64) for t in (x, w, wo, dy))
    F = w.shape[0] // 2
    K, N, M = x.shape[1], wo.shape[0], x.shape[0]
    g, u = x @ w[:F].t(), x @ w[F:].t()
    eg = (K + 8) * U * (x.abs() @ w[:F].abs().t())
    eu = (K + 8) * U * (x.abs() @ w[F:].abs().t())
    a, da = act64(act, g)
    ea = 1.13 * eg + 16 * U * (a.abs() + g.abs())
    h = a * u
    eh = ea * u.abs() + (a.abs() + ea) * eu + B * h.abs()
    y = h @ wo.t()
    ey = (eh + (F + 8) * U * h.abs()) @ wo.abs().t() + B * y.abs()
    dh = dy @ wo
    edh = (N + 8) * U * (dy.abs() @ wo.abs()) + (0 if fused else B) * dh.abs()
    kg, ku = eg + B * g.abs(), eu + B * u.abs()  # the kept projections
    eda = (0.8 * kg if act != "relu" else torch.where(g.abs() <= 4 * eg, 1.0, 0.0)) + 32 * U * (1 + g.abs())
    eka = 1.13 * kg + 16 * U * (a.abs() + g.abs())
    dg, du = dh * u * da, dh * a
    edg = edh * (u.abs() + ku) * (da.abs() + eda) + dh.abs() * (ku * (da.abs() + eda) + u.abs() * eda)
    edu = edh * (a.abs() + eka) + dh.abs() * eka
    d = torch.cat([dg, du], 1)
    ed = torch.cat([edg + B * dg.abs(), edu + B * du.abs()], 1)
    dx = d @ w
    edx = (ed + (2 * F + 8) * U * d.abs()) @ w.abs() + B * dx.abs()
    dw = d.t() @ x
    edw = (ed + (M + 8) * U * d.abs()).t() @ x.abs() + B * dw.abs()
    dwo = dy.t() @ h
    edwo = dy.abs().t() @ (eh + (M + 8) * U * h.abs()) + B * dwo.abs()
    out = {"h": (h, eh), "y": (y, ey), "dx": (dx, edx), "dw_in": (dw, edw), "dw_out": (dwo, edwo)}
    return {k: (v, e + 1e-30) for k, (v, e) in out.items()}


GATED = [  # rows, K, F, N
    (1, 1, 1, 1), (1, 64, 32, 16), (1, 1000, 520, 1000), (2, 7, 5, 3), (5, 72, 100, 33), (16, 256, 128, 64), (17, 130, 63, 65),
    (33, 8, 65, 8), (63, 200, 64, 17), (64, 64, 64, 64), (65, 65, 129, 100), (130, 512, 384, 512), (333, 1000, 217, 1000),
]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,F,N", GATED)
def test_gated_mlp(T, M, K, F, N, act):
    print("gated", M, K, F, N, act, flush=True)
    g = gen(M * 7 + K + F)
    x, dy = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, N, generator=g).bfloat16()
    w = (torch.randn(2 * F, K, generator=g) / math.sqrt(K)).bfloat16()
    wo = (torch.randn(N, F, generator=g) / math.sqrt(F)).bfloat16()
    ref = gated_reference(x, w, wo, dy, act, True)
    leaves = [t.to("xdna").requires_grad_() for t in (x, w, wo)]
    y = T.gated_mlp(*leaves, activation=act)
    got = torch.autograd.grad(y, leaves, dy.to("xdna"))
    close(y, *ref["y"], "y")
    for name, t in zip(("dx", "dw_in", "dw_out"), got):
        close(t, *ref[name], name)
    with torch.no_grad():
        h = T.gated_linear(leaves[0], leaves[1], activation=act)
        close(h, *ref["h"], "h")
        close(T.gated_mlp(*leaves, activation=act), *ref["y"], "y without gradients")


@pytest.mark.parametrize("M,K,F", [(1, 24, 40), (70, 130, 96), (300, 256, 131)])
def test_gated_linear_gradient_and_strides(T, M, K, F):
    print("gated strides", M, K, F, flush=True)
    g = gen(M + F)
    x, dh = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, F, generator=g).bfloat16()
    w = (torch.randn(2 * F, K, generator=g) / math.sqrt(K)).bfloat16()
    xs, ws = padded(x, 5, 1).requires_grad_(), padded(w, 3, 5).requires_grad_()
    h = T.gated_linear(xs, ws, activation="silu")
    # with the identity as w_out, dy is dh itself, exactly
    ref = gated_reference(x, w, torch.eye(F), dh, "silu", True)
    close(h, *ref["h"], "h")
    got = torch.autograd.grad(h, [xs, ws], padded(dh, 9, 3))
    close(got[0], *ref["dx"], "dx")
    close(got[1], *ref["dw_in"], "dw_in")
    # x transposed in memory, w's columns a slice of a wider matrix: the same values
    xt = x.t().contiguous().to("xdna").t()
    assert torch.equal(T.gated_linear(xt, ws).cpu(), h.detach().cpu())
    x3 = x.view(1, M, K).to("xdna")
    assert torch.equal(T.gated_linear(x3, ws).cpu()[0], h.detach().cpu())


def test_gated_without_rows(T):
    w = torch.randn(8, 6, generator=gen(1)).bfloat16().to("xdna").requires_grad_()
    wo = torch.randn(5, 4, generator=gen(2)).bfloat16().to("xdna").requires_grad_()
    x = torch.zeros(0, 6, dtype=BF16, device="xdna").requires_grad_()
    y = T.gated_mlp(x, w, wo)
    assert y.shape == (0, 5)
    dx, dw, dwo = torch.autograd.grad(y, [x, w, wo], torch.zeros(0, 5, dtype=BF16, device="xdna"))
    assert dx.shape == (0, 6) and not dw.float().cpu().any() and not dwo.float().cpu().any()


# ---- rows over a vocabulary -------------------------------------------------------------------

VOCABS = [1, 2, 7, 64, 100, 1003, 2047, 2048, 2049, 4097, 8192, 8193, 32768, 32769, 50001, 131072]


def make_logits(rows, V, dtype, seed, masked=0.0, extra=0):
    g = gen(seed)
    z = 3 * torch.randn(rows, V, generator=g)
    if masked:
        z[torch.rand(rows, V, generator=g) < masked] = -math.inf
    z = z.to(dtype)
    return z, padded(z, extra, extra % 5).requires_grad_()


def logprob_reference(z, y, tau, k):
    x = z.to(F64) / tau
    m = x.amax(1, keepdim=True)
    empty = (m == -math.inf)[:, 0]
    m0 = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(x - m0)
    s = e.sum(1, keepdim=True)
    lq = torch.where(empty[:, None], torch.full_like(x, -math.inf), x - m0 - torch.log(s))
    q = torch.where(empty[:, None], torch.zeros_like(x), e / s)
    h = -torch.where(q > 0, q * lq, torch.zeros_like(q)).sum(1)
    lp = lq.gather(1, y.clamp(min=0)[:, None])[:, 0]
    lp = torch.where(y >= 0, lp, torch.zeros_like(lp))
    ids = torch.argsort(z.to(F64), dim=1, descending=True, stable=True)[:, :k]
    return lp, h, lq.gather(1, ids), ids, q, lq


def tol_log(v):
    return (64 + 8 * torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))) * U


def grad_tol(terms, ref, dtype, lq):
    return (64 + 4 * lq.abs()) * U * terms + rounding(dtype) * ref.abs() + TINY


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("rows,k,tau,masked", [(3, 20, 1.0, 0.0), (5, 64, 0.7, 0.6), (2, 1, 2.0, 0.0)])
def test_token_log_probs(T, rows, V, k, tau, masked, dtype):
    print("log probabilities", rows, V, k, tau, masked, dtype, flush=True)
    k = min(k, V)
    z, zx = make_logits(rows, V, dtype, V + rows, masked, extra=V % 9)
    y = torch.randint(0, V, (rows,), generator=gen(V))
    y[-1] = -100
    r = T.token_log_probs(zx, y.to("xdna"), top_k=k, temperature=tau)
    lp, h, tlp, tid, q, lq = logprob_reference(z, y, tau, k)
    close(r.log_probs, lp, tol_log(lp), "log_probs")
    etol = 4 * U * (64 + 8 * 30 / tau) * (1 + h)
    close(r.entropy, h, etol, "entropy")
    assert torch.equal(r.top_ids.cpu(), tid), "top ids"
    close(r.top_log_probs, tlp, tol_log(tlp), "top log_probs")
    gl, gh = torch.randn(rows, generator=gen(1)), torch.randn(rows, generator=gen(2))
    (dz,) = torch.autograd.grad([r.log_probs, r.entropy], [zx], [gl.to("xdna"), gh.to("xdna")])
    gl64, gh64 = torch.where(y >= 0, gl, torch.zeros(rows)).to(F64)[:, None], gh.to(F64)[:, None]
    hot = torch.zeros(rows, V, dtype=F64).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    some = (q.sum(1, keepdim=True) > 0).to(F64)
    lqf = torch.where(q > 0, lq, torch.zeros_like(lq))
    ref = (gl64 * (hot - q) * some - gh64 * q * (lqf + h[:, None])) / tau
    terms = (gl64.abs() * (hot + q) + gh64.abs() * q * (1 + lqf.abs() + h[:, None])) / tau
    close(dz, ref, grad_tol(terms, ref, dtype, lqf), "gradient")


def test_log_probs_of_many_rows_take_the_wide_workgroups(T):
    """256 rows of 40000: two pieces of a wide workgroup each, joined."""
    rows, V, k = 256, 40000, 8
    print("wide rows", flush=True)
    z, zx = make_logits(rows, V, BF16, 5)
    y = torch.randint(0, V, (rows,), generator=gen(6))
    r = T.token_log_probs(zx.detach(), y.to("xdna"), top_k=k)
    lp, h, tlp, tid, _, _ = logprob_reference(z, y, 1.0, k)
    close(r.log_probs, lp, tol_log(lp), "log_probs")
    close(r.entropy, h, 4 * U * 304 * (1 + h), "entropy")
    assert torch.equal(r.top_ids.cpu(), tid)
    close(r.top_log_probs, tlp, tol_log(tlp), "top")


def order_rows(V, kind, g):
    i = torch.arange(V, dtype=F32)
    if kind == "equal":
        return torch.zeros(V)
    if kind == "falling":
        return -i / 16
    if kind == "rising":
        return i / 16
    if kind == "stride":      # the largest all at one lane's places
        return torch.where(i % 512 < 8, 40 + i / V, torch.randn(V, generator=g))
    if kind == "few":         # fewer tokens allowed than asked for
        z = torch.full((V,), -math.inf)
        z[torch.randperm(V, generator=g)[:3]] = torch.tensor([1.0, 1.0, 2.0])
        return z
    if kind == "zeros":       # -0 and +0 are equal: the lower index comes first
        return torch.where(i % 3 == 0, torch.tensor(-0.0), torch.tensor(0.0))
    z = torch.full((V,), -math.inf)
    return z                  # "barred": nothing allowed


@pytest.mark.parametrize("kind", ["equal", "falling", "rising", "stride", "few", "zeros", "barred"])
@pytest.mark.parametrize("V", [70, 2048, 8192, 20000, 70000])
def test_top_alternatives_of_special_orders(T, V, kind):
    print("order", V, kind, flush=True)
    k = 40
    z = torch.stack([order_rows(V, kind, gen(V + i)) for i in range(2)])
    y = torch.tensor([0, V - 1])
    for dtype in (BF16, F32):
        zd = z.to(dtype)
        r = T.token_log_probs(zd.to("xdna"), y.to("xdna"), top_k=k)
        lp, h, tlp, tid, _, _ = logprob_reference(zd, y, 1.0, k)
        assert torch.equal(r.top_ids.cpu(), tid), dtype
        close(r.top_log_probs, tlp, tol_log(tlp), "top")
        close(r.log_probs, lp, tol_log(lp), "log_probs")
        close(r.entropy, h, 4 * U * 304 * (1 + h), "entropy")


def test_log_probs_of_nan_infinite_and_lowest_logits(T):
    V = 3000
    z = torch.randn(5, V, generator=gen(3))
    z[0, 17] = math.nan
    z[1, 2999] = math.inf
    z[2] = torch.finfo(F32).min          # a mask of the type's lowest value: an even row
    z[3, 5:] = torch.finfo(F32).min
    y = torch.tensor([3, 4, 5, 2, V])    # the last is past the vocabulary
    zx = z.to("xdna").requires_grad_()
    r = T.token_log_probs(zx, y.to("xdna"), top_k=2)
    lp = r.log_probs.detach().cpu()
    assert torch.isnan(lp[0]) and torch.isnan(lp[1]) and torch.isnan(lp[4])
    assert r.top_ids.cpu()[0, 0] == 17 and r.top_ids.cpu()[1, 0] == 2999 and r.top_ids.cpu()[2].tolist() == [0, 1]
    ref = logprob_reference(z[2:4], y[2:4], 1.0, 2)
    close(r.log_probs[2:4], ref[0], tol_log(ref[0]), "log_probs")
    close(r.entropy[2:4], ref[1], 4 * U * 304 * (1 + ref[1]), "entropy")
    (dz,) = torch.autograd.grad(r.log_probs[2:4].sum(), [zx])
    dz = dz.cpu()
    assert not dz[0].any() and not dz[1].any() and not dz[4].any()  # no incoming gradient: not even NaN
    close(dz[3], torch.nn.functional.one_hot(torch.tensor(2), V).to(F64) - ref[4][1], 128 * U * torch.ones(V, dtype=F64), "gradient")


def test_log_probs_shapes_and_one_gradient(T):
    z = torch.randn(2, 3, 11, generator=gen(9))
    y = torch.randint(0, 11, (2, 3), generator=gen(10))
    zx = z.to("xdna").requires_grad_()
    r = T.token_log_probs(zx, y.int().to("xdna"), top_k=4)
    assert r.log_probs.shape == (2, 3) and r.top_ids.shape == (2, 3, 4) and r.top_log_probs.shape == (2, 3, 4)
    assert not r.top_log_probs.requires_grad
    lp, h, _, _, q, lq = logprob_reference(z.view(6, 11), y.view(6), 1.0, 4)
    (dz,) = torch.autograd.grad(r.entropy.sum(), [zx])
    ref = -q * (lq + h[:, None])
    close(dz.view(6, 11), ref, grad_tol(q * (1 + lq.abs() + h[:, None]), ref, F32, lq), "entropy's gradient")
    empty = T.token_log_probs(torch.zeros(0, 5, device="xdna"), torch.zeros(0, dtype=torch.long, device="xdna"), top_k=2)
    assert empty.log_probs.shape == (0,) and empty.top_ids.shape == (0, 2)


def test_log_probs_gradient_against_differences(T):
    """Central differences of the forward: the step's third-order term and the forward's rounding
    over the step are both under 1e-3 of the slope's scale here."""
    V, eps = 301, 2.0 ** -5
    z = torch.randn(4, V, generator=gen(20))
    d = torch.randn(4, V, generator=gen(21))
    y = torch.randint(0, V, (4,), generator=gen(22)).to("xdna")

    def value(t):
        r = T.token_log_probs(t, y, temperature=0.9)
        return r.log_probs.sum() + 0.5 * r.entropy.sum()

    zx = z.to("xdna").requires_grad_()
    (dz,) = torch.autograd.grad(value(zx), [zx])
    slope = (value((z + eps * d).to("xdna")) - value((z - eps * d).to("xdna"))).item() / (2 * eps)
    assert abs(slope - float((dz.cpu() * d).sum())) <= 1e-3 * float((dz.cpu() * d).abs().sum())


# ---- distillation -----------------------------------------------------------------------------

def distill_reference(z, ids, t, tau, w, reduction):
    x = z.to(F64) / tau
    lq = torch.log_softmax(x, 1)
    q = torch.exp(lq)
    valid = (ids >= 0) & (t > -math.inf)
    has = valid.any(1)
    tt = torch.where(valid, t.to(F64) / tau, torch.full(t.shape, -math.inf, dtype=F64))
    p = torch.where(has[:, None], torch.softmax(tt, 1), torch.zeros_like(tt))
    p = torch.nan_to_num(p)
    lp = torch.where(p > 0, torch.log(p), torch.zeros_like(p))
    lqi = lq.gather(1, ids.clamp(min=0))
    rows = tau * tau * torch.where(p > 0, p * (lp - lqi), torch.zeros_like(p)).sum(1)
    mag = tau * tau * torch.where(p > 0, p * (lp.abs() + lqi.abs() + 1), torch.zeros_like(p)).sum(1)
    share = torch.where(has, w.to(F64), torch.zeros(len(w), dtype=F64))
    total = share.sum() if reduction == "mean" else 1.0
    share = torch.where(share != 0, share / (total if total else 1.0), torch.zeros_like(share))
    rows = torch.where(share != 0, share * rows, torch.zeros_like(rows))
    dz = (q.scatter_add(1, ids.clamp(min=0), -p)) * (share * tau)[:, None]
    terms = (q.scatter_add(1, ids.clamp(min=0), p)) * (share.abs() * tau)[:, None]
    return rows, share.abs() * mag, dz, terms


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,V,k,tau,reduction", [
    (1, 2, 1, 1.0, "mean"), (3, 7, 3, 2.0, "sum"), (61, 1003, 8, 1.0, "mean"), (5, 2049, 64, 0.7, "none"), (4, 8192, 65, 1.0, "mean"),
    (7, 40001, 128, 3.0, "mean"), (2, 131072, 1000, 1.0, "sum"), (300, 33000, 5, 1.0, "mean")])
def test_distillation(T, rows, V, k, tau, reduction, dtype):
    print("distillation", rows, V, k, tau, reduction, dtype, flush=True)
    g = gen(rows + V + k)
    z, zx = make_logits(rows, V, dtype, V + 1, extra=V % 7)
    ids = torch.randint(0, V, (rows, k), generator=g)   # names a token twice now and then
    t = 4 * torch.randn(rows, k, generator=g)
    ids[torch.rand(rows, k, generator=g) < 0.2] = -1
    t[torch.rand(rows, k, generator=g) < 0.1] = -math.inf
    w = torch.rand(rows, generator=g)
    if rows > 2:
        w[1] = 0.0
        ids[2] = -1  # a row without entries
    loss = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), temperature=tau, weight=w.to("xdna"), reduction=reduction)
    per_row, mag, dz, terms = distill_reference(z, ids, t, tau, w, reduction)
    if reduction == "none":
        close(loss, per_row, 128 * U * mag, "row losses")
        go = torch.randn(rows, generator=g)
        (got,) = torch.autograd.grad(loss, [zx], go.to("xdna"))
        dz, terms = dz * go.to(F64)[:, None], terms * go.abs().to(F64)[:, None]
    else:
        close(loss, per_row.sum(), 128 * U * mag.sum(), "loss")
        (got,) = torch.autograd.grad(loss, [zx], torch.tensor(-1.5, device="xdna"))
        dz, terms = -1.5 * dz, 1.5 * terms
    close(got, dz, grad_tol(2 * terms, dz, dtype, torch.log_softmax(z.to(F64) / tau, 1)), "gradient")
    again = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), temperature=tau, weight=w.to("xdna"), reduction=reduction)
    assert torch.equal(again.detach().cpu(), loss.detach().cpu())


def test_distillation_without_weight_in_bf16_teacher_and_empty(T):
    z, t = torch.randn(2, 3, 50, generator=gen(1)), torch.randn(2, 3, 4, generator=gen(2)).bfloat16()
    ids = torch.randint(0, 50, (2, 3, 4), generator=gen(3))
    loss = T.distill_loss(z.to("xdna"), ids.int().to("xdna"), t.to("xdna"))
    rows, mag, _, _ = distill_reference(z.view(6, 50), ids.view(6, 4), t.view(6, 4).float(), 1.0, torch.ones(6), "mean")
    close(loss, rows.sum(), 128 * U * mag.sum(), "loss")
    none = T.distill_loss(z.to("xdna"), torch.full_like(ids, -1).to("xdna"), t.to("xdna"))
    assert none.item() == 0.0
    zx = torch.zeros(0, 50, device="xdna", requires_grad=True)
    empty = T.distill_loss(zx, torch.zeros(0, 2, dtype=torch.long, device="xdna"), torch.zeros(0, 2, device="xdna"))
    (dz,) = torch.autograd.grad(empty, [zx])
    assert empty.item() == 0.0 and dz.shape == (0, 50)


def test_distillation_of_masked_and_invalid_rows(T):
    """Weight 0 leaves a row out whatever it holds; -inf student logits outside the entries add
    nothing; a barred entry's loss is infinite; an id past the vocabulary makes the loss NaN."""
    V = 100
    z = torch.randn(4, V, generator=gen(4))
    ids = torch.tensor([[1, 2], [3, 4], [5, 6], [7, 8]])
    t = torch.zeros(4, 2)
    z[0] = math.nan
    z[1, 50:] = -math.inf
    w = torch.tensor([0.0, 1.0, 1.0, 0.0])
    zx = z.to("xdna").requires_grad_()
    loss = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"))
    ref = distill_reference(z[1:3], ids[1:3], t[1:3], 1.0, w[1:3], "mean")
    close(loss, ref[0].sum(), 128 * U * ref[1].sum(), "loss")
    (dz,) = torch.autograd.grad(loss, [zx])
    assert not dz[0].cpu().any() and not dz[3].cpu().any() and not dz[1, 50:].cpu().any()
    close(dz[1:3], ref[2], 128 * U * ref[3] + U * ref[2].abs() + TINY, "gradient")
    z[1, 3] = -math.inf
    each = T.distill_loss(z.to("xdna"), ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"), reduction="none").cpu()
    assert each[0] == 0 and each[1] == math.inf and each[3] == 0
    ids[2, 0] = V
    assert torch.isnan(T.distill_loss(z.to("xdna"), ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"))).item()


@pytest.mark.parametrize("rows, V", [(2, 100), (2, 20000)])
def test_distillation_leaves_out_rows_of_weight_zero_with_invalid_ids(T, rows, V):
    z = torch.randn(rows, V, generator=gen(5))
    ids = torch.tensor([[V + 3, 1], [2, 3]])
    t = torch.zeros(rows, 2)
    zx = z.to("xdna").requires_grad_()
    each = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=torch.tensor([0.0, 1.0]).to("xdna"), reduction="none")
    ref = distill_reference(z[1:], ids[1:], t[1:], 1.0, torch.ones(1), "none")
    assert each[0].item() == 0.0
    close(each[1:], ref[0], 128 * U * ref[1], "loss")
    (dz,) = torch.autograd.grad(each.sum(), [zx])
    assert not dz[0].cpu().any() and torch.isfinite(dz).all().item()


def test_distillation_gradient_against_differences(T):
    V, eps = 200, 2.0 ** -5
    z, d = torch.randn(3, V, generator=gen(30)), torch.randn(3, V, generator=gen(31))
    ids = torch.randint(0, V, (3, 9), generator=gen(32)).to("xdna")
    t = torch.randn(3, 9, generator=gen(33)).to("xdna")

    def value(a):
        return T.distill_loss(a, ids, t, temperature=1.5, reduction="sum")

    zx = z.to("xdna").requires_grad_()
    (dz,) = torch.autograd.grad(value(zx), [zx])
    slope = (value((z + eps * d).to("xdna")) - value((z - eps * d).to("xdna"))).item() / (2 * eps)
    assert abs(slope - float((dz.cpu() * d).sum())) <= 1e-3 * float((dz.cpu() * d).abs().sum())


def test_gated_gradient_against_differences(T):
    """In bf16 the differences are noisy: the forward's rounding, b of the terms of y, over the step."""
    M, K, F = 8, 64, 48
    g = gen(40)
    x = torch.randn(M, K, generator=g).bfloat16()
    w = (torch.randn(2 * F, K, generator=g) / 8).bfloat16()
    wo = (torch.randn(K, F, generator=g) / 7).bfloat16()
    c, d = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, K, generator=g)
    leaves = [t.to("xdna").requires_grad_() for t in (x, w, wo)]
    (dx,) = torch.autograd.grad(T.gated_mlp(*leaves), [leaves[0]], c.to("xdna"))
    eps = 2.0 ** -4
    hi, lo = (x.float() + eps * d).bfloat16(), (x.float() - eps * d).bfloat16()
    with torch.no_grad():
        f = [(T.gated_mlp(t.to("xdna"), leaves[1], leaves[2]).cpu().to(F64) * c.to(F64)) for t in (hi, lo)]
    step = hi.to(F64) - lo.to(F64)
    noise = 2 * B * float((f[0].abs() + f[1].abs()).sum()) + 0.02 * float((dx.cpu().to(F64) * step).abs().sum())
    assert abs(float(f[0].sum() - f[1].sum()) - float((dx.cpu().to(F64) * step).sum())) <= noise


# ---- use --------------------------------------------------------------------------------------

def test_captured_step_replays_like_the_eager_one(T):
    """A whole token step as a graph, replayed with eager work between: the same bits each time."""
    import xdna_train  # noqa: F401
    V, D, F, n = 500, 64, 96, 70
    g = gen(50)
    table = torch.randn(V, D, generator=g).bfloat16().to("xdna").requires_grad_()
    w_in = (torch.randn(2 * F, D, generator=g) / 8).bfloat16().to("xdna").requires_grad_()
    w_out = (torch.randn(D, F, generator=g) / 10).bfloat16().to("xdna").requires_grad_()
    ids = torch.randint(0, V, (n,), generator=g).to("xdna")
    t_ids = torch.randint(0, V, (n, 6), generator=g).to("xdna")
    t = torch.randn(n, 6, generator=g).to("xdna")
    params = [table, w_in, w_out]

    def step():
        x = T.embed(ids, table, scale=8.0)
        logits = torch.mm(x + T.gated_mlp(x, w_in, w_out), table.t())
        loss = T.distill_loss(logits, t_ids, t)
        r = T.token_log_probs(logits, ids, top_k=3)
        return [loss.detach(), r.log_probs.detach(), r.top_ids, *torch.autograd.grad(loss - r.log_probs.mean(), params)]

    def fresh(seed):
        return torch.randint(0, V, (n,), generator=gen(seed))

    for _ in range(2):
        step()
    graph = torch.xdna.Graph()
    with torch.xdna.graph(graph):
        out = step()
    for seed in (60, 61, 62):
        ids.copy_(fresh(seed))
        graph.replay()
        torch.xdna.synchronize()
        got = [o.cpu() for o in out]
        torch.zeros(1000, device="xdna").add_(1).sum().item()
        for a, b in zip(got, step()):
            assert torch.equal(a, b.cpu())


def test_refusals_on_the_device(T):
    z = torch.zeros(2, 5, device="xdna")
    y = torch.zeros(2, dtype=torch.long, device="xdna")
    w = torch.zeros(4, 3, device="xdna")
    x16 = torch.zeros(2, 6, dtype=BF16, device="xdna")
    w16, wo16 = torch.zeros(8, 6, dtype=BF16, device="xdna"), torch.zeros(6, 4, dtype=BF16, device="xdna")
    two = torch.zeros(2, 2, device="xdna")
    bad = [
        lambda: T.embed(y.float(), w), lambda: T.embed(y, w.half()), lambda: T.embed(y, w.view(2, 2, 3)),
        lambda: T.embed(y, w, padding_idx=4), lambda: T.embed(y, w, scale=math.inf), lambda: T.embed(y.cpu(), w),
        lambda: T.gated_linear(x16.float(), w16), lambda: T.gated_linear(x16, w16[:7]), lambda: T.gated_linear(x16, w16[:, :5]),
        lambda: T.gated_linear(x16, w16, activation="tanh"), lambda: T.gated_mlp(x16, w16, wo16[:, :3]),
        lambda: T.gated_mlp(x16, w16, wo16.float()), lambda: T.token_log_probs(z, y, top_k=6), lambda: T.token_log_probs(z, y, top_k=-1),
        lambda: T.token_log_probs(z, y, temperature=0.0), lambda: T.token_log_probs(z, y, temperature=math.nan),
        lambda: T.token_log_probs(z, y[:1]), lambda: T.token_log_probs(z.double(), y), lambda: T.token_log_probs(z, y.float()),
        lambda: T.distill_loss(z, two.long(), two[:1]), lambda: T.distill_loss(z, two, two), lambda: T.distill_loss(z, two.long(), two.half()),
        lambda: T.distill_loss(z, two.long(), two, temperature=-1.0), lambda: T.distill_loss(z, two.long(), two, reduction="max"),
        lambda: T.distill_loss(z, two.long(), two, weight=torch.ones(3, device="xdna")), lambda: T.distill_loss(z, two.long(), two, weight=torch.ones(2)),
        lambda: T.distill_loss(z, torch.zeros(2, 1025, dtype=torch.long, device="xdna"), torch.zeros(2, 1025, device="xdna")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was taken")
    zx = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad(T.token_log_probs(zx, y).entropy.sum(), [zx], retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(T.token_log_probs(zx, y).entropy.sum(), [zx], create_graph=True)


LARGE = [  # rows, K, F, N: up to the largest tiles' sizes (both kernels of the last), ragged at the edges
    (4000, 264, 1000, 264), (2049, 72, 4104, 40), (300, 1024, 16384, 64), (8200, 512, 512, 1024), (4104, 200, 4000, 520),
]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("M,K,F,N", LARGE)
def test_gated_mlp_large(T, M, K, F, N, act):
    """The large tiles: sampled rows and units against the 64-bit block (each row of y, h and dx
    depends on its own row of x and dy only), the weight gradients against the products of the
    kernels' own bf16 operands."""
    print("gated large", M, K, F, N, act, flush=True)
    g = gen(M + K + F)
    x, dy = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, N, generator=g).bfloat16()
    w = (torch.randn(2 * F, K, generator=g) / math.sqrt(K)).bfloat16()
    wo = (torch.randn(N, F, generator=g) / math.sqrt(F)).bfloat16()
    rows = torch.unique(torch.cat([torch.arange(0, M, 97), torch.arange(max(0, M - 20), M)]))
    ref = gated_reference(x[rows], w, wo, dy[rows], act, True)
    leaves = [t.to("xdna").requires_grad_() for t in (x, w, wo)]
    y = T.gated_mlp(*leaves, activation=act)
    dx, dw, dwo = torch.autograd.grad(y, leaves, dy.to("xdna"))
    close(y.detach().cpu()[rows], *ref["y"], "y")
    close(dx.cpu()[rows], *ref["dx"], "dx")
    with torch.no_grad():
        h = T.gated_linear(leaves[0], leaves[1], activation=act)
    close(h.cpu()[rows], *ref["h"], "h")
    units = torch.unique(torch.cat([torch.arange(0, F, 131), torch.arange(F - 9, F)]))
    some = gated_reference(x, torch.cat([w[units], w[F + units]]), wo[:, units], dy, act, True)
    close(dw.cpu()[torch.cat([units, F + units])], *some["dw_in"], "dw_in")
    close(dwo.cpu()[:, units], *some["dw_out"], "dw_out")


@pytest.mark.parametrize("n,V,D", [(16384, 90, 200), (16385, 90, 200), (40000, 5, 70), (70000, 1 << 18, 12), (3000, 1, 600), (100, 100000, 2)])
def test_embedding_gradient_of_long_runs_and_both_orders(T, n, V, D):
    """Around the size where the order's kernels change, few ids (runs over many chunks), many ids."""
    print("embedding runs", n, V, D, flush=True)
    g = gen(n + V)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[: n // 2] = V // 2
    dy = torch.randn(n, D, generator=g).bfloat16()
    w = torch.zeros(V, D, dtype=BF16, device="xdna", requires_grad=True)
    (dw,) = torch.autograd.grad(T.embed(ids.to("xdna"), w), [w], dy.to("xdna"))
    ref = torch.zeros(V, D, dtype=F64).index_add_(0, ids, dy.to(F64))
    mag = torch.zeros(V, D, dtype=F64).index_add_(0, ids, dy.to(F64).abs())
    count = torch.bincount(ids, minlength=V).to(F64)[:, None]
    close(dw, ref, (count + 2) * U * mag + B * ref.abs(), "gradient")


@pytest.mark.parametrize("P,Q,K", [(692, 400, 1999), (131, 77, 700), (64, 300, 2600), (7, 5, 900), (200, 140, 9), (1030, 520, 130), (130, 3000, 5)])
@pytest.mark.parametrize("modes", [(0, 0), (1, 0), (1, 1)])
def test_tile_product(hip, stream, P, Q, K, modes):
    """The gated block's plain products in every layout: odd strides and addresses, k split over the
    grid or not, ragged ends of each direction."""
    from xdna_train import hip_abi
    print("tile product", P, Q, K, modes, flush=True)
    g = gen(P + Q + K)
    p, q = torch.randn(P, K, generator=g).bfloat16(), torch.randn(Q, K, generator=g).bfloat16()

    def laid(t, rows, pad, offset):
        m = t.t() if rows else t
        buf = torch.full((m.shape[0] * (m.shape[1] + pad) + offset + 8,), 9.0, device="cuda", dtype=BF16)
        v = torch.as_strided(buf, m.shape, (m.shape[1] + pad, 1), offset)
        v.copy_(m)
        return v, m.shape[1] + pad

    pv, ldp = laid(p, modes[0], 3, 1)
    qv, ldq = laid(q, modes[1], 2, 3)
    out = torch.full((Q, P + 1), 5.0, device="cuda", dtype=BF16)
    rc = hip.xdna_tile_mm_bf16(pv.data_ptr(), ldp, modes[0], qv.data_ptr(), ldq, modes[1], P, Q, K, out.data_ptr(), P + 1, stream)
    assert rc == 0, hip_abi.last_error()
    ref = q.to(F64) @ p.to(F64).t()
    close(out[:, :P], ref, (K + 8) * U * (q.to(F64).abs() @ p.to(F64).abs().t()) + B * ref.abs() + 1e-30, "product")
    assert (out[:, P].cpu() == 5.0).all(), "stored past a row's end"


@pytest.mark.parametrize("M,K,F,N", [(1, 1, 1, 1), (3, 5, 2, 4), (7, 40, 3, 9), (9, 130, 700, 0), (129, 64, 65, 63), (333, 500, 217, 500),
                                     (65, 200, 900, 3), (2000, 515, 260, 130), (1201, 300, 700, 301)])
@pytest.mark.parametrize("pad", [0, 3])
def test_gated_gradients_in_one_launch(hip, stream, M, K, F, N, pad):
    """dx, dw_in and dw_out from one launch, whatever the rule would choose: narrow and wide tiles,
    operands shorter than a vector, rows with padding, without dw_out."""
    from xdna_train import hip_abi
    print("gated gradients", M, K, F, N, pad, flush=True)
    g = gen(M + K + F)

    def rows(r, c, p):
        v = torch.as_strided(torch.full((r * (c + p),), 9.0, device="cuda", dtype=BF16), (r, c), (c + p, 1))
        return v.copy_(torch.randn(r, c, generator=g).bfloat16())

    dgu, h, x, w, dy = rows(M, 2 * F, 0), rows(M, F, 0), rows(M, K, pad), rows(2 * F, K, pad), rows(M, max(N, 1), pad)
    dx, dwi, dwo = (torch.full(s, 5.0, device="cuda", dtype=BF16) for s in ((M, K), (2 * F, K), (max(N, 1), F)))
    rc = hip.xdna_gated_grads_bf16(dgu.data_ptr(), x.data_ptr(), K + pad, w.data_ptr(), K + pad, dy.data_ptr(), max(N, 1) + pad,
                                   h.data_ptr(), M, K, F, N, dx.data_ptr(), dwi.data_ptr(), dwo.data_ptr(), stream)
    assert rc == 0, hip_abi.last_error()
    d = [t.cpu().to(F64) for t in (dgu, x, w, dy, h)]
    pairs = [(dx, d[0], d[2]), (dwi, d[0].t(), d[1])] + ([(dwo, d[3].t(), d[4])] if N else [])
    for out, a, b in pairs:
        close(out, a @ b, (a.shape[1] + 8) * U * (a.abs() @ b.abs()) + B * (a @ b).abs() + 1e-30, "product")
    assert N or (dwo.cpu() == 5.0).all()


def test_offsets_past_32_bits(T):
    """More than 2^31 elements in the logits, the table, its gradient and the block's projections: the
    last rows against the first, which hold the same values."""
    rows, V = 17000, 131072
    z = torch.randn(1, V, generator=gen(1)).bfloat16().to("xdna").expand(rows, V).contiguous().requires_grad_()
    y = torch.full((rows,), 77, device="xdna")
    r = T.token_log_probs(z, y, top_k=3)
    for t in (r.log_probs, r.entropy, r.top_log_probs, r.top_ids):
        assert torch.equal(t[-1], t[0]) and torch.equal(t[rows // 2], t[0])
    (dz,) = torch.autograd.grad([r.log_probs, r.entropy], [z], [torch.ones(rows, device="xdna")] * 2)
    assert torch.equal(dz[-1], dz[0]) and dz[0].any().item()
    ids = torch.tensor([[5, V - 1]], device="xdna").expand(rows, 2)
    each = T.distill_loss(z, ids, torch.zeros(rows, 2, device="xdna"), reduction="none")
    (dz,) = torch.autograd.grad(each.sum(), [z])
    assert torch.equal(each[-1], each[0]) and torch.equal(dz[-1], dz[0]) and dz[0].any().item()
    del z, r, dz
    V, D = 1050000, 2056
    w = torch.zeros(V, D, device="xdna", dtype=BF16)
    w[V - 2] = torch.randn(D, generator=gen(2)).bfloat16().to("xdna")
    w.requires_grad_()
    x = T.embed(torch.tensor([V - 2, 3], device="xdna"), w, scale=2.0)
    assert torch.equal(x[0], w[V - 2].detach() * 2) and not x[1].any().item()
    dy = torch.randn(2, D, generator=gen(3)).bfloat16().to("xdna")
    (dw,) = torch.autograd.grad(x, [w], dy)
    assert torch.equal(dw[V - 2], dy[0] * 2) and torch.equal(dw[3], dy[1] * 2) and not dw[V - 1].any().item()
    del w, x, dw
    M, K, F = 270000, 8, 4096
    x = torch.randn(1, K, generator=gen(4)).bfloat16().to("xdna").expand(M, K).contiguous().requires_grad_()
    wi = torch.randn(2 * F, K, generator=gen(5)).bfloat16().to("xdna")
    h = T.gated_linear(x, wi)
    assert torch.equal(h[-1], h[0]) and h[0].any().item()
    dh = torch.randn(1, F, generator=gen(6)).bfloat16().to("xdna").expand(M, F)
    (dx,) = torch.autograd.grad(h, [x], dh)
    assert torch.equal(dx[-1], dx[0]) and dx[0].any().item()


@pytest.mark.parametrize("kind", ["equal", "falling", "rising", "stride", "few", "zeros", "barred"])
@pytest.mark.parametrize("V", [3, 9, 1001, 5001, 20000, 20001, 69999])
def test_rows_at_odd_addresses_between_nan(T, V, kind):
    """Rows that start and end inside a word, with NaN on both sides: none of it may be seen."""
    print("odd rows", V, kind, flush=True)
    k = min(V, 40)
    z = torch.stack([order_rows(V, kind, gen(V + i)) for i in range(3)]).bfloat16()
    y = torch.tensor([0, V - 1, V // 2])
    base = torch.full((3, V + 2), math.nan, dtype=BF16)
    base[:, 1:V + 1] = z
    zx = base.to("xdna")[:, 1:V + 1].detach().requires_grad_()
    assert zx.stride(0) == V + 2
    r = T.token_log_probs(zx, y.to("xdna"), top_k=k)
    lp, h, tlp, tid, _, _ = logprob_reference(z, y, 1.0, k)
    assert torch.equal(r.top_ids.cpu(), tid)
    close(r.top_log_probs, tlp, tol_log(tlp), "top")
    close(r.log_probs, lp, tol_log(lp), "log_probs")
    close(r.entropy, h, 4 * U * 304 * (1 + h), "entropy")
    if kind != "barred":
        each = T.distill_loss(zx, y[:, None].to("xdna"), torch.zeros(3, 1, device="xdna"), reduction="none")
        close(each, -lp, tol_log(lp), "loss")


def test_forward_mode_is_refused(T):
    """A tangent that the operators cannot carry on raises, whether or not the tensor also takes part
    in a backward pass, and under no_grad too."""
    import torch.autograd.forward_ad as fw

    x, w, wo = (torch.randn(*s, generator=gen(1)).bfloat16().to("xdna") for s in ((3, 8), (12, 8), (5, 6)))
    z, table = (torch.randn(*s, generator=gen(2)).to("xdna") for s in ((3, 20), (7, 4)))
    y, ids, t = torch.tensor([1, 2, 3], device="xdna"), torch.tensor([[1], [2], [3]], device="xdna"), torch.zeros(3, 1, device="xdna")
    calls = [
        (table, lambda d: T.embed(y, d)), (x, lambda d: T.gated_linear(d, w)), (w, lambda d: T.gated_linear(x, d)),
        (x, lambda d: T.gated_mlp(d, w, wo)), (wo, lambda d: T.gated_mlp(x, w, d)), (z, lambda d: T.token_log_probs(d, y, top_k=2)),
        (z, lambda d: T.distill_loss(d, ids, t)), (t, lambda d: T.distill_loss(z, ids, d)), (t[:, 0], lambda d: T.distill_loss(z, ids, t, weight=d)),
        (z[:0], lambda d: T.token_log_probs(d, y[:0])),
    ]
    for i, (leaf, call) in enumerate(calls):
        for grad in (False, True):
            with fw.dual_level():
                dual = fw.make_dual(leaf.clone().requires_grad_(grad), torch.ones_like(leaf))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
                    pytest.fail(f"call {i} lost a tangent")
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)
    with fw.dual_level():  # no tangent among the operands: nothing to lose
        assert T.embed(y, table).shape == (3, 4)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("tau,gh", [(1e-2, 65536.0), (1e-3, 400.0), (1e-4, 4.0), (1e-9, 1.0), (1.0, 2.0 ** 40)])
def test_entropy_gradient_of_masked_tokens_stays_finite(T, tau, gh, mask, dtype):
    """Masked tokens have probability 0 and gradient 0, however far below the maximum they are in units
    of the temperature and however large the incoming gradient is.  The logits are of the temperature's
    size, so that no other probability underflows."""
    print("masked gradient", tau, gh, mask, dtype, flush=True)
    rows, V = 3, 3001
    z = tau * 3 * torch.randn(rows, V, generator=gen(70))
    barred = torch.rand(rows, V, generator=gen(71)) < 0.5
    barred[:, 5] = False
    z = z.masked_fill(barred, -math.inf if mask == "inf" else torch.finfo(dtype).min).to(dtype)
    y = torch.full((rows,), 5)
    zx = z.to("xdna").requires_grad_()
    r = T.token_log_probs(zx, y.to("xdna"), temperature=tau)
    (dz,) = torch.autograd.grad([r.log_probs, r.entropy], [zx], [torch.ones(rows, device="xdna"), torch.full((rows,), gh, device="xdna")])
    t32 = float(torch.tensor(tau, dtype=F32))
    _, h, _, _, q, lq = logprob_reference(z, y, t32, 1)
    assert not dz.cpu()[barred].any(), "a masked token has a gradient"
    hot = torch.nn.functional.one_hot(y, V).to(F64)
    lqf = torch.where(q > 0, lq, torch.zeros_like(lq))
    ref = (hot - q - gh * q * (lqf + h[:, None])) / t32
    terms = (hot + q + gh * q * (1 + lqf.abs() + h[:, None])) / t32
    close(dz, ref, grad_tol(terms, ref, dtype, lqf), "gradient")


@pytest.mark.parametrize("V", [100, 40000])  # whole rows; pieces and their join
def test_distillation_entries_outside_the_vocabulary(T, V):
    """An entry of logit -inf is absent whatever its id; one that is present makes its row's loss NaN
    and takes the row out of the gradient, and of the other rows' share."""
    z = torch.randn(3, V, generator=gen(90))
    ids = torch.tensor([[1, V, 3], [4, V + 7, 6], [7, 8, -1]])
    t = torch.tensor([[0.5, -math.inf, 1.0], [0.0, -math.inf, -math.inf], [1.0, 0.0, 2.0]])
    w = torch.tensor([0.5, 1.0, 2.0])
    zx = z.to("xdna").requires_grad_()
    loss = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"))
    rows, mag, dz, terms = distill_reference(z, torch.where(ids < V, ids, torch.full_like(ids, -1)), t, 1.0, w, "mean")
    close(loss, rows.sum(), 128 * U * mag.sum(), "loss with absent entries")
    (got,) = torch.autograd.grad(loss, [zx])
    close(got, dz, grad_tol(2 * terms, dz, F32, torch.log_softmax(z.to(F64), 1)), "gradient with absent entries")
    t[1, 1] = 0.0  # present now
    each = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"), reduction="none")
    assert torch.isnan(each[1]).item() and torch.isfinite(each[::2]).all().item()
    (got,) = torch.autograd.grad(each, [zx], torch.ones(3, device="xdna"))
    _, _, dz, terms = distill_reference(z, torch.where(ids < V, ids, torch.full_like(ids, -1)), t, 1.0, w * torch.tensor([1.0, 0.0, 1.0]), "none")
    assert not got[1].cpu().any(), "a row of a NaN loss has a gradient"
    close(got, dz, grad_tol(2 * terms, dz, F32, torch.log_softmax(z.to(F64), 1)), "gradient beside an invalid row")
    mean = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"))
    assert torch.isnan(mean).item()
    (got,) = torch.autograd.grad(mean, [zx])
    _, _, dz, terms = distill_reference(z, torch.where(ids < V, ids, torch.full_like(ids, -1)), t, 1.0, w * torch.tensor([1.0, 0.0, 1.0]), "mean")
    close(got, dz, grad_tol(2 * terms, dz, F32, torch.log_softmax(z.to(F64), 1)), "mean's gradient beside an invalid row")


def test_distillation_of_a_token_named_twice(T):
    """The loss is a sum over the entries, each with its own p; the gradient's target is the sum of a
    token's entries, so that it is the gradient of the row with these entries as one."""
    V = 60
    z = torch.randn(2, V, generator=gen(80))
    ids, t = torch.tensor([[7, 3, 7], [9, 9, 9]]), torch.tensor([[0.5, 1.0, -0.25], [0.0, 0.0, 0.0]])
    zx = z.to("xdna").requires_grad_()
    each = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), reduction="none")
    lq = torch.log_softmax(z.to(F64), 1)
    lp = torch.log_softmax(t.to(F64), 1)
    terms = lp.exp() * (lp - lq.gather(1, ids))
    mag = (lp.exp() * (lp.abs() + lq.gather(1, ids).abs() + 1)).sum(1)
    close(each, terms.sum(1), 128 * U * mag, "loss by entries")
    (dz,) = torch.autograd.grad(each.sum(), [zx])
    target = torch.zeros(2, V, dtype=F64).scatter_add_(1, ids, lp.exp())
    ref = lq.exp() - target
    close(dz, ref, grad_tol(lq.exp() + target, ref, F32, lq), "gradient")
    one_ids = torch.tensor([[7, 3, -1], [9, -1, -1]])
    one_t = torch.where(one_ids >= 0, target.gather(1, one_ids.clamp(min=0)).log(), torch.zeros(2, 3, dtype=F64)).float()
    one = T.distill_loss(zx, one_ids.to("xdna"), one_t.to("xdna"), reduction="none")
    (dz1,) = torch.autograd.grad(one.sum(), [zx])
    close(dz1, ref, grad_tol(lq.exp() + target, ref, F32, lq), "gradient of the joined entries")


def test_gradient_of_a_barred_target(T):
    """The target's own logit has the derivative of a log-softmax also where it is -inf; other masked
    tokens have none, and neither has the row of a target past the vocabulary."""
    V, tau = 300, 0.5
    z = torch.randn(3, V, generator=gen(72))
    z[0, ::2] = -math.inf
    y = torch.tensor([4, 5, V])  # barred in row 0
    zx = z.to("xdna").requires_grad_()
    r = T.token_log_probs(zx, y.to("xdna"), temperature=tau)
    assert r.log_probs.detach().cpu()[0] == -math.inf
    (dz,) = torch.autograd.grad(r.log_probs, [zx], torch.tensor([3.0, 1.0, 1.0], device="xdna"))
    dz = dz.cpu()
    assert dz[0, 4] == 3.0 / tau
    dz[0, 4] = 0.0
    assert not dz[0, ::2].any() and (dz[0, 1::2] < 0).all()
    assert torch.isnan(r.log_probs.detach().cpu()[2]) and dz[1].any() and not dz[2].any()


@pytest.mark.parametrize("tau", [4.5e-39, 1e-30, 1e-10, 1e10, 1e30])
def test_temperatures_at_the_ends_of_the_range(T, tau):
    """Logits of the temperature's size: at any temperature the same distribution, and a loss of
    temperature**2 times the divergence where that is an fp32 number."""
    t32 = float(torch.tensor(tau, dtype=F32))
    V = 40
    z = torch.randn(2, V, generator=gen(95)) * tau
    t = torch.randn(2, 3, generator=gen(96)) * tau
    y, ids = torch.tensor([3, 7]), torch.tensor([[1, 2, 3], [4, 5, 6]])
    r = T.token_log_probs(z.to("xdna"), y.to("xdna"), temperature=tau)
    lp, h, _, _, _, _ = logprob_reference(z, y, t32, 1)
    # the smallest ones have few bits left: an input's own grain is 2^-149, and so is 1 / tau's
    grain = 16 * 2.0 ** -149 / t32 + (16 * 2.0 ** -149 * t32)
    close(r.log_probs, lp, tol_log(lp) + grain, "log_probs")
    close(r.entropy, h, 4 * U * 304 * (1 + h) + 4 * grain, "entropy")
    if 1e-18 < tau < 1e18:
        each = T.distill_loss(z.to("xdna"), ids.to("xdna"), t.to("xdna"), temperature=tau, reduction="none")
        per_row, mag, _, _ = distill_reference(z, ids, t, t32, torch.ones(2), "none")
        close(each, per_row, 128 * U * mag, "row losses")
    with pytest.raises(RuntimeError, match="temperature"):
        T.token_log_probs(z.to("xdna"), y.to("xdna"), temperature=4e-39)


def test_distillation_loss_of_a_temperature_whose_square_underflows(T):
    tau, V = 1e-25, 12
    t32 = float(torch.tensor(tau, dtype=F32))
    z, t = torch.randn(2, V, generator=gen(97)), torch.randn(2, 3, generator=gen(98))
    z[:, 0] += 10.0  # the student's token, none of the teacher's
    ids = torch.tensor([[1, 2, 3], [4, 5, 6]])
    each = T.distill_loss(z.to("xdna"), ids.to("xdna"), t.to("xdna"), temperature=tau, reduction="none")
    per_row, mag, _, _ = distill_reference(z, ids, t, t32, torch.ones(2), "none")
    close(each, per_row, 128 * U * mag, "row losses")
    assert (each.cpu() > 0).all()


@pytest.mark.parametrize("M", [1, 70, 300])  # the kernels of few rows, and of tiles
def test_gelu_keeps_its_lower_tail(T, M):
    """gelu(g) = g Phi(g) relative to its own size where Phi is far below an fp32 ulp of 1.  A relative
    error e of erfc's argument x = g / sqrt 2 is one of 2 x^2 e = g^2 e of the tail, the exponential of
    -g^2 / 2 has the same, and each function is within 16 u of its argument's value; then the roundings:
    h, or dg and the product that hands it out."""
    g = -torch.linspace(2.0, 12.0, 161).bfloat16().float()
    F = g.numel()
    x = torch.zeros(M, 8)
    x[:, 0] = 1.0
    w = torch.zeros(2 * F, 8)
    w[:F, 0], w[F:, 0] = g, 1.0
    xd, wd = x.bfloat16().to("xdna").requires_grad_(), w.bfloat16().to("xdna").requires_grad_()
    h = T.gated_linear(xd, wd, activation="gelu")
    a, da = act64("gelu", g.to(F64))
    rel = (2 * g.to(F64) ** 2 + 64) * U
    close(h, a.expand(M, F), ((rel + B) * a.abs()).expand(M, F), "gelu")
    dh = torch.zeros(M, F)
    dh[M - 1] = 1.0  # one row: dw_in's first column is its dg
    (dw,) = torch.autograd.grad(h, [wd], dh.bfloat16().to("xdna"))
    pdf = torch.exp(-0.5 * g.to(F64) ** 2) / math.sqrt(2 * math.pi)
    close(dw[:F, 0], da, (rel * (da.abs() + 2 * g.to(F64).abs() * pdf) + 2.1 * B * da.abs()), "gelu's derivative")
    close(dw[F:, 0], a, (rel + 2.1 * B) * a.abs(), "du")


def kept_parts(gu, M, F):
    """g and u from the buffer that the backward reads, in 64 bits."""
    hi = gu[: M * F * 4].view(torch.int16).view(M, 2 * F).cpu().to(torch.int32) << 16
    low = gu[M * F * 4:].view(M, F).cpu().to(torch.int32)
    g = (hi[:, :F] | ((low & 15) << 12)).view(F32).to(F64)
    u = (hi[:, F:] | ((low >> 4) << 12)).view(F32).to(F64)
    return g, u


@pytest.mark.parametrize("M,K,F", [(1, 8, 64), (1, 24, 37), (16, 8, 50), (33, 16, 65), (64, 40, 96), (65, 24, 64), (70, 9, 61), (130, 5, 66),
                                   (1000, 16, 516), (1300, 24, 1031), (2048, 16, 4096), (2050, 8, 4104), (4000, 8, 4104)])
def test_kept_projections_hold_20_bits(hip, stream, M, K, F):
    """What the forward keeps of g and u, by itself: a bf16 and 4 more bits are half an ulp of 2^-11 from
    the sum, which is (K + 8) u of its terms from the exact one.  Few rows, both tiles, the large tiles."""
    from xdna_train import hip_abi
    print("kept", M, K, F, flush=True)
    g = gen(M + K + F)
    x, w = torch.randn(M, K, generator=g).bfloat16(), torch.randn(2 * F, K, generator=g).bfloat16()
    xd, wd = x.cuda(), w.cuda()
    h = torch.zeros(M, F, device="cuda", dtype=BF16)
    size = hip.xdna_gated_kept_bytes(M, F)
    gu = torch.full((size + 16,), 0x5A, device="cuda", dtype=torch.uint8)
    rc = hip.xdna_gated_bf16(xd.data_ptr(), K, wd.data_ptr(), K, M, K, F, 0, h.data_ptr(), gu.data_ptr(), stream)
    assert rc == 0, hip_abi.last_error()
    got = kept_parts(gu[:size], M, F)
    assert (gu[size:].cpu() == 0x5A).all(), "stored past the end"
    for part, rows, what in ((got[0], w[:F], "g"), (got[1], w[F:], "u")):
        ref = x.to(F64) @ rows.to(F64).t()
        close(part, ref, 2.0 ** -12 * ref.abs() + (K + 8) * U * (x.to(F64).abs() @ rows.to(F64).abs().t()), what)


@pytest.mark.parametrize("form,M,F", [("linear", 5, 64), ("linear", 7, 37), ("linear", 33, 66), ("block", 5, 64), ("block", 70, 37), ("block", 300, 1031),
                                      ("block", 2000, 2000), ("block", 4096, 4096), ("block", 4401, 4872)])
def test_kept_projections_are_read_in_20_bits(hip, stream, form, M, F):
    """The backward of a buffer of known bits.  With relu, dh = 1 and positive g the result is [u, g],
    rounded once from their 20 bits: exact."""
    from xdna_train import hip_abi
    print("kept bits", form, M, F, flush=True)
    g = gen(M + F)
    bits = torch.randint(0x3F000, 0x41000, (2, M, F), generator=g, dtype=torch.int32)  # 0.5 .. 8 by 2^-11 of themselves
    bits[1] |= torch.randint(0, 2, (M, F), generator=g, dtype=torch.int32) << 19           # u of both signs
    hi = torch.cat([bits[0] >> 4, bits[1] >> 4], 1)
    low = (bits[0] & 15) | ((bits[1] & 15) << 4)
    gu = torch.cat([hi.to(torch.int64).to(torch.uint16).view(torch.uint8).flatten(), low.to(torch.uint8).flatten()]).cuda()
    assert gu.numel() == hip.xdna_gated_kept_bytes(M, F)
    out = torch.zeros(M, 2 * F, device="cuda", dtype=BF16)
    if form == "linear":
        dh = torch.ones(M, F, device="cuda", dtype=BF16)
        rc = hip.xdna_gated_bwd_bf16(dh.data_ptr(), F, gu.data_ptr(), M, F, 2, out.data_ptr(), stream)
    else:
        N = 8
        dy, wo = torch.zeros(M, N, device="cuda", dtype=BF16), torch.zeros(N, F, device="cuda", dtype=BF16)
        dy[:, 3] = 1
        wo[3] = 1
        rc = hip.xdna_gated_mlp_bwd_bf16(dy.data_ptr(), N, wo.data_ptr(), F, gu.data_ptr(), M, N, F, 2, out.data_ptr(), stream)
    assert rc == 0, hip_abi.last_error()
    value = (bits << 12).view(F32).bfloat16()
    assert torch.equal(out[:, :F].cpu(), value[1]) and torch.equal(out[:, F:].cpu(), value[0])


def gpu_reference(z, y, tau, k):
    """logprob_reference of many rows, on the GPU in 64 bits (-0 as +0: they are equal)."""
    return [t.cpu() for t in logprob_reference(z.cuda().to(F64) + 0.0, y.cuda(), tau, k)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,V,k", [(255, 40000, 8), (300, 70001, 64), (383, 70000, 5), (130, 131071, 40)])
def test_log_probs_of_hundreds_of_rows_in_pieces(T, rows, V, k, dtype):
    """Just below the row counts that take whole rows: pieces and their join."""
    print("pieces", rows, V, k, dtype, flush=True)
    z, zx = make_logits(rows, V, dtype, rows, masked=0.2, extra=3)
    z[3] = order_rows(V, "equal", gen(1)).to(dtype)
    z[4] = order_rows(V, "stride", gen(2)).to(dtype)
    z[5] = order_rows(V, "few", gen(3)).to(dtype)
    with torch.no_grad():
        zx.copy_(z)
    y = torch.randint(0, V, (rows,), generator=gen(6))
    r = T.token_log_probs(zx.detach(), y.to("xdna"), top_k=k)
    lp, h, tlp, tid, _, _ = gpu_reference(z, y, 1.0, k)
    close(r.log_probs, lp, tol_log(lp), "log_probs")
    close(r.entropy, h, 4 * U * 304 * (1 + h), "entropy")
    assert torch.equal(r.top_ids.cpu(), tid)
    close(r.top_log_probs, tlp, tol_log(tlp), "top")


def test_distillation_of_hundreds_of_rows_in_pieces(T):
    rows, V, k = 255, 40000, 70
    g = gen(7)
    z, zx = make_logits(rows, V, BF16, 8, extra=1)
    ids, t, w = torch.randint(0, V, (rows, k), generator=g), 4 * torch.randn(rows, k, generator=g), torch.rand(rows, generator=g)
    ids[torch.rand(rows, k, generator=g) < 0.2] = -1
    loss = T.distill_loss(zx, ids.to("xdna"), t.to("xdna"), weight=w.to("xdna"))
    per_row, mag, dz, terms = distill_reference(z, ids, t, 1.0, w, "mean")
    close(loss, per_row.sum(), 128 * U * mag.sum(), "loss")
    (got,) = torch.autograd.grad(loss, [zx])
    close(got, dz, grad_tol(2 * terms, dz, BF16, torch.log_softmax(z.to(F64), 1)), "gradient")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("V", [2049, 4097, 6001, 6144, 6145])
@pytest.mark.parametrize("k", [0, 5, 64])
def test_log_probs_of_many_short_rows(T, V, k, dtype):
    """Rows that one wave takes (up to 6144 tokens from 1024 rows on), over a step of it and a tail, the
    selection in more than one round; special orders among them, odd row strides."""
    print("short rows", V, k, dtype, flush=True)
    rows, tau = 1031, 0.9
    z, zx = make_logits(rows, V, dtype, V, masked=0.3, extra=V % 4 + 1)
    for i, kind in enumerate(("equal", "falling", "rising", "stride", "few", "zeros", "barred")):
        z[i] = z[rows - 1 - i] = order_rows(V, kind, gen(i)).to(dtype)
    with torch.no_grad():
        zx.copy_(z)
    y = torch.randint(0, V, (rows,), generator=gen(V))
    y[::7] = -1
    r = T.token_log_probs(zx, y.to("xdna"), top_k=k, temperature=tau)
    t32 = float(torch.tensor(tau, dtype=F32))
    lp, h, tlp, tid, q, lq = gpu_reference(z, y, t32, k)
    close(r.log_probs, lp, tol_log(lp), "log_probs")
    close(r.entropy, h, 4 * U * (64 + 8 * 400 / tau) * (1 + h), "entropy")
    assert torch.equal(r.top_ids.cpu(), tid)
    close(r.top_log_probs, tlp, tol_log(tlp), "top")


def test_gated_block_of_the_most_rows(T):
    """2^22 rows are taken and one more is not: the first and the last rows, which hold the same values."""
    M, K, F = 1 << 22, 2, 3
    x = torch.randn(64, K, generator=gen(99)).bfloat16().to("xdna").repeat(M // 64, 1).requires_grad_()
    w, wo = torch.randn(2 * F, K, generator=gen(100)).bfloat16().to("xdna"), torch.randn(K, F, generator=gen(101)).bfloat16().to("xdna")
    y = T.gated_mlp(x, w, wo)
    (dx,) = torch.autograd.grad(y, [x], torch.ones(1, K, dtype=BF16, device="xdna").expand(M, K))
    for t in (y.detach(), dx):
        assert torch.equal(t[-64:], t[:64]) and t[:64].any().item()
    with pytest.raises(RuntimeError, match="too many rows"):
        T.gated_mlp(torch.zeros(M + 1, 1, dtype=BF16, device="xdna"), w[:, :1], wo)


def test_embedding_refuses_a_scale_past_fp32(T):
    """It would be infinite in the kernels, and the zeros of a row NaN."""
    w = torch.zeros(4, 3, device="xdna")
    for scale in (1e39, -1e300):
        with pytest.raises(RuntimeError, match="scale"):
            T.embed(torch.tensor([1], device="xdna"), w, scale=scale)
    assert not T.embed(torch.tensor([1], device="xdna"), w, scale=3e38).cpu().any()


def test_npu_modes_do_not_concern_the_functions(T):
    """They have one route: the same bits in every mode, from the same kernels."""
    import xdna_train

    g = gen(110)
    x, w, wo = (torch.randn(*s, generator=g).bfloat16().to("xdna").requires_grad_() for s in ((70, 64), (96, 64), (40, 48)))
    ids, t = torch.randint(0, 40, (70, 4), generator=g).to("xdna"), torch.randn(70, 4, generator=g).to("xdna")

    def step():
        y = T.gated_mlp(x, w, wo)
        loss = T.distill_loss(y, ids, t) - T.token_log_probs(y, ids[:, 0], top_k=3).log_probs.mean() + T.embed(ids, w).float().mean()
        return [y.detach(), *torch.autograd.grad(loss, [x, w, wo])]

    want = [v.cpu() for v in step()]
    before = xdna_train.npu_mode()
    try:
        for mode in (0, 1, 2):
            xdna_train.set_npu_mode(mode)
            xdna_train.reset_mapped_cpu_stats()
            got = [v.cpu() for v in step()]
            stats = xdna_train.mapped_cpu_stats()
            assert all(stats.get(f"hip_tokens.{k}.{d}.run", {}).get("calls", 0) > 0 for k in ("embed", "gated", "distill", "logprobs") for d in ("fwd", "bwd")), mode
            assert all(torch.equal(a, b) for a, b in zip(got, want)), mode
    finally:
        xdna_train.set_npu_mode(before)


@pytest.mark.parametrize("M,K,F,N", [(8192, 1024, 2048, 1024), (5000, 1024, 4096, 1024), (7000, 1024, 4096, 1024)])
def test_gated_gradients_on_both_sides_of_the_short_block(T, M, K, F, N):
    """One launch for the three gradients although the GEMM would take some of them, and beyond it."""
    test_gated_mlp_large(T, M, K, F, N, "silu")
