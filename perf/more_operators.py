"""Performance cases of a token model's block: layer norm, linear layer with its epilogue, decay attention.

Each case has two forms of one pass: the plain one (elementary torch operations in 32 bits, rounded once at the end) and the
call a user makes of ``xdna_train.tokens``.  ``own`` says which of them ``prepare`` and ``run`` take; ``exact`` gives the same
outputs from the definitions in 64 bits.

A case is a dict: "op" names the operator, "train" asks for gradients too, the rest are its sizes and options.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # one new token's residual sum and norm, at the MLP's width: only latency counts
        {"name": "add norm T1 D1024", "op": "norm", "train": False, "rows": 1, "dim": 1024, "dtype": "bf16", "add": True},
        # odd sizes in fp32: a small model's norm
        {"name": "norm train T4099 D515 f32", "op": "norm", "train": True, "rows": 4099, "dim": 515, "dtype": "f32", "add": False},
        # an ordinary training batch (8 sequences of 1024), the residual stream's sum with it
        {"name": "add norm train T8192 D1024", "op": "norm", "train": True, "rows": 8192, "dim": 1024, "dtype": "bf16", "add": True},
        # a large batch: 268 MB a tensor, far past the caches
        {"name": "norm train T65536 D2048", "op": "norm", "train": True, "rows": 65536, "dim": 2048, "dtype": "bf16", "add": False},
        # a projection back into the residual stream for one new token: the weight's bytes are the work
        {"name": "linear decode M1 4096-1024", "op": "linear", "train": False, "rows": 1, "width": 4096, "units": 1024, "act": "none", "bias": True,
         "residual": True},
        # a short ragged batch, nothing a multiple of a tile
        {"name": "linear train M333 1000-1367", "op": "linear", "train": True, "rows": 333, "width": 1000, "units": 1367, "act": "gelu", "bias": True,
         "residual": False},
        # a layer at the MLP benchmark's sizes with its ReLU, forward and backward
        {"name": "linear train M8192 1024-4096", "op": "linear", "train": True, "rows": 8192, "width": 1024, "units": 4096, "act": "relu", "bias": True,
         "residual": True},
        # one new token of one small sequence: latency
        {"name": "decay step B1 H8 D64", "op": "step", "train": False, "batch": 1, "heads": 8, "kv_heads": 8, "dk": 64, "dv": 64, "slots": 1},
        # a serving step: 64 sequences with their states in a pool of 80
        {"name": "decay step B64 H16 D128", "op": "step", "train": False, "batch": 64, "heads": 16, "kv_heads": 16, "dk": 128, "dv": 128, "slots": 80},
        # a long prompt behind a cached prefix: few heads, the length is the work; q, k and v are slices of one projection
        {"name": "decay prompt B1 T8192 H16 D128", "op": "decay", "train": False, "batch": 1, "tokens": 8192, "heads": 16, "kv_heads": 16, "dk": 128,
         "dv": 128, "ragged": False, "state": True},
        # a ragged batch, shared key heads, head sizes off the tiles
        {"name": "decay train B3 T777 H6/2 D48/80", "op": "decay", "train": True, "batch": 3, "tokens": 777, "heads": 6, "kv_heads": 2, "dk": 48, "dv": 80,
         "ragged": True, "state": True},
        # an ordinary training batch
        {"name": "decay train B8 T2048 H16 D128", "op": "decay", "train": True, "batch": 8, "tokens": 2048, "heads": 16, "kv_heads": 16, "dk": 128,
         "dv": 128, "ragged": False, "state": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "decay", "decay", "step"])
    train = rng.random() < 0.7
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        dim = _log_int(rng, 64, 4096) if rng.random() < 0.5 else 64 * rng.choice([1, 2, 4, 8, 12, 16, 32, 64])
        return {"op": op, "train": train, "rows": _log_int(rng, 1, min(65536, (1 << 27) // (dim * (2 if dtype == "f32" else 1)))), "dim": dim,
                "dtype": dtype, "add": rng.random() < 0.5}
    if op == "linear":
        few = rng.random() < 0.4  # serving steps beside training batches
        return {"op": op, "train": train and not few, "rows": _log_int(rng, 1, 64) if few else _log_int(rng, 65, 8192),
                "width": _log_int(rng, 128, 1024) if rng.random() < 0.5 else 64 * rng.randint(2, 16),
                "units": _log_int(rng, 128, 4096) if rng.random() < 0.5 else 128 * rng.choice([1, 2, 4, 7, 8, 11, 16, 32]),
                "act": rng.choice(["none", "silu", "gelu", "relu"]), "bias": rng.random() < 0.7, "residual": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2])
    dk, dv = [rng.choice([32, 64, 64, 128, 128, rng.randint(16, 128)]) for _ in range(2)]
    if rng.random() < 0.6:
        dv = dk
    if op == "step":
        batch = _log_int(rng, 1, 128)
        return {"op": op, "train": False, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv, "slots": batch + rng.choice([0, 0, 5])}
    batch = _log_int(rng, 1, 8)
    return {"op": op, "train": train, "batch": batch, "tokens": _log_int(rng, 2, min(8192, 262144 // (batch * heads))), "heads": heads,
            "kv_heads": kv_heads, "dk": dk, "dv": dv, "ragged": rng.random() < 0.5, "state": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------
# Values
# ---------------------------------------------------------------------------------------
def _values(case, seed):
    """The pass's tensors on the GPU, by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bf16 = torch.bfloat16

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op = case["op"]
    if op == "norm":
        dt, r, d = DTYPES[case["dtype"]], case["rows"], case["dim"]
        # a residual stream: a few channels are large, means differ from row to row
        spread = 1.0 + 4.0 * (uniform(d) < 0.02).float()
        v = {"x": (normal(r, d) * spread + 0.3 * normal(r, 1)).to(dt), "weight": (1.0 + 0.1 * normal(d)).to(dt), "bias": (0.1 * normal(d)).to(dt)}
        if case["add"]:
            v["residual"] = (2.0 * normal(r, d)).to(dt)
        if case["train"]:
            v["dy"] = normal(r, d).to(dt)
            if case["add"]:
                v["dsum"] = normal(r, d).to(dt)
        return v
    if op == "linear":
        m, k, n = case["rows"], case["width"], case["units"]
        v = {"x": normal(m, k).to(bf16), "weight": ((2 * uniform(n, k) - 1) / math.sqrt(k)).to(bf16)}
        if case["bias"]:
            v["bias"] = ((2 * uniform(n) - 1) / math.sqrt(k)).to(bf16)
        if case["residual"]:
            v["residual"] = normal(m, n).to(bf16)
        if case["train"]:
            v["dy"] = normal(m, n).to(bf16)
        return v
    b, h, kv, dk, dv = case["batch"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
    # heads forget at rates from a few tokens to a few hundred
    v = {"log_decay": -torch.exp2(-1.0 - 8.0 * torch.arange(h, device="cuda") / h)}
    if op == "step":
        v |= {"q": normal(b, h, dk).to(bf16), "k": normal(b, kv, dk).to(bf16), "v": normal(b, kv, dv).to(bf16), "state": normal(case["slots"], h, dk, dv)}
        if case["slots"] > b:
            v["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:b]
        return v
    t = case["tokens"]
    qkv = normal(b, t, h * dk + kv * (dk + dv)).to(bf16)
    if case["train"]:
        q, k, w = torch.split(qkv, [h * dk, kv * dk, kv * dv], 2)
        v |= {"q": q.reshape(b, t, h, dk), "k": k.reshape(b, t, kv, dk), "v": w.reshape(b, t, kv, dv)}
        v |= {"dout": normal(b, t, h, dv).to(bf16)}
    else:
        v["qkv"] = qkv
    if case["state"]:
        v["state"] = 4.0 * normal(b, h, dk, dv)
        if case["train"]:
            v["dstate"] = 0.25 * normal(b, h, dk, dv)
    if case["ragged"]:
        v["lengths"] = torch.randint(t // 2, t + 1, (b,), generator=g, device="cuda")
    return v


def _tokens():
    path = str(Path(__file__).resolve().parent.parent / "pytorch-xdna2_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import xdna_train.tokens

    return xdna_train.tokens


def _learnt(case, v):
    """The tensors whose gradients a training pass returns."""
    names = {"norm": ["x", "residual", "weight", "bias"], "linear": ["x", "weight", "bias"], "decay": ["q", "k", "v", "state"]}[case["op"]]
    return [v[n] for n in names if n in v]


def prepare(case, seed):
    v = _values(case, seed)
    state = {"case": dict(case), "v": v}
    if own:
        state["tokens"] = _tokens()
        state["v"] = v = {n: t.to("xdna") for n, t in v.items()}
        if case["train"]:
            for t in _learnt(case, v):
                t.requires_grad_()
    return state


# ---------------------------------------------------------------------------------------
# run: the framework's calls
# ---------------------------------------------------------------------------------------
def _heads(case, qkv):
    """q, k and v as slices of one projection."""
    b, t, h, kv, dk, dv = qkv.size(0), qkv.size(1), case["heads"], case["kv_heads"], case["dk"], case["dv"]
    q, k, v = torch.split(qkv, [h * dk, kv * dk, kv * dv], 2)
    return q.view(b, t, h, dk), k.view(b, t, kv, dk), v.view(b, t, kv, dv)


def _own(case, v, T):
    op, train = case["op"], case["train"]
    if op == "norm":
        if case["add"]:
            r = T.add_layer_norm(v["x"], v["residual"], v["weight"], v["bias"], eps=EPS)
            out, grads = [r.norm, r.sum], ["dy", "dsum"]
        else:
            out, grads = [T.layer_norm(v["x"], v["weight"], v["bias"], eps=EPS)], ["dy"]
    elif op == "linear":
        out, grads = [T.linear(v["x"], v["weight"], v.get("bias"), activation=case["act"], residual=v.get("residual"))], ["dy"]
    elif op == "step":
        return [T.decay_attention_step(v["q"], v["k"], v["v"], v["log_decay"], v["state"], slots=v.get("slots"), scale=_scale(case)), v["state"]]
    else:
        q, k, w = (v["q"], v["k"], v["v"]) if train else _heads(case, v["qkv"])
        r = T.decay_attention(q, k, w, v["log_decay"], state=v.get("state"), lengths=v.get("lengths"), scale=_scale(case))
        out, grads = [r.out, r.state], ["dout", "dstate"] if case["state"] else ["dout"]
    if not train:
        return out
    return [o.detach() for o in out] + list(torch.autograd.grad(out[: len(grads)], _learnt(case, v), [v[n] for n in grads]))


def _scale(case):
    return case["dk"] ** -0.5


# ---------------------------------------------------------------------------------------
# run: the plain forms, in 32 bits
# ---------------------------------------------------------------------------------------
def _act(name, g):
    """(act(g), act'(g))"""
    if name == "none":
        return g, torch.ones_like(g)
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(g * -math.sqrt(0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    on = (g > 0).float()
    return g * on, on


def _plain_norm(case, v):
    dt, w, x = v["x"].dtype, v["weight"].float(), v["x"].float()
    out = []
    if case["add"]:  # the norm is that of the sum as it is stored
        total = (x + v["residual"].float()).to(dt)
        x = total.float()
        out = [total]
    d = x - x.mean(1, keepdim=True)
    inv = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * inv
    out.insert(0, (xh * w + v["bias"].float()).to(dt))
    if case["train"]:
        dy = v["dy"].float()
        a = dy * w
        dx = inv * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
        if case["add"]:
            dx = dx + v["dsum"].float()
        dx = dx.to(dt)
        out += ([dx, dx] if case["add"] else [dx]) + [(dy * xh).sum(0).to(dt), dy.sum(0).to(dt)]
    return out


def _plain_linear(case, v):
    dt = v["x"].dtype
    x, w = v["x"].float(), v["weight"].float()
    pre = x @ w.t()
    if case["bias"]:
        pre = pre + v["bias"].float()
    y, slope = _act(case["act"], pre)
    if case["residual"]:
        y = y + v["residual"].float()
    out = [y]
    if case["train"]:
        dp = v["dy"].float() * slope
        out += [dp @ w, dp.t() @ x] + ([dp.sum(0)] if case["bias"] else [])
    return [t.to(dt) for t in out]


def _plain_step(case, v):
    group = case["heads"] // case["kv_heads"]
    q, k, w = v["q"].float(), v["k"].float().repeat_interleave(group, 1), v["v"].float().repeat_interleave(group, 1)
    at = v["slots"] if "slots" in v else slice(None)
    s = v["state"][at] * torch.exp(v["log_decay"])[:, None, None] + k[..., None] * w[..., None, :]
    v["state"][at] = s
    return [(_scale(case) * (q[..., None] * s).sum(2)).to(v["q"].dtype), v["state"]]


def _chunks(x, n, c):
    """[B, T, H, D] as [B, H, n, c, D], zeros behind the last token."""
    b, t, h, d = x.shape
    return torch.cat([x, x.new_zeros(b, n * c - t, h, d)], 1).view(b, n, c, h, d).permute(0, 3, 1, 2, 4)


def _plain_decay(case, v, q, k, w, state):
    group, g = case["heads"] // case["kv_heads"], v["log_decay"]
    b, t, h, dk = q.shape
    dv = w.size(3)
    q, k, w = q.float(), k.float().repeat_interleave(group, 2), w.float().repeat_interleave(group, 2)
    at = torch.arange(t, device=q.device)
    length = v["lengths"] if case["ragged"] else torch.full((b,), t, device=q.device)
    inside = (at < length[:, None])[:, :, None, None].float()
    k, w = k * inside, w * inside
    c = min(128, t)
    n = -(-t // c)
    qc, kc, wc = _chunks(q, n, c), _chunks(k, n, c), _chunks(w, n, c)
    i, m = torch.arange(c, device=q.device), torch.arange(n, device=q.device)
    decay = torch.exp((i[:, None] - i).clamp(min=0) * g[:, None, None]) * (i[:, None] >= i)
    local = (kc * torch.exp((c - 1 - i) * g[:, None])[:, None, :, None]).transpose(3, 4) @ wc
    between = torch.exp(c * (m[:, None] - 1 - m).clamp(min=0) * g[:, None, None]) * (m[:, None] > m)
    start = (between @ local.reshape(b, h, n, dk * dv)).view(b, h, n, dk, dv)
    if state is not None:
        start = start + torch.exp(c * m * g[:, None])[:, :, None, None] * state[:, :, None]
    out = ((qc @ kc.transpose(3, 4)) * decay[:, None]) @ wc + torch.exp((i + 1) * g[:, None])[:, None, :, None] * (qc @ start)
    out = _scale(case) * out.permute(0, 2, 3, 1, 4).reshape(b, n * c, h, dv)[:, :t] * inside
    left = torch.exp((length[:, None] - 1 - at).clamp(min=0)[:, :, None] * g)
    last = (k * left[..., None]).permute(0, 2, 3, 1) @ w.permute(0, 2, 1, 3)
    if state is not None:
        last = last + torch.exp(length[:, None] * g)[:, :, None, None] * state
    return out.to(torch.bfloat16), last


def _plain(case, v):
    op = case["op"]
    if op == "norm":
        return _plain_norm(case, v)
    if op == "linear":
        return _plain_linear(case, v)
    if op == "step":
        return _plain_step(case, v)
    if not case["train"]:
        return list(_plain_decay(case, v, *_heads(case, v["qkv"]), v.get("state")))
    # (the gradients of the elementary operations, in 32 bits)
    leaves = [t.detach().float().requires_grad_() for t in _learnt(case, v)]
    with torch.enable_grad():
        out, last = _plain_decay(case, v, *leaves[:3], leaves[3] if case["state"] else None)
        ends = [out, last] if case["state"] else [out]
        grads = torch.autograd.grad(ends, leaves, [v[n] for n in ("dout", "dstate")[: len(ends)]])
    return [out.detach(), last.detach()] + [d.to(t.dtype) for d, t in zip(grads, _learnt(case, v))]


def run(state):
    case = state["case"]
    if "tokens" in state:
        if case["train"]:
            return _own(case, state["v"], state["tokens"])
        with torch.no_grad():
            return _own(case, state["v"], state["tokens"])
    with torch.no_grad():
        return _plain(case, state["v"])


# ---------------------------------------------------------------------------------------
# The definitions in 64 bits: the forwards written out, their gradients by differentiation
# ---------------------------------------------------------------------------------------
def _exact_norm(case, v):
    names = ["x", "weight", "bias"]
    leaves = [v[n].double() for n in names]
    out = []
    if case["add"]:
        total = leaves[0] + v["residual"].double()
        leaves[0] = total.to(v["x"].dtype).double()
        out = [total]
    x, w, b = [t.requires_grad_(case["train"]) for t in leaves]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = (x - mean) * torch.rsqrt(var + EPS) * w + b
    out.insert(0, y.detach())
    if case["train"]:
        dx, dw, db = torch.autograd.grad(y, [x, w, b], v["dy"].double())
        if case["add"]:
            dx = dx + v["dsum"].double()
        out += ([dx, dx] if case["add"] else [dx]) + [dw, db]
    return out


def _exact_linear(case, v):
    leaves = [t.double().requires_grad_(case["train"]) for t in _learnt(case, v)]
    y = torch.mm(leaves[0], leaves[1].t())
    if case["bias"]:
        y = y + leaves[2]
    if case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
    elif case["act"] == "relu":
        y = y.clamp(min=0)
    if case["residual"]:
        y = y + v["residual"].double()
    return [y.detach(), *torch.autograd.grad(y, leaves, v["dy"].double())] if case["train"] else [y]


def _exact_step(case, v):
    s, out = v["state"].double(), []
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        at = int(v["slots"][b]) if "slots" in v else b
        k, w = (v[n][b].double().repeat_interleave(group, 0) for n in ("k", "v"))
        s[at] = v["log_decay"].double().exp()[:, None, None] * s[at] + k[:, :, None] @ w[:, None, :]
        out.append(_scale(case) * (v["q"][b].double()[:, None, :] @ s[at])[:, 0])
    return [torch.stack(out), s]


def _exact_decay(case, v):
    """Head by head: every pair of tokens, without chunks."""
    train, group, g = case["train"], case["heads"] // case["kv_heads"], v["log_decay"].double()
    q, k, w = (v["q"], v["k"], v["v"]) if train else _heads(case, v["qkv"])
    b, t, h, dk = q.shape
    dv = w.size(3)
    new = {"device": "cuda", "dtype": torch.float64}
    out, last = torch.zeros(b, t, h, dv, **new), torch.zeros(b, h, dk, dv, **new)
    grads = [torch.zeros(x.shape, **new) for x in (q, k, w)] + ([torch.zeros(b, h, dk, dv, **new)] if case["state"] else [])
    for i in range(b):
        n = int(v["lengths"][i]) if case["ragged"] else t
        at = torch.arange(n, device="cuda", dtype=torch.float64)
        apart = at[:, None] - at
        for j in range(h):
            leaves = [x[i, :n, jj].double() for x, jj in ((q, j), (k, j // group), (w, j // group))]
            leaves.append(v["state"][i, j].double() if case["state"] else torch.zeros(dk, dv, **new))
            qh, kh, wh, s0 = [x.requires_grad_(train) for x in leaves]
            weight = torch.exp(g[j] * apart).masked_fill_(apart < 0, 0.0)
            o = _scale(case) * (((qh @ kh.t()) * weight) @ wh + torch.exp(g[j] * (at + 1))[:, None] * (qh @ s0))
            s = (kh * torch.exp(g[j] * (n - 1 - at))[:, None]).t() @ wh + torch.exp(g[j] * n) * s0
            out[i, :n, j], last[i, j] = o.detach(), s.detach()
            if train:
                given = [v["dout"][i, :n, j].double()] + ([v["dstate"][i, j].double()] if case["state"] else [])
                found = torch.autograd.grad([o, s][: len(given)], [qh, kh, wh, s0], given)
                grads[0][i, :n, j] = found[0]
                grads[1][i, :n, j // group] += found[1]
                grads[2][i, :n, j // group] += found[2]
                if case["state"]:
                    grads[3][i, j] = found[3]
    return [out, last] + (grads if train else [])


def exact(case, seed):
    v = _values(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "step": _exact_step, "decay": _exact_decay}[case["op"]](case, v)


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    op, train = case["op"], case["train"]
    if op == "norm":
        n, e = case["rows"] * case["dim"], DTYPES[case["dtype"]].itemsize
        # x (and the residual) read, y (and the sum) written; dy (and the sum's gradient) read, dx written; x again for the gradient is not counted
        tensors = (4 if case["add"] else 2) + ((3 if case["add"] else 2) if train else 0)
        return {"bytes": tensors * n * e + case["dim"] * e * (4 if train else 2), "flops": n * (20 if train else 8)}
    if op == "linear":
        m, k, n = case["rows"], case["width"], case["units"]
        rows, weight = 2 * m * (k + n), 2 * n * k
        if case["residual"]:
            rows += 2 * m * n
        return {"bytes": rows + weight + (2 * m * (n + k) + weight if train else 0), "flops": 2 * m * k * n * (3 if train else 1)}
    b, h, kv, dk, dv = case["batch"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
    states = 4 * b * h * dk * dv
    if op == "step":
        return {"bytes": 2 * states + 2 * b * (h * (dk + dv) + kv * (dk + dv)), "flops": 5 * b * h * dk * dv}
    t = case["tokens"] * (0.75 if case["ragged"] else 1.0)
    tensors = 2 * b * t * (h * (dk + dv) + kv * (dk + dv))
    # a chunk of c tokens costs c (dk + dv) operations a token inside it and 4 dk dv between chunks
    c = min(case["tokens"], 64)
    flops = b * t * h * (c * (dk + dv) + 4 * dk * dv)
    moved = tensors + states * (2 if case["state"] else 1)
    return {"bytes": moved + (tensors + (states if case["state"] else 0) if train else 0), "flops": flops * (3 if train else 1)}
