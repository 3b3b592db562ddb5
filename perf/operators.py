"""Performance cases of the token-model operators: embedding, gated feed-forward, distillation, token log probabilities.

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
IGNORED = -100  # a target that a batch does not score


def listed():
    return [
        # the next token of one sequence: a single row, where only latency counts
        {"name": "embed lookup T1 V32768 D1024", "op": "embed", "train": False, "tokens": 1, "vocab": 32768, "dim": 1024, "dtype": "bf16"},
        # odd sizes everywhere, a small vocabulary in fp32: a byte- or sign-level model's table
        {"name": "embed train T4099 V5003 D515 f32", "op": "embed", "train": True, "tokens": 4099, "vocab": 5003, "dim": 515, "dtype": "f32"},
        # an ordinary training batch (8 sequences of 1024) on a table of the MLP's width
        {"name": "embed train T8192 V50001 D1024", "op": "embed", "train": True, "tokens": 8192, "vocab": 50001, "dim": 1024, "dtype": "bf16"},
        # a large batch on a large table: the gradient alone is half a gigabyte
        {"name": "embed train T65536 V131072 D2048", "op": "embed", "train": True, "tokens": 65536, "vocab": 131072, "dim": 2048, "dtype": "bf16"},
        # the feed-forward block for one new token: the weights' bytes are the work
        {"name": "gated decode M1 1024-4096", "op": "gated", "train": False, "rows": 1, "width": 1024, "hidden": 4096, "act": "silu"},
        # a short ragged batch, nothing a multiple of a tile
        {"name": "gated train M333 1000-1367", "op": "gated", "train": True, "rows": 333, "width": 1000, "hidden": 1367, "act": "gelu"},
        # the block at the MLP benchmark's sizes, forward and backward
        {"name": "gated train M8192 1024-4096", "op": "gated", "train": True, "rows": 8192, "width": 1024, "hidden": 4096, "act": "silu"},
        # a small student on a small vocabulary, in fp32
        {"name": "distill train T61 V1003 k8 f32", "op": "distill", "train": True, "rows": 61, "vocab": 1003, "k": 8, "dtype": "f32", "tau": 1.0},
        # a student's training batch over a large vocabulary: a gigabyte of logits
        {"name": "distill train T4096 V131072 k64", "op": "distill", "train": True, "rows": 4096, "vocab": 131072, "k": 64, "dtype": "bf16", "tau": 2.0},
        # four answers in progress under a mask of allowed tokens: the chosen tokens' log probabilities beside 20 alternatives
        {"name": "logprobs decode T4 V131072 k20", "op": "logprobs", "train": False, "rows": 4, "vocab": 131072, "k": 20, "dtype": "bf16", "tau": 0.8,
         "masked": 0.5},
        # scoring a batch of given texts
        {"name": "logprobs score T4096 V50001 k5", "op": "logprobs", "train": False, "rows": 4096, "vocab": 50001, "k": 5, "dtype": "bf16", "tau": 1.0,
         "masked": 0.0},
        # a policy-gradient step: log probabilities and entropy with the gradient of both, fp32 logits
        {"name": "logprobs train T1024 V32768 f32", "op": "logprobs", "train": True, "rows": 1024, "vocab": 32768, "k": 0, "dtype": "f32", "tau": 1.0,
         "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n in (1536, 3072) else n


def draw(rng):
    op = rng.choice(["embed", "gated", "distill", "logprobs"])
    train = rng.random() < 0.7
    if op == "embed":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        widest = 32 if dtype == "bf16" else 16
        return {"op": op, "train": train, "tokens": _log_int(rng, 1, 65536), "vocab": _log_int(rng, 256, 131072),
                "dim": _log_int(rng, 64, 64 * widest) if rng.random() < 0.5 else 64 * rng.choice([1, 2, 4, 8, 12, 16, widest]),
                "dtype": dtype}
    if op == "gated":
        few = rng.random() < 0.4  # serving steps beside training batches
        return {"op": op, "train": train and not few, "rows": _log_int(rng, 1, 64) if few else _log_int(rng, 65, 8192),
                "width": _log_int(rng, 128, 1024) if rng.random() < 0.5 else 64 * rng.randint(2, 16),
                "hidden": _log_int(rng, 256, 4096) if rng.random() < 0.5 else 256 * rng.choice([1, 2, 3, 4, 7, 8, 11, 16]),
                "act": rng.choice(["silu", "silu", "gelu", "relu"])}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    vocab = _log_int(rng, 500, 131072)
    rows = _log_int(rng, 1, min(8192, (1 << 29) // (vocab * (2 if dtype == "f32" else 1))))
    tau = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op == "distill":
        return {"op": op, "train": train, "rows": rows, "vocab": vocab, "k": _log_int(rng, 1, 128), "dtype": dtype, "tau": tau}
    return {"op": op, "train": train, "rows": rows, "vocab": vocab, "k": rng.choice([0, 1, 5, 20, 32]), "dtype": dtype, "tau": tau,
            "masked": rng.choice([0.0, 0.0, 0.5])}


# ---------------------------------------------------------------------------------------
# Values
# ---------------------------------------------------------------------------------------
def _zipf(n, vocab, gen):
    """Token ids of a text: rank r with probability ~ 1 / r, ranks scattered over the vocabulary."""
    rank = torch.exp(torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * math.log(vocab + 1)).long().clamp_(1, vocab) - 1
    return torch.randperm(vocab, generator=gen, device="cuda")[rank]


def _values(case, seed):
    """The pass's tensors on the GPU, by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op = case["op"]
    if op == "embed":
        dt = DTYPES[case["dtype"]]
        v = {"weight": (0.02 * normal(case["vocab"], case["dim"])).to(dt), "ids": _zipf(case["tokens"], case["vocab"], g)}
        if case["train"]:
            v["dy"] = normal(case["tokens"], case["dim"]).to(dt)
            v["ids"][uniform(case["tokens"]) < 0.05] = _padding(case)  # padded ends of sequences
        return v
    if op == "gated":
        m, k, f = case["rows"], case["width"], case["hidden"]
        bf16 = torch.bfloat16
        v = {"x": normal(m, k).to(bf16), "w_in": ((2 * uniform(2 * f, k) - 1) / math.sqrt(k)).to(bf16),
             "w_out": ((2 * uniform(k, f) - 1) / math.sqrt(f)).to(bf16)}
        if case["train"]:
            v["dy"] = normal(m, k).to(bf16)
        return v
    t, n, k = case["rows"], case["vocab"], case["k"]
    z = 2.5 * normal(t, n)
    if op == "distill":
        # distinct ids: a random start and random gaps around the vocabulary
        gap = max(1, n // max(k, 1))
        ids = (torch.randint(0, n, (t, 1), generator=g, device="cuda") + torch.randint(1, gap + 1, (t, k), generator=g, device="cuda").cumsum(1)) % n
        teacher = 14.0 - torch.empty(t, k, device="cuda").exponential_(1.0, generator=g).cumsum(1)
        z.scatter_add_(1, ids, teacher * 0.5)  # a student that has learnt some of it
        valid = torch.arange(k, device="cuda")[None] < torch.randint(max(1, k // 2), k + 1, (t, 1), generator=g, device="cuda")
        ids = torch.where(valid, ids, torch.full_like(ids, -1))
        weight = (uniform(t) > 0.1).float()  # padded positions are not trained on
        weight[0] = 1.0
        return {"logits": z.to(DTYPES[case["dtype"]]), "ids": ids, "teacher": teacher, "weight": weight}
    targets = torch.randint(0, n, (t,), generator=g, device="cuda")
    z.scatter_add_(1, targets[:, None], 6.0 * uniform(t, 1))
    if case["masked"]:
        barred = uniform(t, n) < case["masked"]
        barred.scatter_(1, targets[:, None], False)
        z.masked_fill_(barred, -math.inf)
    if case["train"]:
        targets[1:][uniform(t - 1) < 0.05] = IGNORED
    v = {"logits": z.to(DTYPES[case["dtype"]]), "targets": targets}
    if case["train"]:
        v["d_log_probs"], v["d_entropy"] = normal(t), 0.01 * normal(t)
    return v


def _padding(case):
    return case["vocab"] - 1


def _tokens():
    path = str(Path(__file__).resolve().parent.parent / "pytorch-xdna2_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import xdna_train.tokens

    return xdna_train.tokens


def prepare(case, seed):
    v = _values(case, seed)
    state = {"case": dict(case), "v": v}
    if own:
        state["tokens"] = _tokens()
        state["v"] = v = {n: t.to("xdna") for n, t in v.items()}
        if case["train"]:
            for n in ("weight",) if case["op"] == "embed" else ("x", "w_in", "w_out", "logits"):
                if n in v:
                    v[n].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------
# run: the framework's calls
# ---------------------------------------------------------------------------------------
def _own(case, v, T):
    op = case["op"]
    if op == "embed":
        y = T.embed(v["ids"], v["weight"], scale=_scale(case), padding_idx=_padding(case))
        return [y.detach(), *torch.autograd.grad(y, [v["weight"]], v["dy"])] if case["train"] else [y]
    if op == "gated":
        y = T.gated_mlp(v["x"], v["w_in"], v["w_out"], activation=case["act"])
        return [y.detach(), *torch.autograd.grad(y, [v["x"], v["w_in"], v["w_out"]], v["dy"])] if case["train"] else [y]
    if op == "distill":
        loss = T.distill_loss(v["logits"], v["ids"], v["teacher"], temperature=case["tau"], weight=v["weight"])
        return [loss.detach(), *torch.autograd.grad(loss, [v["logits"]])] if case["train"] else [loss]
    r = T.token_log_probs(v["logits"], v["targets"], top_k=case["k"], temperature=case["tau"])
    out = [r.log_probs.detach(), r.entropy.detach()] + ([r.top_log_probs, r.top_ids] if case["k"] else [])
    if case["train"]:
        out += torch.autograd.grad([r.log_probs, r.entropy], [v["logits"]], [v["d_log_probs"], v["d_entropy"]])
    return out


def _scale(case):
    return math.sqrt(case["dim"])


# ---------------------------------------------------------------------------------------
# run: the plain forms, in 32 bits
# ---------------------------------------------------------------------------------------
def _act(name, g):
    """(act(g), act'(g))"""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    on = (g > 0).float()
    return g * on, on


def _plain(case, v):
    op = case["op"]
    if op == "embed":
        dt, s = v["weight"].dtype, _scale(case)
        out = [(v["weight"][v["ids"]].float() * s).to(dt)]
        if case["train"]:
            dy = v["dy"].float() * (v["ids"] != _padding(case)).float()[:, None]
            dw = torch.zeros(case["vocab"], case["dim"], device=dy.device).index_add_(0, v["ids"], dy)
            out.append((dw * s).to(dt))
        return out
    if op == "gated":
        dt, f = v["x"].dtype, case["hidden"]
        x, w_in, w_out = v["x"].float(), v["w_in"].float(), v["w_out"].float()
        gu = x @ w_in.t()
        g, u = gu[:, :f], gu[:, f:]
        a, da = _act(case["act"], g)
        h = a * u
        out = [h @ w_out.t()]
        if case["train"]:
            dy = v["dy"].float()
            dh = dy @ w_out
            dgu = torch.cat([dh * u * da, dh * a], 1)
            out += [dgu @ w_in, dgu.t() @ x, dy.t() @ h]
        return [t.to(dt) for t in out]
    z = v["logits"].float()
    x = z / case["tau"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    lse = m + torch.log(s)
    if op == "distill":
        tau = case["tau"]
        valid = v["ids"] >= 0
        ids = v["ids"].clamp(min=0)
        t = torch.where(valid, v["teacher"] / tau, torch.full_like(v["teacher"], -math.inf))
        p = torch.exp(t - t.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        log_p = torch.log(torch.where(valid, p, torch.ones_like(p)))
        rows = tau * tau * (p * (log_p - torch.gather(x, 1, ids) + lse)).sum(1)
        share = v["weight"] / v["weight"].sum()
        out = [(share * rows).sum()]
        if case["train"]:
            dz = (e / s).scatter_add_(1, ids, -p) * (share * tau)[:, None]
            out.append(dz.to(v["logits"].dtype))
        return out
    scored = v["targets"] >= 0
    lp = torch.gather(x, 1, v["targets"].clamp(min=0)[:, None]) - lse
    lp = torch.where(scored, lp[:, 0], torch.zeros_like(lp[:, 0]))
    q = e / s
    xs = torch.where(q > 0, x, torch.zeros_like(x))
    ent = lse[:, 0] - (q * xs).sum(1)
    out = [lp, ent]
    if case["k"]:
        order = torch.sort(z, dim=1, descending=True, stable=True)
        ids = order.indices[:, : case["k"]].contiguous()
        out += [torch.gather(x, 1, ids) - lse, ids]
    if case["train"]:
        glp = torch.where(scored, v["d_log_probs"], torch.zeros_like(lp))
        dz = -q * (glp[:, None] + v["d_entropy"][:, None] * (xs - lse + ent[:, None]))
        dz.scatter_add_(1, v["targets"].clamp(min=0)[:, None], glp[:, None])
        out.append((dz / case["tau"]).to(v["logits"].dtype))
    return out


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
def exact(case, seed):
    v = _values(case, seed)
    op = case["op"]
    if op == "embed":
        out = [v["weight"].double()[v["ids"]] * math.sqrt(case["dim"])]
        if case["train"]:
            keep = v["ids"] != _padding(case)
            total = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
            step = max(1, (1 << 26) // case["dim"])
            for at in range(0, case["tokens"], step):
                k = keep[at:at + step]
                total.index_put_((v["ids"][at:at + step][k],), v["dy"][at:at + step][k].double(), accumulate=True)
            out.append(total.mul_(math.sqrt(case["dim"])))
        return out
    if op == "gated":
        leaves = [v[n].double().requires_grad_(case["train"]) for n in ("x", "w_in", "w_out")]
        x, w_in, w_out = leaves
        gate, up = torch.mm(x, w_in[: case["hidden"]].t()), torch.mm(x, w_in[case["hidden"]:].t())
        if case["act"] == "silu":
            a = gate * torch.sigmoid(gate)
        elif case["act"] == "gelu":
            a = gate * 0.5 * torch.erfc(-gate / math.sqrt(2.0))
        else:
            a = gate.clamp(min=0)
        y = torch.mm(a * up, w_out.t())
        return [y.detach(), *torch.autograd.grad(y, leaves, v["dy"].double())] if case["train"] else [y]
    step = max(1, (1 << 27) // case["vocab"])
    parts = []
    for at in range(0, case["rows"], step):
        sl = slice(at, at + step)
        z = v["logits"][sl].double().requires_grad_(case["train"])
        log_q = torch.log_softmax(z / case["tau"], 1)
        parts.append(_exact_distill(case, v, sl, z, log_q) if op == "distill" else _exact_logprobs(case, v, sl, z, log_q))
    joined = [torch.cat([p[i] for p in parts]) for i in range(len(parts[0]))]
    return [joined[0].sum(), *joined[1:]] if op == "distill" else joined


def _exact_distill(case, v, sl, z, log_q):
    tau, share = case["tau"], (v["weight"].double() / v["weight"].double().sum())[sl]
    ids = v["ids"][sl]
    log_p = torch.log_softmax((v["teacher"][sl].double() / tau).masked_fill(ids < 0, -math.inf), 1)
    terms = log_p.exp() * (log_p.masked_fill(ids < 0, 0.0) - log_q.gather(1, ids.clamp(min=0)))
    rows = share * tau ** 2 * terms.sum(1)
    return [rows.detach(), *torch.autograd.grad(rows.sum(), [z])] if case["train"] else [rows]


def _exact_logprobs(case, v, sl, z, log_q):
    y = v["targets"][sl]
    lp = log_q.gather(1, y.clamp(min=0)[:, None])[:, 0].masked_fill(y < 0, 0.0)
    finite = torch.isfinite(z)
    ent = -(log_q.exp() * log_q.masked_fill(~finite, 0.0)).sum(1)
    out = [lp.detach(), ent.detach()]
    if case["k"]:
        ids = torch.argsort(z.detach(), dim=1, descending=True, stable=True)[:, : case["k"]]
        out += [log_q.detach().gather(1, ids), ids]
    if case["train"]:
        d = v["d_log_probs"][sl].double() * lp + v["d_entropy"][sl].double() * ent
        (dz,) = torch.autograd.grad(d.sum(), [z])
        out.append(dz.masked_fill(~finite, 0.0))
    return out


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    op, train = case["op"], case["train"]
    if op == "embed":
        t, n, d, e = case["tokens"], case["vocab"], case["dim"], DTYPES[case["dtype"]].itemsize
        looked_up = n * (1 - math.exp(-t / n))  # at most: distinct rows of uniformly drawn ids
        moved = 8 * t + (looked_up + t) * d * e
        ops = t * d
        if train:
            moved += (t + n) * d * e
            ops += 2 * t * d
        return {"bytes": moved, "flops": ops}
    if op == "gated":
        m, k, f = case["rows"], case["width"], case["hidden"]
        flops = 6 * m * k * f
        weights, rows = 3 * f * k * 2, m * k * 2
        return {"bytes": 2 * weights + 4 * rows if train else weights + 2 * rows, "flops": 3 * flops if train else flops}
    t, n, e = case["rows"], case["vocab"], DTYPES[case["dtype"]].itemsize
    per_row = 12 * case["k"] + (8 if op == "distill" else 16)
    return {"bytes": t * (n * e * (2 if train else 1) + per_row), "flops": t * n * (8 if train else 4)}
