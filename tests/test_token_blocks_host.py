"""A token model's block on the host: the C ABI's argument checks (every call is refused before any launch,
or has nothing to do) and the Python functions' refusals of CPU tensors."""
import ctypes
import math

import pytest
import torch

from xdna_train import hip_abi, tokens

A = 0x1000  # an aligned address that no call dereferences


def refused(rc, why):
    return rc == -1 and why in hip_abi.last_error()


def test_layer_norm_refuses_bad_arguments():
    lib = hip_abi.load()

    def fwd(x=A, ldx=8, r=None, ldr=8, dt=2, n=4, D=8, w=A, b=A, pt=2, eps=1e-5, s=None, y=A, st=A):
        return lib.xdna_layer_norm(x, ldx, r, ldr, dt, n, D, w, b, pt, eps, s, y, st, None)

    for kw, why in [({"x": None}, "null"), ({"y": None}, "null"), ({"r": A}, "null"), ({"dt": 3}, "dtype"), ({"dt": 1, "pt": 2}, "parameters"),
                    ({"n": -1}, "row count"), ({"n": (1 << 30) + 1}, "row count"), ({"D": 0}, "length"), ({"D": (1 << 24) + 1}, "length"),
                    ({"ldx": 7}, "overlap"), ({"r": A, "s": A, "ldr": 7}, "overlap"), ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"),
                    ({"eps": math.inf}, "eps"), ({"x": A + 1}, "misaligned"), ({"w": A + 2, "pt": 1}, "misaligned"), ({"st": A + 2}, "misaligned")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(n=0, x=None, y=None) == 0
    need = lib.xdna_layer_norm_bwd_workspace_bytes(4, 8)
    assert need > 0 and lib.xdna_layer_norm_bwd_workspace_bytes(0, 8) == 0 and lib.xdna_layer_norm_bwd_workspace_bytes(4, 0) == 0

    def bwd(dy=A, lddy=8, ds=None, ldds=8, x=A, ldx=8, dt=2, n=4, D=8, w=A, pt=2, st=A, dx=A, dw=A, db=A, ws=A, have=need):
        return lib.xdna_layer_norm_bwd(dy, lddy, ds, ldds, x, ldx, dt, n, D, w, pt, st, dx, dw, db, ws, have, None)

    for kw, why in [({"dy": None}, "null"), ({"x": None}, "null"), ({"st": None}, "null"), ({"lddy": 7}, "overlap"), ({"ldx": 7}, "overlap"),
                    ({"ds": A, "ldds": 7}, "overlap"), ({"ws": None}, "workspace"), ({"ws": A + 8}, "workspace"), ({"have": need - 1}, "workspace"),
                    ({"dx": A + 1}, "misaligned"), ({"db": A + 1}, "misaligned"), ({"dt": 0}, "dtype")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())
    assert bwd(dx=None, dw=None, db=None) == 0 and bwd(n=0, dw=None, db=None) == 0


def test_linear_refuses_bad_arguments():
    lib = hip_abi.load()

    def fwd(x=A, ldx=8, w=A, ldw=8, M=2, K=8, N=4, act=0, b=A, r=A, ldr=4, y=A, s=A):
        return lib.xdna_linear_bf16(x, ldx, w, ldw, M, K, N, act, b, r, ldr, y, s, None)

    for kw, why in [({"x": None}, "null"), ({"w": None}, "null"), ({"y": None}, "null"), ({"act": 4}, "activation"), ({"act": -1}, "activation"),
                    ({"M": -1}, "sizes"), ({"K": 0}, "sizes"), ({"N": 0}, "sizes"), ({"M": (1 << 22) + 1}, "sizes"), ({"ldx": 7}, "overlap"),
                    ({"ldw": 7}, "overlap"), ({"ldr": 3}, "overlap"), ({"act": 3}, "slopes"), ({"x": A + 1}, "misaligned"), ({"b": A + 1}, "misaligned"),
                    ({"s": A + 1}, "misaligned"), ({"M": 1 << 22, "N": 1 << 21}, "outputs")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(M=0, x=None, y=None) == 0
    need = lib.xdna_linear_bwd_workspace_bytes(2, 4)
    assert need > 0 and lib.xdna_linear_bwd_workspace_bytes(0, 4) == 0

    assert [lib.xdna_linear_kept_bytes(3, 10, act) for act in range(4)] == [60, 60, 9, 0] and lib.xdna_linear_kept_bytes(0, 10, 0) == 0

    def bwd(dy=A, ld=4, s=A, act=0, M=2, N=4, dp=A, db=A, ws=A, have=need):
        return lib.xdna_linear_bwd_bf16(dy, ld, s, act, M, N, dp, db, ws, have, None)

    for kw, why in [({"dy": None}, "null"), ({"s": None}, "null"), ({"act": 4}, "activation"), ({"ld": 3}, "overlap"), ({"ws": None}, "workspace"), ({"ws": A + 8}, "workspace"),
                    ({"have": need - 1}, "workspace"), ({"dp": A + 1}, "misaligned"), ({"N": 0}, "sizes")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())
    assert bwd(dp=None, db=None) == 0 and bwd(M=0, db=None) == 0

    def grads(dp=A, lddp=4, x=A, ldx=8, w=A, ldw=8, M=2, K=8, N=4, dx=A, dw=A):
        return lib.xdna_linear_grads_bf16(dp, lddp, x, ldx, w, ldw, M, K, N, dx, dw, None)

    for kw, why in [({"dp": None}, "null"), ({"dx": None}, "null"), ({"dw": None}, "null"), ({"M": 0}, "no rows"), ({"lddp": 3}, "overlap"),
                    ({"ldx": 7}, "overlap"), ({"ldw": 7}, "overlap"), ({"K": 0}, "sizes"), ({"dw": A + 1}, "misaligned")]:
        assert refused(grads(**kw), why), (kw, hip_abi.last_error())

    def pick(M, K, N, at=A, ld=0):
        return lib.xdna_linear_grads_pick(at, ld or N, at, ld or K, at, ld or K, M, K, N)

    assert pick(0, 8, 8) == 0 and pick(333, 1000, 1367) == 1 and pick(8192, 1024, 4096) == 2
    assert pick(8192, 1024, 4096, at=A + 2) != 2 and pick(8192, 1024, 4096, ld=4097) != 2  # (no whole vectors)
    assert pick(8192, 1024, 4096, ld=1 << 20) != 2  # (offsets past 32 bits)


def test_decay_attention_refuses_bad_arguments():
    lib = hip_abi.load()
    ok = hip_abi.Heads(A, 64, 16, 8)

    def ref(h):
        return ctypes.byref(h) if h is not None else None

    # few long sequences: segments
    need = lib.xdna_decay_workspace_bytes(1, 8192, 2, 8, 8)
    assert need > 0 and lib.xdna_decay_workspace_bytes(1, 64, 2, 8, 8) == 0 and lib.xdna_decay_workspace_bytes(0, 8192, 2, 8, 8) == 0
    assert lib.xdna_decay_workspace_bytes(512, 8192, 2, 8, 8) == 0

    def fwd(q=ok, k=ok, v=ok, Bn=1, T=8192, H=2, G=1, dk=8, dv=8, g=A, n=A, ib=8, scale=1.0, s=A, o=A, so=A, ws=A, have=need):
        return lib.xdna_decay_attention(ref(q), ref(k), ref(v), Bn, T, H, G, dk, dv, g, n, ib, scale, s, o, so, ws, have, None)

    bad = [({"q": None}, "null"), ({"k": hip_abi.Heads(None, 1, 1, 1)}, "null"), ({"v": hip_abi.Heads(A + 1, 1, 1, 1)}, "misaligned"),
           ({"q": hip_abi.Heads(A, -1, 1, 1)}, "negative"), ({"Bn": -1}, "range"), ({"T": -1}, "range"), ({"T": 0}, "no tokens"), ({"H": 0}, "range"),
           ({"G": 0}, "divide"), ({"H": 3, "G": 2}, "divide"), ({"G": 4}, "divide"), ({"dk": 0}, "1 .. 128"), ({"dv": 129}, "1 .. 128"), ({"g": None}, "null"),
           ({"g": A + 2}, "misaligned"), ({"ib": 2}, "4 or 8"), ({"n": A + 4}, "misaligned"), ({"scale": math.inf}, "scale"), ({"scale": math.nan}, "scale"),
           ({"Bn": 1 << 20, "H": 1 << 12}, "too many"), ({"Bn": 1398102, "H": 1}, "out of range"), ({"Bn": 699051, "H": 2}, "too many")]
    for kw, why in bad + [({"o": None}, "null"), ({"o": A + 1}, "misaligned"), ({"s": A + 2}, "misaligned"), ({"so": A + 2}, "misaligned"),
                          ({"ws": None}, "workspace"), ({"ws": A + 8}, "workspace"), ({"have": need - 1}, "workspace")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(Bn=0, q=None) == 0
    need_b = lib.xdna_decay_bwd_workspace_bytes(1, 8192, 2, 1, 8, 8)
    assert need_b > lib.xdna_decay_bwd_workspace_bytes(1, 8192, 2, 2, 8, 8) > 0

    def bwd(do=ok, ds=A, q=ok, k=ok, v=ok, Bn=1, T=8192, H=2, G=1, dk=8, dv=8, g=A, n=A, ib=8, scale=1.0, s=A, dq=A, dkk=A, dvv=A, d0=A, ws=A, have=need_b):
        return lib.xdna_decay_attention_bwd(ref(do), ds, ref(q), ref(k), ref(v), Bn, T, H, G, dk, dv, g, n, ib, scale, s, dq, dkk, dvv, d0, ws, have, None)

    for kw, why in bad + [({"do": None}, "null"), ({"dq": None}, "null"), ({"dkk": None}, "null"), ({"dvv": None}, "null"), ({"dq": A + 1}, "misaligned"),
                          ({"ds": A + 2}, "misaligned"), ({"d0": A + 2}, "misaligned"), ({"ws": None}, "workspace"), ({"have": need_b - 1}, "workspace")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())
    assert bwd(Bn=0, q=None) == 0

    def step(q=ok, k=ok, v=ok, Bn=3, H=2, G=1, dk=8, dv=8, g=A, s=A, slots=3, i=None, ib=8, scale=1.0, o=A):
        return lib.xdna_decay_step(ref(q), ref(k), ref(v), Bn, H, G, dk, dv, g, s, slots, i, ib, scale, o, None)

    for kw, why in [({"q": None}, "null"), ({"g": None}, "null"), ({"s": None}, "null"), ({"o": None}, "null"), ({"slots": 2}, "fewer states"),
                    ({"slots": -1, "i": A}, "fewer states"), ({"i": A, "ib": 1}, "4 or 8"), ({"s": A + 2}, "misaligned"), ({"H": 3, "G": 2}, "divide"),
                    ({"dk": 129}, "1 .. 128"), ({"scale": math.nan}, "scale"), ({"Bn": 699051, "slots": 699051}, "too many")]:
        assert refused(step(**kw), why), (kw, hip_abi.last_error())
    assert step(Bn=0, q=None, slots=0) == 0


def test_functions_refuse_cpu_tensors():
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16)
    g, s = torch.zeros(1), torch.zeros(1, 1, 8, 8)
    for call in (lambda: tokens.layer_norm(x), lambda: tokens.add_layer_norm(x, x), lambda: tokens.linear(x, x), lambda: tokens.decay_attention(q, q, q, g),
                 lambda: tokens.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], g, s)):
        with pytest.raises(RuntimeError, match="xdna"):
            call()
    with pytest.raises(ValueError, match="one of"):
        tokens.linear(x, x, activation="tanh")
