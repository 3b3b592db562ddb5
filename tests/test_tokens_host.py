"""Token-model operators on the host: the C ABI's argument checks (every call is refused before
any launch, or has nothing to do) and the Python functions' refusals of CPU tensors."""
import math

import pytest
import torch

from xdna_train import hip_abi, tokens

A = 0x1000  # an aligned address that no call dereferences


def refused(rc, why):
    return rc == -1 and why in hip_abi.last_error()


def test_embedding_refuses_bad_arguments():
    lib = hip_abi.load()

    def fwd(ids=A, ib=8, n=4, w=A, dt=2, V=10, D=8, ld=8, out=A):
        return lib.xdna_embed(ids, ib, n, w, dt, V, D, ld, 1.0, out, None)

    for kw, why in [({"ids": None}, "null"), ({"w": None}, "null"), ({"out": None}, "null"), ({"ib": 2}, "4 or 8"), ({"dt": 3}, "dtype"),
                    ({"n": -1}, "token count"), ({"n": (1 << 30) + 1}, "token count"), ({"V": 0}, "rows"), ({"V": (1 << 30) + 1}, "rows"),
                    ({"D": 0}, "length"), ({"ld": 7}, "overlap"), ({"w": A + 1}, "misaligned"), ({"out": A + 2, "dt": 1}, "misaligned")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(n=0, ids=None, w=None, out=None) == 0
    need = lib.xdna_embed_bwd_workspace_bytes(4, 10, 8)
    assert need > 0 and lib.xdna_embed_bwd_workspace_bytes(0, 10, 8) == 0

    def bwd(ids=A, ib=8, n=4, g=A, dt=2, V=10, D=8, dw=A, ws=A, have=need):
        return lib.xdna_embed_bwd(ids, ib, n, g, dt, 8, V, D, -1, 1.0, dw, ws, have, None)

    for kw, why in [({"ids": None}, "null"), ({"g": None}, "null"), ({"dw": None}, "null"), ({"dw": A + 8}, "misaligned"),
                    ({"ws": None}, "workspace"), ({"ws": A + 8}, "workspace"), ({"have": need - 1}, "workspace"), ({"ib": 1}, "4 or 8"),
                    ({"dt": 0}, "dtype"), ({"V": 0}, "rows")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())


def test_gated_refuses_bad_arguments():
    lib = hip_abi.load()

    def fwd(x=A, ldx=8, w=A, ldw=8, M=2, K=8, F=4, act=0, h=A, gu=A):
        return lib.xdna_gated_bf16(x, ldx, w, ldw, M, K, F, act, h, gu, None)

    for kw, why in [({"x": None}, "null"), ({"w": None}, "null"), ({"h": None}, "null"), ({"act": 3}, "activation"), ({"act": -1}, "activation"),
                    ({"M": -1}, "sizes"), ({"K": 0}, "sizes"), ({"F": 0}, "sizes"), ({"ldx": 7}, "overlap"), ({"ldw": 7}, "overlap"),
                    ({"M": 1 << 29}, "rows"), ({"x": A + 1}, "misaligned"), ({"gu": A + 1}, "misaligned")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(M=0, x=None, h=None) == 0

    def bwd(dh=A, gu=A, M=2, F=4, act=0, dgu=A):
        return lib.xdna_gated_bwd_bf16(dh, 4, gu, M, F, act, dgu, None)

    for kw, why in [({"dh": None}, "null"), ({"gu": None}, "null"), ({"dgu": None}, "null"), ({"act": 9}, "activation"), ({"F": -1}, "sizes"),
                    ({"dgu": A + 1}, "misaligned")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())


def test_rows_over_a_vocabulary_refuse_bad_arguments():
    lib = hip_abi.load()
    assert lib.xdna_token_logprobs_workspace_bytes(2, 100, 0) == 0
    need = lib.xdna_token_logprobs_workspace_bytes(2, 100000, 5)
    assert need > 0 and lib.xdna_token_logprobs_workspace_bytes(2, 1 << 23, 5) == 0

    def fwd(z=A, dt=2, n=2, V=100000, ld=100000, y=A, ib=8, tau=1.0, top=5, lp=A, h=A, st=A, tl=A, ti=A, ws=A, have=need):
        return lib.xdna_token_logprobs(z, dt, n, V, ld, y, ib, tau, top, lp, h, st, tl, ti, ws, have, None)

    for kw, why in [({"z": None}, "null"), ({"y": None}, "null"), ({"lp": None}, "null"), ({"h": None}, "null"), ({"st": None}, "null"),
                    ({"ti": None}, "null"), ({"dt": 3}, "dtype"), ({"n": -1}, "row count"), ({"V": 0}, "vocabulary"), ({"V": (1 << 22) + 1}, "vocabulary"),
                    ({"ld": 99999}, "overlap"), ({"tau": 0.0}, "temperature"), ({"tau": math.inf}, "temperature"), ({"tau": math.nan}, "temperature"),
                    ({"top": 65}, "top"), ({"top": -1}, "top"), ({"V": 4, "ld": 4}, "top"), ({"ib": 2}, "4 or 8"), ({"z": A + 1}, "misaligned"),
                    ({"ws": None}, "workspace"), ({"have": need - 1}, "workspace"), ({"ws": A + 4}, "workspace"), ({"st": A + 4}, "misaligned")]:
        assert refused(fwd(**kw), why), (kw, hip_abi.last_error())
    assert fwd(n=0, z=None, y=None) == 0

    def bwd(z=A, dt=2, n=2, V=100, ld=100, y=A, st=A, h=A, dz=A):
        return lib.xdna_token_logprobs_bwd(z, dt, n, V, ld, y, 8, 1.0, st, h, None, None, dz, None)

    for kw, why in [({"z": None}, "null"), ({"st": None}, "null"), ({"dz": None}, "null"), ({"dz": A + 1}, "misaligned"), ({"ld": 10}, "overlap")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())

    def dis(z=A, n=2, V=100, ld=100, ids=A, ib=8, t=A, td=1, k=4, tau=1.0, red=1, rl=A, sh=A, st=A, p=A, loss=A, inv=A):
        return lib.xdna_distill(z, 2, n, V, ld, ids, ib, t, td, k, tau, None, red, rl, sh, st, p, loss, inv, None, 0, None)

    for kw, why in [({"z": None}, "null"), ({"ids": None}, "null"), ({"t": None}, "null"), ({"p": None}, "null"), ({"loss": None}, "null"),
                    ({"inv": None, "red": 2}, "null"), ({"k": 0}, "entries"), ({"k": 1025}, "entries"), ({"td": 3}, "teacher"), ({"red": 3}, "reduction"),
                    ({"tau": -1.0}, "temperature"), ({"V": 100000, "ld": 100000}, "workspace"), ({"st": A + 4}, "misaligned")]:
        assert refused(dis(**kw), why), (kw, hip_abi.last_error())

    def dbwd(z=A, k=4, go=A, gd=1, dz=A, st=A):
        return lib.xdna_distill_bwd(z, 2, 2, 100, 100, A, 8, k, 1.0, A, st, A, None, go, gd, 0, dz, None)

    for kw, why in [({"z": None}, "null"), ({"go": None}, "null"), ({"dz": None}, "null"), ({"gd": 0}, "incoming"), ({"k": 2000}, "entries"),
                    ({"dz": A + 1}, "misaligned")]:
        assert refused(dbwd(**kw), why), (kw, hip_abi.last_error())


def test_cpu_tensors_and_unknown_names_are_refused():
    y, z = torch.zeros(2, dtype=torch.long), torch.zeros(2, 5)
    x16, w16 = torch.zeros(2, 6, dtype=torch.bfloat16), torch.zeros(8, 6, dtype=torch.bfloat16)
    for call in (lambda: tokens.embed(y, z), lambda: tokens.gated_linear(x16, w16), lambda: tokens.gated_mlp(x16, w16, w16[:6, :4]),
                 lambda: tokens.token_log_probs(z, y), lambda: tokens.distill_loss(z, y[:, None], z[:, :1])):
        with pytest.raises(RuntimeError, match="xdna tensor"):
            call()
    for call in (lambda: tokens.gated_linear(x16, w16, activation="tanh"), lambda: tokens.distill_loss(z, y[:, None], z[:, :1], reduction="max")):
        with pytest.raises(ValueError, match="must be one of"):
            call()


def test_gated_products_refuse_bad_arguments():
    lib = hip_abi.load()

    def mm(p=A, ldp=8, pr=0, q=A, ldq=8, qr=0, P=4, Q=4, K=8, out=A, ldc=4):
        return lib.xdna_tile_mm_bf16(p, ldp, pr, q, ldq, qr, P, Q, K, out, ldc, None)

    for kw, why in [({"p": None}, "null"), ({"q": None}, "null"), ({"out": None}, "null"), ({"K": 0}, "sizes"), ({"P": -1}, "sizes"),
                    ({"Q": 1 << 23}, "sizes"), ({"pr": 2}, "contiguous"), ({"qr": 1}, "contiguous"), ({"ldp": 7}, "overlap"), ({"ldq": 7}, "overlap"),
                    ({"ldc": 3}, "overlap"), ({"pr": 1, "ldp": 3}, "overlap"), ({"p": A + 1}, "misaligned")]:
        assert refused(mm(**kw), why), (kw, hip_abi.last_error())
    assert mm(P=0, p=None) == 0

    def bwd(dy=A, ld=8, wo=A, ldw=4, gu=A, M=2, N=8, F=4, act=0, dgu=A):
        return lib.xdna_gated_mlp_bwd_bf16(dy, ld, wo, ldw, gu, M, N, F, act, dgu, None)

    for kw, why in [({"dy": None}, "null"), ({"wo": None}, "null"), ({"gu": None}, "null"), ({"dgu": None}, "null"), ({"ld": 7}, "overlap"),
                    ({"ldw": 3}, "overlap"), ({"act": 4}, "activation"), ({"N": 0}, "sizes"), ({"dgu": A + 1}, "misaligned")]:
        assert refused(bwd(**kw), why), (kw, hip_abi.last_error())
    assert lib.xdna_gated_kept_bytes(3, 4) == 60 and lib.xdna_gated_kept_bytes(0, 4) == 0


def test_gated_gradients_refuse_bad_arguments():
    lib = hip_abi.load()

    def grads(dgu=A, x=A, ldx=8, w=A, ldw=8, dy=A, lddy=6, h=A, M=2, K=8, F=4, N=6, dx=A, dwi=A, dwo=A):
        return lib.xdna_gated_grads_bf16(dgu, x, ldx, w, ldw, dy, lddy, h, M, K, F, N, dx, dwi, dwo, None)

    for kw, why in [({"dgu": None}, "null"), ({"x": None}, "null"), ({"w": None}, "null"), ({"dy": None}, "null"), ({"h": None}, "null"),
                    ({"dx": None}, "null"), ({"dwi": None}, "null"), ({"dwo": None}, "null"), ({"M": 0}, "rows"), ({"K": 0}, "sizes"),
                    ({"N": -1}, "sizes"), ({"N": 1 << 23}, "sizes"), ({"ldx": 7}, "overlap"), ({"ldw": 7}, "overlap"), ({"lddy": 5}, "overlap"),
                    ({"x": A + 1}, "misaligned"), ({"dwo": A + 1}, "misaligned")]:
        assert refused(grads(**kw), why), (kw, hip_abi.last_error())
    assert lib.xdna_gated_grads_pick(0, 8, 4, 6) == 0 and lib.xdna_gated_grads_pick(2, 0, 4, 6) == 0
    # few hundred rows at once; a long k over few tiles, and batches that fill the chip, apart
    assert lib.xdna_gated_grads_pick(333, 1000, 1367, 1000) == 1
    assert lib.xdna_gated_grads_pick(143, 308, 3370, 308) == 0
    assert lib.xdna_gated_grads_pick(64, 512, 512, 0) == 1


def test_backward_rows_may_not_overlap():
    """A row stride under the row's length (a negative one would be read before the operand)."""
    lib = hip_abi.load()
    need = lib.xdna_embed_bwd_workspace_bytes(4, 10, 8)
    for ld in (7, 0, -8):
        assert refused(lib.xdna_embed_bwd(A, 8, 4, A, 2, ld, 10, 8, -1, 1.0, A, A, need, None), "overlap"), ld
        assert refused(lib.xdna_gated_bwd_bf16(A, ld, A, 2, 8, 0, A, None), "overlap"), ld


def test_forward_mode_is_refused_before_anything_else():
    import torch.autograd.forward_ad as fw

    y, z = torch.zeros(2, dtype=torch.long), torch.zeros(2, 5)
    x, w, wo = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((2, 6), (8, 6), (6, 4)))
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))

        for call in (lambda: tokens.embed(y, dual(z)), lambda: tokens.gated_linear(dual(x), w), lambda: tokens.gated_linear(x, dual(w)),
                     lambda: tokens.gated_mlp(dual(x), w, wo), lambda: tokens.gated_mlp(x, dual(w), wo), lambda: tokens.gated_mlp(x, w, dual(wo)),
                     lambda: tokens.token_log_probs(dual(z), y), lambda: tokens.distill_loss(dual(z), y[:, None], z[:, :1]),
                     lambda: tokens.distill_loss(z, y[:, None], dual(z[:, :1])),
                     lambda: tokens.distill_loss(z, y[:, None], z[:, :1], weight=dual(z[:, 0]))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_temperatures_whose_scale_is_infinite_are_refused():
    """log2(e) / tau multiplies differences that may be 0, which would make NaN of the row's maximum."""
    lib = hip_abi.load()
    for tau in (4.0e-39, 2.0e-39, 1e-45):
        assert refused(lib.xdna_token_logprobs(A, 2, 2, 100, 100, A, 8, tau, 0, A, A, A, None, None, None, 0, None), "temperature"), tau
        assert refused(lib.xdna_token_logprobs_bwd(A, 2, 2, 100, 100, A, 8, tau, A, A, None, None, A, None), "temperature"), tau
        assert refused(lib.xdna_distill(A, 2, 2, 100, 100, A, 8, A, 1, 4, tau, None, 1, A, A, A, A, A, A, None, 0, None), "temperature"), tau
        assert refused(lib.xdna_distill_bwd(A, 2, 2, 100, 100, A, 8, 4, tau, A, A, A, None, A, 1, 0, A, None), "temperature"), tau
