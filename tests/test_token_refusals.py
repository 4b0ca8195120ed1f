"""What the token family's C entry points refuse, and the restatement they are tested against: no GPU (every refusal returns
before a launch)."""
import ctypes as C

import numpy as np
import pytest

from oracle import tokens as otok

P = 1 << 20          # stands for a device address: nothing dereferences it on the host


def embed_fwd(lib, n=4, D=8, V=5, tok=P, stride=1, table=P, td=0, ldt=8, out=P, od=0, ldo=8):
    return lib.tad_token_embed_fwd(n, D, V, tok, stride, 1.0, table, td, ldt, out, od, ldo, None)


def embed_bwd(lib, n=4, D=8, V=5, tok=P, stride=1, dout=P, dd=0, ldd=8, dt=P, ldg=8, acc=1, ws=P, wb=1 << 20):
    return lib.tad_token_embed_bwd(n, D, V, tok, stride, 1.0, dout, dd, ldd, dt, ldg, acc, ws, wb, None)


def distill(lib, rows=2, V=9, K=3, x=P, dtype=0, ld=9, idx=P, val=P, ldt=3, tau=1.0, loss=P, d=P + 4096, ldd=9):
    return lib.tad_distill_loss(rows, V, K, x, dtype, ld, idx, val, ldt, tau, None, 1.0, loss, d, ldd, None)


def sample(lib, rows=2, V=9, x=P, dtype=0, ld=9, T=1.0, k=0, p=1.0, m=0.0, u=P, out=P):
    return lib.tad_sample_tokens(rows, V, x, dtype, ld, T, None, k, None, p, None, m, None, u, out, None)


@pytest.mark.parametrize("call,bad", [
    (embed_fwd, dict(n=-1)), (embed_fwd, dict(D=0)), (embed_fwd, dict(V=-1)), (embed_fwd, dict(td=2)), (embed_fwd, dict(od=-1)), (embed_fwd, dict(ldt=7)),
    (embed_fwd, dict(ldo=0)), (embed_fwd, dict(stride=-1)), (embed_fwd, dict(tok=None)), (embed_fwd, dict(out=None)), (embed_fwd, dict(table=None)),
    (embed_bwd, dict(n=1 << 31)), (embed_fwd, dict(n=1 << 40)), (embed_bwd, dict(V=1 << 30, acc=0, wb=1 << 40)), (embed_bwd, dict(V=(1 << 31) - 1)), (embed_bwd, dict(D=0)), (embed_bwd, dict(dd=3)), (embed_bwd, dict(ldd=0)),
    (embed_bwd, dict(ldg=7)), (embed_bwd, dict(tok=None)), (embed_bwd, dict(dout=None)), (embed_bwd, dict(dt=None)), (embed_bwd, dict(ws=None)),
    (embed_bwd, dict(ws=P + 8)), (embed_bwd, dict(wb=64)),
    (distill, dict(rows=-1)), (distill, dict(V=0)), (distill, dict(K=0)), (distill, dict(K=1025, ldt=1025)), (distill, dict(dtype=5)), (distill, dict(ld=8)),
    (distill, dict(ldt=2)), (distill, dict(ldd=8)), (distill, dict(tau=0.0)), (distill, dict(tau=-1.0)), (distill, dict(tau=float("nan"))),
    (distill, dict(tau=float("inf"))), (distill, dict(tau=1e-30)), (distill, dict(tau=1e30)), (distill, dict(x=None)), (distill, dict(idx=None)), (distill, dict(val=None)), (distill, dict(loss=None)),
    (distill, dict(d=P, ldd=12)),
    (sample, dict(rows=-1)), (sample, dict(V=0)), (sample, dict(dtype=2)), (sample, dict(ld=8)), (sample, dict(T=-0.5)), (sample, dict(T=float("nan"))),
    (sample, dict(k=-1)), (sample, dict(p=-0.1)), (sample, dict(p=float("nan"))), (sample, dict(m=-0.1)), (sample, dict(m=1.5)), (sample, dict(x=None)),
    (sample, dict(u=None)), (sample, dict(out=None))])
def test_refused(lib, call, bad):
    assert call(lib, **bad) == 1                     # TAD_ERR_INVALID
    assert lib.tad_last_error().decode().startswith("tad_")


def test_nothing_to_do(lib):
    assert embed_fwd(lib, n=0, tok=None, out=None, table=None) == 0
    assert embed_bwd(lib, n=0, tok=None, dout=None, ws=None, wb=0) == 0
    assert embed_bwd(lib, V=0, dt=None) == 0
    assert distill(lib, rows=0, x=None) == 0
    assert sample(lib, rows=0, x=None) == 0
    assert lib.tad_token_embed_bwd_workspace_bytes(0, 8) == 0


def test_workspace_covers_every_cut(lib):
    """The stated size is enough for either element type, aligned or not: the entry point accepts exactly that size."""
    for n in (1, 63, 4096, 5000, 131073, 1 << 24):
        for D in (1, 64, 127, 128, 1000, 4096):
            need = lib.tad_token_embed_bwd_workspace_bytes(n, D)
            assert need >= 16 * n
            for dd in (0, 1):
                for ldd in (D, D + 1):
                    # (refused for another reason that is checked later than the workspace: none; a short one is refused)
                    assert embed_bwd(lib, n=n, D=D, dd=dd, ldd=ldd, ldg=D, wb=15 * n) == 1


def test_restatement_gradients_against_differences():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 6))
    index = np.array([[0, 2, 2], [1, -1, 9], [5, 4, 3]])
    value = rng.standard_normal((3, 3)).astype(np.float32)
    w = np.array([1.0, 0.5, 2.0])
    _, g = otok.distill(x, index, value, 1.3, w, 1.0)
    for j in range(6):
        hi, lo = x.copy(), x.copy()
        hi[:, j] += 1e-6
        lo[:, j] -= 1e-6
        diff = (otok.distill(hi, index, value, 1.3, w, 1.0)[0] - otok.distill(lo, index, value, 1.3, w, 1.0)[0]) / 2e-6
        assert np.allclose(diff, g[:, j], atol=1e-8)
    tok, table, weight = np.array([2, 0, 2, -1, 7]), rng.standard_normal((4, 3)), rng.standard_normal((5, 3))
    grad = otok.embed_bwd(tok, weight, 4, 1.5)[0]
    for v in range(4):
        for c in range(3):
            hi = table.copy()
            hi[v, c] += 1e-6
            diff = ((otok.embed_fwd(tok, hi, 1.5) - otok.embed_fwd(tok, table, 1.5)) * weight).sum() / 1e-6
            assert abs(diff - grad[v, c]) < 1e-8


def test_restatement_draw():
    row = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [otok.sample(row, u, 1.0, 0, 1.0, 0.0)[0] for u in (0.0, 0.05, 0.15, 0.49, 0.55, 0.65, 0.75, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [otok.sample(row, u, 1.0, 2, 1.0, 0.0)[0] for u in (0.0, 0.5, 0.6, 0.99)] == [1, 1, 3, 3]
    assert otok.sample(row, 0.99, 1.0, 0, 0.6, 0.0)[0] == 3 and otok.sample(row, 0.99, 1.0, 0, 0.3, 0.0)[0] == 1
    assert otok.sample(row, 0.99, 1.0, 0, 1.0, 0.9)[0] == 1 and otok.sample(row, 0.5, 0.0, 0, 1.0, 0.0)[0] == 1
    tied = np.zeros(4)
    assert otok.sample(tied, 0.99, 1.0, 2, 1.0, 0.0)[0] == 1 and otok.sample(tied, 0.99, 1.0, 0, 0.5, 0.0)[0] == 1
    assert otok.sample(np.full(3, -np.inf), 0.5, 1.0, 0, 1.0, 0.0)[0] == -1
