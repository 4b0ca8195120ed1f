"""Token family on the GPU against the float64 restatement (oracle/tokens.py): embedding lookup and gradient by sorted tokens,
distillation loss and gradient, token draw.

Tolerances, with e = 2^-24 (half a float32 step): a rounding to bfloat16 is off by at most 2^-8 of the value.
  lookup:    one float32 product, one rounding to the result's type.
  gradient:  m terms in any order: at most (m + 2) e times the sum of |terms|; times the scale, added to dtable: 3 e more.
  loss:      with A the largest |argument| of an exponential or logarithm in the row, an argument is off by 4 e A, an
             exponential by that and 2 e of its own, the sum of V of them by V / 32 + 16 e more (32 or more partial sums), each
             ln by its argument's error: every ln p or ln q by at most E = e (16 A + V / 32 + K + 64).  The loss is their sum
             weighted with q, whose own error is E relative: w tau^2 E (1 + sum q (|ln q| + |ln p|)) 2.
  gradient:  p and q within E relative each: |g| E (p + q) 2, and the rounding to the type.
  draw:      equal, unless the float64 sums lie within 2^-36 of a border (an input draws none or few of those)."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu

E24 = 2.0 ** -24
B16 = 2.0 ** -8


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops(lib):
    from timeautodiff_amd import ops as _ops
    return _ops


def f64(t):
    return t.detach().cpu().double().numpy()


def strided(rows, cols, extra, dtype, dev, fill=None, offset=0):
    """A [rows, cols] view of a wider matrix (row stride cols + extra, base `offset` elements in), and the matrix."""
    flat = torch.full((rows * (cols + extra) + offset,), 7.5 if fill is None else fill, dtype=dtype, device=dev)
    wide = flat[offset:].view(rows, cols + extra)
    return wide[:, :cols], wide


def round_err(dtype):
    return B16 if dtype == torch.bfloat16 else E24


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (5, 7, 3), (33, 50, 64), (257, 11, 100), (64, 300, 1024), (1000, 4, 136), (7, 40, 2056)])
@pytest.mark.parametrize("ti", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("to", [torch.float32, torch.bfloat16])
def test_token_embed_fwd(ops, dev, n, V, D, ti, to):
    rng = np.random.default_rng(n * 7 + V + D)
    tok = rng.integers(0, V, n)
    tok[rng.random(n) < 0.2] = rng.choice([-1, V, V + 5, -(1 << 62), (1 << 62)])
    for extra, off in ((0, 0), (8, 0), (3, 1)):
        table, _ = strided(V, D, extra, ti, dev, offset=off)
        table.copy_(torch.from_numpy(rng.standard_normal((V, D))).to(dev))
        out, wide = strided(n, D, extra, to, dev, fill=-3.0, offset=off)
        ops.token_embed_fwd(torch.from_numpy(tok).to(dev), table, out, scale=1.75)
        want = otok.embed_fwd(tok, f64(table), 1.75)
        assert np.all(np.abs(f64(out) - want) <= (E24 + round_err(to)) * np.abs(want))
        assert float((wide[:, D:] + 3.0).abs().max() if extra else 0.0) == 0.0     # nothing written beside the slice


def test_token_embed_fwd_strided_tokens_and_none(ops, dev):
    table = torch.randn(9, 16, device=dev)
    tok = torch.randint(0, 9, (6, 5), device=dev)
    out = torch.empty(6, 16, device=dev)
    ops.token_embed_fwd(tok[:, 2], table, out)
    assert torch.equal(out, table[tok[:, 2]])
    out3 = torch.empty(6, 5, 16, device=dev)
    ops.token_embed_fwd(tok, table, out3)
    assert torch.equal(out3, table[tok])
    one = torch.full((1,), 4, device=dev).expand(7)
    out = torch.empty(7, 16, device=dev)
    ops.token_embed_fwd(one, table, out)
    assert torch.equal(out, table[4].expand(7, 16))
    ops.token_embed_fwd(tok[:0, 0], table, out[:0])


# ------------------------------------------------------------------ gradient of the lookup
def bwd_tokens(kind, n, V, rng):
    if kind == "same":
        return np.full(n, V // 2)
    if kind == "padding":
        return np.full(n, -1)
    if kind == "once":                       # every token at most once, in falling order
        return np.arange(n)[::-1] % max(V, n) - (0 if V >= n else n)
    tok = np.minimum(((V + 1.0) ** rng.random(n)).astype(np.int64) - 1, V - 1)
    if kind == "ragged":
        tok[rng.random(n) < 0.3] = rng.choice([-1, V, 1 << 40])
        tok[n - n // 5:] = -1
    return tok


def check_bwd(ops, dev, tok, dout, V, scale, accumulate, extra=0):
    n, D = dout.shape
    dtable, wide = strided(V, D, extra, torch.float32, dev, fill=0.5)
    ops.token_embed_bwd(torch.from_numpy(tok).to(dev), dout, dtable, scale=scale, accumulate=accumulate)
    grad, size, count = otok.embed_bwd(tok, f64(dout), V, scale)
    got = f64(dtable)
    want = grad + (0.5 if accumulate else 0.0)
    tol = E24 * ((count[:, None] + 5) * size + np.abs(want) + 0.5 * (accumulate & (count[:, None] > 0)))
    assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()
    assert np.all(got[count == 0] == (0.5 if accumulate else 0.0))
    if extra:
        assert float((wide[:, D:] - 0.5).abs().max()) == 0.0
    return dtable


@pytest.mark.parametrize("kind", ["zipf", "ragged", "same", "padding", "once"])
@pytest.mark.parametrize("n,V,D,dtype", [(1, 1, 1, torch.float32), (63, 5, 3, torch.bfloat16), (64, 200, 64, torch.float32),
                                         (129, 17, 100, torch.bfloat16), (1000, 33, 128, torch.float32), (2400, 50, 520, torch.bfloat16),
                                         (300, 5000, 260, torch.float32), (1, 2500, 5, torch.float32), (63, 2100, 3, torch.bfloat16),
                                         (1000, 3000, 128, torch.float32), (2400, 4000, 520, torch.bfloat16)])
def test_token_embed_bwd(ops, dev, kind, n, V, D, dtype):
    rng = np.random.default_rng(n + V + D)
    tok = bwd_tokens(kind, n, V, rng)
    for extra in (0, 4, 3):
        dout, _ = strided(n, D, extra, dtype, dev)
        dout.copy_(torch.from_numpy(rng.standard_normal((n, D))).to(dev))
        for accumulate in (False, True):
            a = check_bwd(ops, dev, tok, dout, V, 1.25, accumulate, extra)
            b = check_bwd(ops, dev, tok, dout, V, 1.25, accumulate, extra)
            assert torch.equal(a, b)         # a fixed order of the sums: the same bits


@pytest.mark.parametrize("kind", ["zipf", "ragged", "same", "once"])
@pytest.mark.parametrize("n,V,D", [(4095, 700, 8), (4096, 3, 5), (4097, 9000, 4), (9001, 40, 33), (40000, 30000, 2), (140001, 1000, 3)])
def test_token_embed_bwd_many_tokens(ops, dev, kind, n, V, D):
    """Lengths around the sort's tiles, several tiles, and more than one merge of tiles."""
    rng = np.random.default_rng(n)
    dout = torch.from_numpy(rng.standard_normal((n, D)).astype(np.float32)).to(dev)
    check_bwd(ops, dev, bwd_tokens(kind, n, V, rng), dout, V, 0.5, False)
    check_bwd(ops, dev, bwd_tokens(kind, n, V, rng), dout, V, 0.5, True)


def test_token_embed_bwd_none_and_workspace(ops, dev):
    dtable = torch.full((6, 9), 2.0, device=dev)
    none = torch.empty(0, dtype=torch.int64, device=dev)
    ops.token_embed_bwd(none, torch.empty(0, 9, device=dev), dtable)
    assert bool((dtable == 2.0).all())
    ops.token_embed_bwd(none, torch.empty(0, 9, device=dev), dtable, accumulate=False)
    assert bool((dtable == 0.0).all())
    # a workspace of exactly the stated size, its neighbours untouched, whatever it held
    tok, dout = torch.randint(0, 6, (500,), device=dev), torch.randn(500, 9, device=dev)
    nb = ops.token_embed_bwd_workspace_bytes(500, 9)
    buf = torch.full((nb + 512,), 0xAB, dtype=torch.uint8, device=dev)
    a, b = torch.empty(6, 9, device=dev), torch.empty(6, 9, device=dev)
    ops.token_embed_bwd(tok, dout, a, accumulate=False, workspace=buf[256:256 + nb])
    ops.token_embed_bwd(tok, dout, b, accumulate=False)
    assert torch.equal(a, b) and bool((buf[:256] == 0xAB).all()) and bool((buf[256 + nb:] == 0xAB).all())
    from timeautodiff_amd import _lib
    with pytest.raises(_lib.TadError, match="workspace"):
        ops.token_embed_bwd(tok, dout, a, workspace=buf[256:256 + nb - 16])


# ------------------------------------------------------------------ distillation
def check_distill(ops, dev, logits, index, value, tau, weight, grad_scale, grad=True, inplace=False):
    rows, V = logits.shape
    K = index.shape[1]
    x = f64(logits)
    loss = torch.full((rows,), float("nan"), device=dev)
    if grad and not inplace:
        d, wide = strided(rows, V, logits.stride(0) - V if rows > 1 else 0, logits.dtype, dev, fill=9.0)
    else:
        d = logits if grad else None
    ti = torch.from_numpy(index).to(dev)
    tv = torch.from_numpy(value.astype(np.float32)).to(dev)
    tw = None if weight is None else torch.from_numpy(weight.astype(np.float32)).to(dev)
    ops.distill_loss(logits, ti, tv, loss, temperature=tau, row_weight=tw, grad_scale=grad_scale, dlogits=d)
    t32 = float(np.float32(tau))
    want, wgrad = otok.distill(x, index, value.astype(np.float32), t32, weight, grad_scale)
    got = f64(loss)
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(got)) and np.array_equal(want[~fin], got[~fin])
    for r in range(rows):
        w = 1.0 if weight is None else float(weight[r])
        z = x[r][x[r] > -np.inf] / t32
        ok = (index[r] >= 0) & (index[r] < V) & (value[r] > -np.inf)
        if want[r] == 0.0 and not wgrad[r].any():
            assert got[r] == 0.0 and (not grad or not f64(d[r]).any())
            continue
        t = value[r][ok].astype(np.float64) / t32
        A = max(z.max() - z.min(), t.max() - t.min(), np.log(V), np.log(K), 1.0)
        err = E24 * (16 * A + V / 32 + K + 64)
        q = np.exp(t - t.max())
        q /= q.sum()
        lnp = x[r][index[r][ok]] / t32 - z.max() - np.log(np.exp(z - z.max()).sum())
        if fin[r]:
            size = 1 + np.sum(q * (np.abs(np.log(np.maximum(q, 1e-300))) + np.where(q > 0, np.abs(lnp), 0.0)))
            assert abs(got[r] - want[r]) <= 2 * w * t32 ** 2 * err * size, (r, got[r], want[r])
        if grad:
            g = abs(grad_scale * w * t32)
            p = np.exp(x[r] / t32 - z.max()) / np.exp(z - z.max()).sum()
            qq = np.zeros(V)
            np.add.at(qq, index[r][ok], q)
            tol = g * (2 * err * (p + qq) + 1e-37) + (round_err(logits.dtype) + 3 * E24) * np.abs(wgrad[r])
            assert np.all(np.abs(f64(d[r]) - wgrad[r]) <= tol), (r, np.abs(f64(d[r]) - wgrad[r]).max())
    if grad and not inplace and wide.shape[1] > V:
        assert float((wide[:, V:].float() - 9.0).abs().max()) == 0.0
    return loss


def distill_inputs(rows, V, K, dtype, dev, rng, extra=0, offset=0):
    logits, _ = strided(rows, V, extra, dtype, dev, offset=offset)
    logits.copy_(torch.from_numpy(rng.standard_normal((rows, V)) * 2.5).to(dev))
    index = np.stack([rng.permutation(max(V, K))[:K] for _ in range(rows)]).astype(np.int64) if V >= K else rng.integers(0, V, (rows, K))
    value = np.sort(rng.standard_normal((rows, K)).astype(np.float32) * 2 + 6)[:, ::-1].copy()
    return logits, index, value


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (3, 2, 2), (70, 9, 4), (130, 48, 8), (33, 64, 3), (17, 65, 20), (9, 300, 5), (21, 1000, 64), (5, 2048, 300),
                                      (6, 5003, 17), (3, 32001, 32), (2, 70000, 1000)])
def test_distill_loss(ops, dev, dtype, rows, V, K):
    rng = np.random.default_rng(rows + V + K)
    for tau, extra, offset in ((1.0, 0, 0), (2.5, 8, 0), (0.7, 3, 1)):
        logits, index, value = distill_inputs(rows, V, K, dtype, dev, rng, extra, offset)
        index[rng.random((rows, K)) < 0.1] = rng.choice([-1, V, 1 << 50])
        weight = rng.random(rows) + 0.5
        weight = weight.astype(np.float32).astype(np.float64)
        weight[::3] = 0.0 if rows > 3 else weight[::3]
        a = check_distill(ops, dev, logits, index, value, tau, weight, 0.125)
        b = check_distill(ops, dev, logits, index, value, tau, weight, 0.125, grad=False)
        c = check_distill(ops, dev, logits, index, value, tau, weight, 0.125, inplace=True)
        assert torch.equal(a, b) and torch.equal(a, c)         # one loss, whatever else is asked for


@pytest.mark.parametrize("V", [6, 48, 700, 9000])
def test_distill_loss_masks_and_empty_rows(ops, dev, V):
    """Masked logits (-inf and the type's lowest), rows without entries, rows without logits, the same index twice, entries of
    -inf, rows of weight zero that hold NaN and infinity."""
    rng = np.random.default_rng(V)
    K, rows = 5, 9
    for dtype in (torch.float32, torch.bfloat16):
        logits, index, value = distill_inputs(rows, V, K, dtype, dev, rng)
        weight = np.ones(rows)
        index[0] = [-1] * K                                    # no entry
        value[1] = -np.inf                                     # no entry above -inf
        logits[2] = -float("inf")                              # no student logit
        index[3] = [2, 2, 1, 2, V - 1]                         # one index three times
        value[4, 1:] = -np.inf
        logits[4, [j for j in range(V) if j != index[4, 0]]] = -float("inf")       # p = q = 1 at one place: loss 0
        logits[5] = torch.finfo(dtype).min                     # every logit the lowest: p is even
        logits[6, index[6, 0]] = -float("inf")                 # q above 0 where p = 0
        logits[7, :V // 2] = torch.finfo(dtype).min
        index[7] = V - 1 - np.arange(K) % (V // 2)
        logits[8, 0], logits[8, 1] = float("nan"), float("inf")
        weight[8] = 0.0
        check = otok.distill(f64(logits), index, value, 1.0, weight, 1.0)[0]
        assert check[6] == np.inf and check[0] == check[1] == check[2] == check[8] == 0.0
        check_distill(ops, dev, logits, index, value, 1.0, weight, 1.0)
        check_distill(ops, dev, logits, index, value, 0.5, weight, -2.0)


def test_distill_gradient_against_differences(ops, dev):
    """The gradient against central differences of the loss in 64 bits: the restatement's loss, shifted by 1e-5 (error
    of the difference: 1e-10 of the third derivative and 1e-11 of rounding, far below the float32 tolerance)."""
    rng = np.random.default_rng(2)
    logits, index, value = distill_inputs(2, 7, 3, torch.float32, dev, rng)
    index[0, 1] = index[0, 0]
    loss, d = torch.empty(2, device=dev), torch.empty(2, 7, device=dev)
    ops.distill_loss(logits, torch.from_numpy(index).to(dev), torch.from_numpy(value).to(dev), loss, temperature=1.5, dlogits=d)
    x = f64(logits)
    for j in range(7):
        hi, lo = x.copy(), x.copy()
        hi[:, j] += 1e-5
        lo[:, j] -= 1e-5
        diff = (otok.distill(hi, index, value, 1.5, None, 1.0)[0] - otok.distill(lo, index, value, 1.5, None, 1.0)[0]) / 2e-5
        assert np.all(np.abs(diff - f64(d)[:, j]) < 1e-5)


# ------------------------------------------------------------------ draw
def check_sample(ops, dev, logits, u, T, k, p, m, some=0.98):
    rows = logits.shape[0]
    out = torch.full((rows,), -7, dtype=torch.int64, device=dev)

    def arg(v, dt):
        return torch.from_numpy(np.asarray(v)).to(dev, dt) if isinstance(v, np.ndarray) else v
    ops.sample_tokens(logits, torch.from_numpy(u.astype(np.float32)).to(dev), out, temperature=arg(T, torch.float32), top_k=arg(k, torch.int32),
                      top_p=arg(p, torch.float32), min_p=arg(m, torch.float32))
    x, got = f64(logits), out.cpu().numpy()

    def at(v, r):
        return float(np.float32(v[r])) if isinstance(v, np.ndarray) else v
    clear = 0
    for r in range(rows):
        want, near = otok.sample(x[r], np.float32(u[r]), at(T, r), int(at(k, r)), at(p, r), at(m, r))
        if near > 2.0 ** -36:
            clear += 1
            assert got[r] == want, (r, got[r], want, near)
    assert clear >= some * rows
    return out


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.02), (1.3, 0, 0.9, 0.0), (1.0, 7, 1.0, 0.0), (0.7, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (2.0, 300, 0.5, 0.0),
            (1.0, 1, 0.3, 0.5), (1.0, 0, 0.0, 0.0), (1.0, 0, 0.999, 1.0), (1.0, 1500, 1.0, 0.0), (1.2, 1500, 0.95, 0.0), (30.0, 3000, 0.6, 0.0),
            (50.0, 0, 0.7, 0.5), (0.05, 2000, 0.999, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 5, 16, 17, 48, 64, 65, 100, 128, 129, 256, 257, 500, 1000, 1024, 1025, 2048, 2049, 4099, 16384, 16385, 20000, 32000])
def test_sample_tokens(ops, dev, dtype, V):
    rng = np.random.default_rng(V)
    rows = 40 if V <= 2048 else 6
    for i, s in enumerate(SETTINGS):
        extra, offset = ((0, 0), (8, 0), (5, 1))[i % 3]
        logits, _ = strided(rows, V, extra, dtype, dev, offset=offset)
        logits.copy_(torch.from_numpy(rng.standard_normal((rows, V)) * 2.5).to(dev))
        check_sample(ops, dev, logits, rng.random(rows) * (1 - 2.0 ** -24), *s)


@pytest.mark.parametrize("V", [33, 700, 9000])
def test_sample_tokens_settings_per_row(ops, dev, V):
    rng = np.random.default_rng(V + 1)
    rows = 64
    logits = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 2.5).to(dev)
    T = rng.uniform(0.3, 2.0, rows)
    T[:4] = [0.0, -1.0, np.nan, 5.0]
    k = rng.integers(-1, V + 5, rows).astype(np.float64)
    p = rng.uniform(0.1, 1.1, rows)
    m = rng.uniform(-0.05, 0.2, rows)
    check_sample(ops, dev, logits, rng.random(rows) * 0.999, T, k, p, m)
    # one number and a tensor of it give the same
    full = lambda v, dt: torch.full((rows,), v, dtype=dt, device=dev)  # noqa: E731
    u = torch.rand(rows, device=dev)
    a, b = torch.empty(rows, dtype=torch.int64, device=dev), torch.empty(rows, dtype=torch.int64, device=dev)
    ops.sample_tokens(logits, u, a, temperature=0.75, top_k=20, top_p=0.5, min_p=0.125)
    ops.sample_tokens(logits, u, b, temperature=full(0.75, torch.float32), top_k=full(20, torch.int32), top_p=full(0.5, torch.float32),
                      min_p=full(0.125, torch.float32))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [12, 90, 3000, 40000])
def test_sample_tokens_masks_ties_and_ends(ops, dev, dtype, V):
    rng = np.random.default_rng(V + 2)
    rows = 16
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.9, 8, 0.9, 0.01), (1.0, 0, 0.8, 0.0), (0.0, 3, 1.0, 0.0)):
        logits = torch.from_numpy(rng.standard_normal((rows, V)) * 2).to(dev, dtype)
        logits[0] = -float("inf")                                   # nothing to draw
        logits[1] = float("nan")
        logits[2] = torch.finfo(dtype).min                          # all the lowest: even
        logits[3, :] = -float("inf")
        logits[3, V - 1] = -2.0                                     # a single one
        logits[4] = 0.0                                             # all equal
        logits[5, ::2] = -float("inf")
        logits[6, 1::3] = float("nan")
        logits[7] = (logits[7] * 2).round() / 2                     # many ties
        logits[8, 5:8] = 30.0                                       # ties at the top
        logits[9] = torch.where(torch.arange(V, device=dev) % 2 == 0, 0.0, -0.0)
        logits[10, V // 2:] = torch.finfo(dtype).min
        logits[11, 3] = float("inf")
        logits[12, 2:4] = float("inf")
        logits[13] = -1e4 - torch.arange(V, device=dev) % 7
        u = rng.random(rows) * 0.999
        u[14], u[15] = 0.0, 1.0 - 2.0 ** -24
        out = check_sample(ops, dev, logits, u, T, k, p, m, some=0.5)
        assert out[0] == -1 and out[1] == -1 and out[3] == V - 1 and out[11] == 3 and out[12] in (2, 3)


def test_sample_tokens_numbers_outside_their_range(ops, dev):
    """u below 0 and NaN count as 0, u of 1 and more gives the last kept token."""
    logits = torch.zeros(5, 300, device=dev)
    u = torch.tensor([-3.0, float("nan"), 1.0, 2.0, float("inf")], device=dev)
    for V in (40, 300):
        out = torch.empty(5, dtype=torch.int64, device=dev)
        ops.sample_tokens(logits[:, :V], u, out)
        assert out.tolist() == [0, 0, V - 1, V - 1, V - 1]
        ops.sample_tokens(logits[:, :V], u, out, top_k=10)
        assert out.tolist() == [0, 0, 9, 9, 9]
    ops.sample_tokens(logits[:0], u[:0], out[:0])


@pytest.mark.parametrize("V", [9, 300, 5000])
def test_sample_tokens_extreme_temperatures(ops, dev, V):
    """Next to 0 only the largest logits are drawn, at infinity every finite one is alike."""
    rng = np.random.default_rng(V)
    logits = torch.from_numpy(rng.standard_normal((8, V)).astype(np.float32)).to(dev)
    logits[1, 2] = logits[1, 5] = 50.0
    logits[2, ::2] = -float("inf")
    for T in (1e-310, 1e-40, 1e-5, 1e30, float("inf")):
        for k, p in ((0, 1.0), (3, 1.0), (0, 0.5)):
            # (weights that are all 1, an even number of them: half their sum IS the sum of half of them, so every row is
            # decided on a border and none is clear)
            some = 0.0 if T >= 1e30 and p == 0.5 else 0.3
            check_sample(ops, dev, logits, rng.random(8) * 0.999, T, k, p, 0.0, some=some)
    T = np.array([1e-45, 1e-38, 1.0, 1e38, np.inf, 0.0, 1e-3, 1e3])
    check_sample(ops, dev, logits, rng.random(8) * 0.999, T, 4, 0.9, 0.0, some=0.3)


@pytest.mark.parametrize("V", [48, 2000])
def test_sample_tokens_follows_the_distribution(ops, dev, V):
    """Every token's borders: u on a fine grid visits the kept tokens in index order, each for its share of the grid (off by at
    most one point at either border)."""
    rng = np.random.default_rng(V)
    row = torch.from_numpy(rng.standard_normal(V).astype(np.float32) * 2).to(dev)
    N = 20000
    u = (torch.arange(N, device=dev, dtype=torch.float64) / N).float()
    out = torch.empty(N, dtype=torch.int64, device=dev)
    ops.sample_tokens(row.expand(N, V).contiguous(), u, out, temperature=0.8, top_k=30, top_p=0.9)
    w, _ = otok.kept(f64(row), 0.8, 30, 0.9, 0.0)
    count = np.bincount(out.cpu().numpy(), minlength=V)
    assert bool((out[1:] >= out[:-1]).all()) and np.all(np.abs(count - N * w / w.sum()) <= 1 + N * 2.0 ** -22) and np.all(count[w == 0] == 0)


# ------------------------------------------------------------------ streams, graphs, a run of them together
def test_token_ops_on_another_stream_and_replayed_from_a_graph(ops, dev):
    """Captured once, replayed between other work of the process on new inputs; two graphs at once have workspaces of their own."""
    rng = np.random.default_rng(4)
    n, V, D, K = 5000, 300, 96, 6

    def inputs():
        return (torch.from_numpy(rng.integers(-1, V, n)).to(dev), torch.from_numpy(rng.standard_normal((n, D)).astype(np.float32)).to(dev),
                torch.from_numpy(rng.standard_normal((64, V)).astype(np.float32)).to(dev), torch.rand(64, device=dev))
    tok, dout, logits, u = inputs()
    table = torch.randn(V, D, device=dev)
    index, value = torch.randint(0, V, (64, K), device=dev), torch.randn(64, K, device=dev)

    def buffers():
        return (torch.empty(n, D, device=dev), torch.empty(V, D, device=dev), torch.empty(64, device=dev), torch.empty(64, V, device=dev),
                torch.empty(64, dtype=torch.int64, device=dev))

    def go(b):
        ops.token_embed_fwd(tok, table, b[0], scale=2.0)
        ops.token_embed_bwd(tok, dout, b[1], accumulate=False)
        ops.distill_loss(logits, index, value, b[2], dlogits=b[3])
        ops.sample_tokens(logits, u, b[4], top_p=0.9)
    eager, other, ba, bb = buffers(), buffers(), buffers(), buffers()
    go(eager)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(other)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for b in (ba, bb):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(b)
        graphs.append(g)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(5):
        for dst, src in zip((tok, dout, logits, u), inputs()):
            dst.copy_(src)
        for b in ba + bb:
            b.zero_()
        go(eager)
        torch.cuda.synchronize()
        for s, g in zip(sides, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert float(dout.square().sum()) > 0
        for b in (ba, bb):
            assert all(torch.equal(x, y) for x, y in zip(eager, b)), rep


def test_token_ops_reject_other_types_and_places(ops, dev):
    from timeautodiff_amd import _lib
    tok, table, out = torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(5, 8, device=dev), torch.zeros(4, 8, device=dev)
    with pytest.raises(AssertionError):
        ops.token_embed_fwd(tok.int(), table, out)
    with pytest.raises(AssertionError):
        ops.token_embed_fwd(tok, table.half(), out)
    with pytest.raises(AssertionError):
        ops.token_embed_fwd(tok, table, out[:3])
    with pytest.raises(_lib.TadError):
        ops.token_embed_fwd(tok.cpu(), table, out)
    with pytest.raises(AssertionError):
        ops.token_embed_bwd(tok, out, table.bfloat16())
    with pytest.raises(_lib.TadError):
        ops.token_embed_bwd(tok, out[:1].expand(4, 8), table)                  # rows that overlap: no row stride
    with pytest.raises(AssertionError):
        ops.sample_tokens(out, torch.zeros(3, device=dev), tok)
    with pytest.raises(AssertionError):
        ops.sample_tokens(out, torch.zeros(4, device=dev), tok, top_k=torch.zeros(4, device=dev))
    with pytest.raises(AssertionError):
        ops.distill_loss(out, tok.view(4, 1), torch.zeros(4, 2, device=dev), torch.zeros(4, device=dev))
    with pytest.raises(_lib.TadError, match="temperature"):
        ops.distill_loss(out, tok.view(4, 1), torch.zeros(4, 1, device=dev), torch.zeros(4, device=dev), temperature=0.0)
    with pytest.raises(_lib.TadError, match="temperature"):
        ops.sample_tokens(out, torch.zeros(4, device=dev), tok, temperature=-1.0)


def test_token_column_model_end_to_end(ops, dev):
    """As a program uses them: codes -> lookup -> a product -> logits -> distillation loss and gradient -> back to the table,
    then a draw from the logits whose codes are looked up again.  float64 reference of the whole chain."""
    rng = np.random.default_rng(11)
    B, T, V, D, K, scale, tau = 6, 24, 53, 32, 8, 4.0, 1.5
    n = B * T
    tok = rng.integers(0, V, n)
    tok[-10:] = -1
    table, W = (rng.standard_normal((V, D)) * 0.2).astype(np.float32), (rng.standard_normal((V, D)) * 0.5).astype(np.float32)
    index = np.stack([rng.permutation(V)[:K] for _ in range(n)]).astype(np.int64)
    value = (rng.standard_normal((n, K)) * 2).astype(np.float32)
    weight = (tok >= 0).astype(np.float32)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    h, logits, loss = torch.empty(n, D, device=dev), torch.empty(n, V, device=dev), torch.empty(n, device=dev)
    ops.token_embed_fwd(d(tok), d(table), h, scale=scale)
    ops.linear_fwd(ops.F32, h, d(W), None, logits)
    dlogits = torch.empty_like(logits)
    ops.distill_loss(logits, d(index), d(value), loss, temperature=tau, row_weight=d(weight), grad_scale=1.0 / n, dlogits=dlogits)
    dh, dW, dtable = torch.empty_like(h), torch.zeros(V, D, device=dev), torch.zeros(V, D, device=dev)
    ops.linear_bwd_data(ops.F32, dlogits, d(W), dh)
    ops.linear_bwd_weight(ops.F32, dlogits, h, dW)
    ops.token_embed_bwd(d(tok), dh, dtable, scale=scale)
    h64 = otok.embed_fwd(tok, table, scale)
    l64 = h64 @ W.astype(np.float64).T
    loss64, dl64 = otok.distill(l64, index, value, tau, weight, 1.0 / n)
    dt64 = otok.embed_bwd(tok, dl64 @ W.astype(np.float64), V, scale)[0]

    def rel(a, b):
        return np.linalg.norm(f64(a) - b) / np.linalg.norm(b)
    # products of 32 and 53 float32 terms and the operators above: 100 roundings of 2^-24 at most
    assert rel(loss, loss64) < 1e-5 and rel(dlogits, dl64) < 1e-5 and rel(dtable, dt64) < 1e-5 and rel(dW, dl64.T @ h64) < 1e-5
    # the table's gradient against a difference of the whole chain
    v, c = int(tok[0]), 3
    ends = []
    for s in (1e-4, -1e-4):
        t64 = table.astype(np.float64).copy()
        t64[v, c] += s
        ends.append(otok.distill(otok.embed_fwd(tok, t64, scale) @ W.astype(np.float64).T, index, value, tau, weight, 1.0)[0].sum() / n)
    assert abs((ends[0] - ends[1]) / 2e-4 - float(dtable[v, c])) < 1e-5 * np.abs(dt64).max() + 1e-7
    u, code = torch.rand(n, device=dev), torch.empty(n, dtype=torch.int64, device=dev)
    ops.sample_tokens(logits, u, code, temperature=0.7, top_k=10)
    for r in range(0, n, 7):
        want, near = otok.sample(f64(logits[r]), float(u[r]), 0.7, 10, 1.0, 0.0)
        assert near < 2.0 ** -36 or int(code[r]) == want
    ops.token_embed_fwd(code, d(table), h)
    assert torch.equal(h, d(table)[code])


def test_decoder_codes_drawn_from_its_distributions(ops, dev):
    """DeapStack.decode_to_tensor(draw=...): the categorical columns are draws from the head outputs that ae.decoder returns,
    the rest of the table is what it is without."""
    from timeautodiff_amd import VAE
    torch.manual_seed(8)
    B, T, lat, nb, cards, nn = 9, 7, 4, 2, [3, 11, 70], 3
    F = nb + len(cards) + nn
    ae = VAE.DeapStack(1, nb, len(cards), nn, cards, F, 24, 2, 16, 8, lat)
    z, mask = torch.randn(B, T, lat, device=dev) * 3, (torch.rand(B, T, F, device=dev) < 0.8).float()
    heads = ae.decoder(z, mask)
    plain = ae.decode_to_tensor(z, mask)
    u = torch.rand(len(cards), B, T, device=dev)
    got = ae.decode_to_tensor(z, mask, draw=dict(temperature=1.5, top_p=0.95, u=u))
    keep = [c for c in range(F) if not nb <= c < nb + len(cards)]
    assert torch.equal(got[..., keep], plain[..., keep])
    for j, card in enumerate(cards):
        logits = f64(heads["cats"][j]).reshape(B * T, card)
        for r in range(B * T):
            want, near = otok.sample(logits[r], float(u[j].reshape(-1)[r]), 1.5, 0, 0.95, 0.0)
            assert near < 2.0 ** -36 or int(got[..., nb + j].reshape(-1)[r]) == want
    assert bool((ae.decode_to_tensor(z, mask, draw=dict(top_k=1)) == plain).all())          # the largest alone: the argmax
    assert not torch.equal(ae.decode_to_tensor(z, mask, draw=dict(temperature=5.0)), plain)
    with pytest.raises(ValueError):
        ae.decode_to_tensor(z, mask, draw=dict(u=u[:2]))


@pytest.mark.parametrize("dtype,V,rows", [(torch.float32, 2500, 300), (torch.bfloat16, 9000, 257), (torch.bfloat16, 60000, 260), (torch.float32, 40000, 258),
                                          (torch.bfloat16, 70001, 5)])
def test_sample_tokens_many_rows_and_long_ones(ops, dev, dtype, V, rows):
    """Every size of workgroup that a row gets, for few rows and for many (a share of the rows is checked)."""
    rng = np.random.default_rng(V)
    logits = (torch.randn(rows, V, device=dev, generator=torch.Generator(device=dev).manual_seed(V)) * 2.5).to(dtype)
    u = rng.random(rows) * 0.999
    ask = np.arange(0, rows, max(1, rows // 12))
    for T, k, p, m in [(1.0, 0, 0.9, 0.0), (0.5, 0, 0.9, 0.0), (0.9, 60, 0.95, 0.02), (1.0, 0, 1.0, 0.0), (1.0, 700, 0.99, 0.0), (0.0, 0, 1.0, 0.0)]:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
        ops.sample_tokens(logits, torch.from_numpy(u.astype(np.float32)).to(dev), out, temperature=T, top_k=k, top_p=p, min_p=m)
        for r in ask:
            want, near = otok.sample(f64(logits[r]), np.float32(u[r]), T, k, p, m)
            assert near < 2.0 ** -36 or int(out[r]) == want, (T, k, p, m, r)


@pytest.mark.parametrize("V", [150001, 300000])
def test_sample_tokens_very_long_rows(ops, dev, V):
    """Rows whose sums leave fewer bits to a weight (off by 2^-43 of the largest at 300000 logits, 3e5 of them: 2^-33 of the
    sum at the very most where it is the largest alone, 2^-42 where they are alike)."""
    rng = np.random.default_rng(V)
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.from_numpy(rng.standard_normal((3, V)) * 2.5).to(dev, dtype)
        u = rng.random(3)
        for T, k, p, m in SETTINGS:
            check_sample(ops, dev, logits, u, T, k, p, m, some=0.6)


# a list of candidates holds few of them; its length, and whether each is compared with each, hang on top-k, the row and the rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,tops", [(3, 2500, (111, 112, 113, 160, 224, 225, 448)), (260, 2500, (112, 113, 160, 161, 225)),
                                         (2, 30000, (224, 225, 320, 321, 448)), (257, 50000, (225, 320)), (2, 70000, (224, 300, 447, 448, 449))])
def test_sample_tokens_top_k_around_the_lists_lengths(ops, dev, dtype, rows, V, tops):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((rows, V)) * 2.5
    x[0] = np.round(x[0] * 4) / 4                # few values, many ties at the cut
    x[1, :400] += 9.0                            # the largest side by side
    logits = torch.from_numpy(x).to(dev, dtype)
    for k in tops:
        check_sample(ops, dev, logits, rng.random(rows) * (1 - 2.0 ** -24), 1.0, k, 0.95, 0.001)
        if rows < 9:
            check_sample(ops, dev, logits, rng.random(rows) * (1 - 2.0 ** -24), 1.5, k, 1.0, 0.0)


@pytest.mark.parametrize("V", [3000, 20000])
def test_sample_tokens_of_peaked_rows(ops, dev, V):
    """Rows where a few logits hold the mass, also at one end of the row, with top-p alone and with everything."""
    rng = np.random.default_rng(V)
    rows = 12
    x = rng.standard_normal((rows, V))
    x[:, :5] += 9.0
    x[3:6, V - 3:] += 12.0
    x[6, 77] = 60.0
    x[7] = np.floor(x[7])                       # few values, many ties
    x[8], x[9] = np.sort(x[8]), -np.sort(x[9])  # in order
    for dtype in (torch.float32, torch.bfloat16):
        for s in SETTINGS:
            check_sample(ops, dev, torch.from_numpy(x).to(dev, dtype), rng.random(rows) * 0.999, *s, some=0.8)


def test_token_ops_are_traced_with_their_costs(ops, dev):
    """An installed LaunchTrace sees every call with its bytes: each operand and result once."""
    tok, table, out = torch.randint(0, 5, (30,), device=dev), torch.randn(5, 8, device=dev), torch.empty(30, 8, device=dev)
    logits, u, code = torch.randn(6, 40, device=dev), torch.rand(6, device=dev), torch.empty(6, dtype=torch.int64, device=dev)
    index, value, loss = torch.randint(0, 40, (6, 3), device=dev), torch.randn(6, 3, device=dev), torch.empty(6, device=dev)
    with ops.LaunchTrace() as tr:
        ops.token_embed_fwd(tok, table, out)
        ops.token_embed_bwd(tok, out, table)
        ops.token_embed_bwd(tok, out, table, accumulate=False)
        ops.distill_loss(logits, index, value, loss)
        ops.distill_loss(logits, index, value, loss, dlogits=logits)
        ops.sample_tokens(logits, u, code)
    seen = {}
    for key, (calls, ms, flops, nbytes, issued) in tr.summary().items():
        seen.setdefault(key[0], []).append((calls, nbytes))
    assert seen["tad_token_embed_fwd"] == [(1, 30 * 8 + 5 * 32 + 30 * 32)]
    assert sum(c for c, _ in seen["tad_token_embed_bwd"]) == 2 and sum(c for c, _ in seen["tad_distill_loss"]) == 2
    assert seen["tad_sample_tokens"] == [(1, 6 * (160 + 12))]
