"""Token family where it can go wrong: sums of whole numbers, which leave a gradient no tolerance, over every form of its
sort and cut; workspaces of exactly the stated size whatever they hold; teacher's entries on masked logits; rows cut out of
wider tensors; draws of infinite logits, and next to a border.

Restatement: oracle/tokens.py.  e = 2^-24 is half a float32 step."""
import numpy as np
import pytest
import torch

from oracle import tokens as otok

pytestmark = pytest.mark.gpu

E24 = 2.0 ** -24


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


def tokens_of(kind, n, V, rng):
    if kind == "same":
        return np.full(n, V // 2)
    if kind == "padding":
        return np.full(n, V + 3)
    if kind == "spread":
        return rng.integers(0, V, n)
    tok = np.minimum(((V + 1.0) ** rng.random(n)).astype(np.int64) - 1, V - 1)
    if kind == "ragged":
        tok[rng.random(n) < 0.3] = rng.choice([-1, V, 1 << 40])
        tok[n - n // 5:] = -1
    return tok


# ------------------------------------------------------------------ gradient of the lookup
# one launch (n <= 4096 and few rows); all pairs compared (n <= 8192); digits: one of 9 bits with every bin in use (511 rows and
# padding), two of 5 and of 9, three of 7; waves of 64 positions (270000); one, two, four columns a lane, two packs of four (bf16)
GRADIENTS = [(4096, 100, 256, torch.float32), (4096, 3, 260, torch.bfloat16), (4097, 40, 128, torch.float32), (8192, 500, 128, torch.bfloat16),
             (8193, 500, 128, torch.float32), (8193, 3, 520, torch.bfloat16), (20000, 511, 520, torch.bfloat16), (20000, 512, 260, torch.float32),
             (20001, 131072, 128, torch.float32), (20000, 300000, 20, torch.bfloat16), (70001, 37, 256, torch.bfloat16), (70001, 4000, 132, torch.float32),
             (140001, 1000, 3, torch.float32), (270000, 1000, 8, torch.float32)]


@pytest.mark.parametrize("kind", ["zipf", "ragged", "same", "spread", "padding"])
@pytest.mark.parametrize("n,V,D,dtype", GRADIENTS)
def test_gradient_of_whole_numbers_is_exact(ops, dev, kind, n, V, D, dtype):
    """Terms 1 .. 8 and a scale of 1/2: every sum is exact in any order (270000 * 8 < 2^24), so a row, a chunk or an edge left
    out or taken twice shows whatever the length of a run."""
    rng = np.random.default_rng(n + V + D)
    tok = torch.from_numpy(tokens_of(kind, n, V, rng))
    terms = torch.from_numpy(rng.integers(1, 9, (n, D)))
    fine = (tok >= 0) & (tok < V)
    want = torch.zeros(V, D, dtype=torch.int64).index_add_(0, tok[fine], terms[fine]).to(dev).double() * 0.5
    for extra in (0, 3):
        wide = torch.full((n, D + extra), float("nan"), dtype=dtype, device=dev)
        dout = wide[:, :D]
        dout.copy_(terms.to(dev))
        dout[~fine.to(dev)] = float("nan")                      # what padding holds has no share
        table = torch.full((V, D + extra), 3.0, device=dev)
        for accumulate in (False, True):
            table.fill_(3.0)
            ops.token_embed_bwd(tok.to(dev), dout, table[:, :D], scale=0.5, accumulate=accumulate)
            assert torch.equal(table[:, :D].double(), want + 3.0 if accumulate else want)
            assert bool((table[:, D:] == 3.0).all())


@pytest.mark.parametrize("n,V,D,dtype", GRADIENTS)
def test_gradient_of_long_runs(ops, dev, n, V, D, dtype):
    """A term goes through at most 256 additions of the one launch, or 64 of its wave, 8 of the workgroup and one for every fourth
    chunk of 64 or more positions: 300 + n / 256 roundings, whatever the number of a row's terms; twice, the same bits."""
    rng = np.random.default_rng(n)
    x = torch.from_numpy(rng.standard_normal((n, D)).astype(np.float32)).to(dev, dtype)
    for kind in ("same", "zipf"):
        tok = torch.from_numpy(tokens_of(kind, n, V, rng)).to(dev)
        a, b = torch.empty(V, D, device=dev), torch.empty(V, D, device=dev)
        ops.token_embed_bwd(tok, x, a, scale=1.25, accumulate=False)
        ops.token_embed_bwd(tok, x, b, scale=1.25, accumulate=False)
        assert torch.equal(a, b)
        d, t = x.cpu().double(), tok.cpu()
        want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, t, d) * 1.25
        size = torch.zeros(V, D, dtype=torch.float64).index_add_(0, t, d.abs()) * 1.25
        assert bool(((a.cpu().double() - want).abs() <= E24 * (300 + n / 256) * size).all())


@pytest.mark.parametrize("n", [300, 9000])
def test_accumulating_gradient_of_a_very_large_table(ops, dev, n):
    """Rows of a table of more than 2^29 that no token names are not touched, so their number costs nothing."""
    V = (1 << 29) + 7
    rng = np.random.default_rng(n)
    tok = rng.integers(0, V, n)
    tok[::3] = V - 1 - rng.integers(0, 40, tok[::3].size)
    terms = rng.integers(1, 9, n)
    table = torch.zeros(V, 1, device=dev)
    ops.token_embed_bwd(torch.from_numpy(tok).to(dev), torch.from_numpy(terms).to(dev).float().view(n, 1), table)
    at, inverse = np.unique(tok, return_inverse=True)
    want = np.bincount(inverse, weights=terms)
    assert np.array_equal(f64(table[torch.from_numpy(at).to(dev), 0]), want)
    assert int(torch.count_nonzero(table)) == at.size


@pytest.mark.parametrize("n,V,D,dtype", [(4096, 3, 9, torch.float32), (5000, 40, 9, torch.float32), (5000, 5000, 128, torch.bfloat16), (8192, 2, 520, torch.bfloat16),
                                         (9001, 500, 520, torch.bfloat16), (9001, 300000, 4, torch.float32), (70001, 3, 128, torch.float32),
                                         (70001, 70000, 9, torch.bfloat16)])
def test_gradient_in_a_workspace_of_the_stated_size(ops, dev, n, V, D, dtype):
    """Forms that sort and join: nothing is written beside the workspace, and what it holds before the call changes nothing."""
    rng = np.random.default_rng(n + D)
    nb = ops.token_embed_bwd_workspace_bytes(n, D)
    buf = torch.empty(nb + 512, dtype=torch.uint8, device=dev)
    for kind in ("zipf", "same"):
        tok = torch.from_numpy(tokens_of(kind, n, V, rng)).to(dev)
        for extra in (0, 4, 3):
            dout = torch.from_numpy(rng.standard_normal((n, D + extra))).to(dev, dtype)[:, :D]
            want, got = torch.empty(V, D, device=dev), torch.empty(V, D, device=dev)
            ops.token_embed_bwd(tok, dout, want, accumulate=False)
            for held in (0xAB, 0xFF, 0x00):                     # (0xFF: every float32 in it a NaN)
                buf.fill_(held)
                ops.token_embed_bwd(tok, dout, got, accumulate=False, workspace=buf[256:256 + nb])
                assert torch.equal(want, got)
                assert bool((buf[:256] == held).all()) and bool((buf[256 + nb:] == held).all())


# ------------------------------------------------------------------ distillation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [6, 48, 700, 9000])
def test_distill_loss_of_entries_on_masked_logits(ops, dev, dtype, V):
    """A logit masked with the type's lowest value is finite: p = 0 there, and the loss of an entry on it is w tau q (max - logit) to
    within the others' share, finite wherever float32 holds it.  q is off by e (16 A + K + 64) relative, A the range of value /
    tau; four roundings more."""
    rng = np.random.default_rng(V)
    rows, K = 12, 5
    for tau in (1.0, 0.25, 3.0):
        x = rng.standard_normal((rows, V)) * 2.5
        logits = torch.from_numpy(x).to(dev, dtype)
        low = torch.finfo(dtype).min
        logits[:, 1], logits[:, V - 1] = low, low
        index = np.tile(np.array([0, 1, 2, V - 1, 3]), (rows, 1))
        value = rng.standard_normal((rows, K)).astype(np.float32)
        index[0] = [1, 1, V - 1, 1, V - 1]                       # every entry on a masked logit
        logits[1, 2] = -low                                      # max - logit itself is more than float32 holds
        weight = rng.uniform(0.02, 0.3, rows).astype(np.float32)
        weight[2] = 8.0
        loss, d = torch.empty(rows, device=dev), torch.empty(rows, V, dtype=dtype, device=dev)
        ops.distill_loss(logits, torch.from_numpy(index).to(dev), torch.from_numpy(value).to(dev), loss, temperature=tau,
                         row_weight=torch.from_numpy(weight).to(dev), dlogits=d)
        want, grad = otok.distill(f64(logits), index, value, tau, weight, 1.0)
        got = f64(loss)
        most = float(np.finfo(np.float32).max)
        A = float(np.ptp(value, axis=1).max()) / tau
        rel = E24 * (16 * A + K + 64 + 4)
        fits, over = want < most * (1 - rel), want > most * (1 + rel)
        assert fits.sum() >= 8 and np.all(fits | over)
        assert np.all(np.isinf(got[over]) & (got[over] > 0))
        assert np.all(np.abs(got[fits] - want[fits]) <= rel * want[fits]), (got, want)
        # p as in the loss of any other row: arguments of up to A' = range of the live logits / tau
        live = np.ptp(x, axis=1).max() / tau + np.log(V)
        err = E24 * (16 * max(A, live) + V / 32 + K + 64)
        for r in range(rows):
            if r == 1:
                continue                                         # (its largest logit holds all of p)
            q = np.exp(value[r].astype(np.float64) / tau)
            q /= q.sum()
            qq = np.zeros(V)
            np.add.at(qq, index[r], q)
            g = weight[r] * tau
            tol = g * 2 * err * (np.abs(grad[r]) / g + 2 * qq) + ((2.0 ** -8 if dtype == torch.bfloat16 else E24) + 3 * E24) * np.abs(grad[r]) + 1e-37
            assert np.all(np.abs(f64(d[r]) - grad[r]) <= tol), r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [16, 17, 32, 33, 49, 128, 129, 256, 257, 512, 513, 1024, 1025, 16384, 16385, 32768, 32769])
def test_distill_loss_where_its_forms_change(ops, dev, dtype, V):
    from test_gpu_tokens import check_distill, distill_inputs
    rng = np.random.default_rng(V)
    for extra, offset in ((0, 0), (3, 1)):
        logits, index, value = distill_inputs(5, V, 12, dtype, dev, rng, extra, offset)
        index[1, 3] = index[1, 7]
        check_distill(ops, dev, logits, index, value, 1.25, None, 0.5)
        check_distill(ops, dev, logits, index, value, 1.25, None, 0.5, inplace=True)


# ------------------------------------------------------------------ rows out of wider tensors
@pytest.mark.parametrize("B,T,V", [(4, 5, 300), (3, 1, 40), (1, 6, 17)])
def test_last_step_of_a_sequence(ops, dev, B, T, V):
    """x[:, -1:, :] has the rows of x[:, -1, :]: a dimension of one element has no stride of its own."""
    rng = np.random.default_rng(B * T)
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).to(dev)
    a, b = x[:, -1:, :], x[:, -1, :]
    u = torch.rand(B, device=dev)
    got, want = torch.empty(B, 1, dtype=torch.int64, device=dev), torch.empty(B, dtype=torch.int64, device=dev)
    ops.sample_tokens(a, u, got, top_p=0.9)
    ops.sample_tokens(b, u, want, top_p=0.9)
    assert torch.equal(got.view(-1), want)
    index, value = torch.randint(0, V, (B, 1, 3), device=dev), torch.randn(B, 1, 3, device=dev)
    da, db = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    la, lb = torch.empty(B, 1, device=dev), torch.empty(B, device=dev)
    ops.distill_loss(a, index, value, la, dlogits=da[:, -1:, :])
    ops.distill_loss(b, index[:, 0], value[:, 0], lb, dlogits=db[:, -1, :])
    assert torch.equal(la.view(-1), lb) and torch.equal(da, db)
    table, tok = torch.randn(9, V, device=dev), torch.randint(0, 9, (B, 1), device=dev)
    ops.token_embed_fwd(tok, table, da[:, -1:, :])
    assert torch.equal(da[:, -1], table[tok[:, 0]]) and bool((da[:, :-1] == 7.0).all())
    ga, gb = torch.empty_like(table), torch.empty_like(table)
    ops.token_embed_bwd(tok, a, ga, accumulate=False)
    ops.token_embed_bwd(tok[:, 0], b, gb, accumulate=False)
    assert torch.equal(ga, gb)
    with pytest.raises(AssertionError):                          # two strides: no rows
        ops.sample_tokens(torch.zeros(4, 6, V, device=dev)[:, :3], torch.rand(12, device=dev), torch.empty(12, dtype=torch.int64, device=dev))


# ------------------------------------------------------------------ draw
@pytest.mark.parametrize("V", [12, 100, 3000, 40000])
def test_infinite_logits_count_as_the_largest_number(ops, dev, V):
    """+inf is the largest float32 number: the two tie, and the lowest index is taken."""
    logits = torch.randn(3, V, device=dev)
    most = torch.finfo(torch.float32).max
    logits[0, V - 2], logits[0, 5] = float("inf"), most
    logits[1, 4], logits[1, V - 1] = float("inf"), most
    logits[2, 7], logits[2, V - 3] = most, most
    out = torch.empty(3, dtype=torch.int64, device=dev)
    ops.sample_tokens(logits, torch.rand(3, device=dev), out, temperature=0.0)
    assert out.tolist() == [5, 4, 7]
    for opt in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.5)):
        ops.sample_tokens(logits, torch.zeros(3, device=dev), out, **opt)
        assert out.tolist() == [5, 4, 7], opt
        ops.sample_tokens(logits, torch.full((3,), 0.999, device=dev), out, **opt)
        assert out.tolist() == [V - 2, V - 1, V - 3], opt
    ops.sample_tokens(logits, torch.full((3,), 0.999, device=dev), out, top_k=1)
    assert out.tolist() == [5, 4, 7]


@pytest.mark.parametrize("V,F", [(500, 44), (2048, 42), (32000, 44), (131072, 44), (300000, 42)])
def test_draw_next_to_a_border(ops, dev, V, F):
    """One logit leads and all others are equal, so that their weights are rounded alike and the roundings add up.  Each weight is
    off by at most 2^-(F+1) of the largest, so a border by at most V times that (u times the sum is a whole number of 2^-F too: 4
    more); sums in float64 to 2^-48 of them."""
    N = 64
    # (tails that hold a share of the row, next to which 2^-(F+1) is small)
    for tail in (-6.0, -18.0):
        w = np.exp(tail)
        for lead in (0, V // 3, V - 1):
            row = torch.full((V,), tail, device=dev)
            row[lead] = 0.0
            c = np.arange(1, V + 1) * w
            c[lead:] += 1.0 - w
            # numbers that fall among the tail before the leader and behind it, where there are any
            before, behind = lead * w / c[-1], 1.0 - (V - 1 - lead) * w / c[-1]
            g = np.random.default_rng(V + lead)
            u = np.concatenate([g.uniform(0.0, max(before, 1e-9), N // 2), g.uniform(min(behind, 1 - 1e-7), 1.0, N // 2)]).astype(np.float32)
            u = np.minimum(u, np.float32(1 - E24))
            for dtype in (torch.bfloat16, torch.float32):
                out = torch.empty(N, dtype=torch.int64, device=dev)
                ops.sample_tokens(row.to(dtype).expand(N, V).contiguous(), torch.from_numpy(u).to(dev), out)
                at = out.cpu().numpy()
                off = (V + 4) * 2.0 ** -(F + 1) + c[-1] * 2.0 ** -48
                target = u.astype(np.float64) * c[-1]
                assert np.all(target <= c[at] + off) and np.all(target >= np.where(at > 0, c[at - 1], 0.0) - off)


@pytest.mark.parametrize("V", [30, 700, 5000])
def test_weights_below_half_a_unit_are_never_drawn(ops, dev, V):
    """e^-40 is below 2^-45: such a logit is kept by a filter that counts, and has no mass."""
    logits = torch.full((3, V), -40.0, device=dev)
    logits[:, 3] = 0.0
    u = torch.tensor([0.0, 0.5, 1.0], device=dev)
    out = torch.empty(3, dtype=torch.int64, device=dev)
    for opt in (dict(), dict(top_k=10), dict(top_p=0.99), dict(top_k=10, min_p=1e-30)):
        ops.sample_tokens(logits, u, out, **opt)
        assert out.tolist() == [3, 3, 3], opt


def test_decoder_code_of_a_column_without_a_number_to_draw(ops, dev):
    """Where no logit of a column is a number above -inf the drawn code is -1; the other columns are what they are without it."""
    from timeautodiff_amd import VAE
    torch.manual_seed(3)
    B, T, lat, nb, cards, nn = 3, 4, 4, 1, [5, 90], 2
    F = nb + len(cards) + nn
    ae = VAE.DeapStack(1, nb, len(cards), nn, cards, F, 24, 2, 16, 8, lat)
    z, mask = torch.randn(B, T, lat, device=dev), torch.ones(B, T, F, device=dev)
    u = torch.rand(len(cards), B, T, device=dev)
    fine = ae.decode_to_tensor(z, mask, draw=dict(u=u))
    assert bool((fine[..., nb:nb + 2] >= 0).all())
    for number in (float("nan"), -float("inf")):
        with torch.no_grad():
            ae.get_parameter("cats_linears.0.bias").fill_(number)
        got = ae.decode_to_tensor(z, mask, draw=dict(u=u))
        assert bool((got[..., nb] == -1).all()) and bool((ae.decode_to_tensor(z, mask)[..., nb] == 0).all())
        rest = [c for c in range(F) if c != nb]
        assert torch.equal(got[..., rest], fine[..., rest])
