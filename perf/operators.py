"""The operators at the two ends of a discrete column: what reads a code (the embedding lookup and its gradient) and what
answers with one (a loss on its logits against a teacher's, the draw of a code from them).

Each of them twice: in a plain form of elementary torch operations, and as the calls that a program makes of
``timeautodiff_amd.ops``.  ``own`` says which of the two ``run`` computes.

    embed_fwd   out[i] = scale * table[tokens[i]]                                  a token outside [0, V): a row of zeros
    embed_bwd   dtable[v] = scale * sum of dout[i] over the i with tokens[i] = v   ... and no share in any gradient
    distill     q = softmax(teacher's k logits / tau), p = softmax(logits / tau):  an index outside [0, V) is no entry
                loss[r] = w[r] tau^2 sum_k q_k (ln q_k - ln p[index_k]),   dlogits = grad_scale * d loss[r] / d logits
    sample      w = exp((logits - max) / T); kept: the top_k largest, of those the shortest prefix (largest first) that
                holds top_p of their mass, of those the ones with w >= min_p; the answer is the lowest index at which the
                running sum of the kept w, by index, exceeds u times their sum.  Ties go to the lowest index, T = 0 is argmax
"""
import math

import torch

own = False

F32, B16 = "float32", "bfloat16"


def listed():
    return [
        # ---- lookup
        # one decoding step of a batch of 32 sequences: latency
        dict(name="embed_fwd step", op="embed_fwd", n=32, vocab=32000, dim=1024, table=B16, out=B16, pad=0.0),
        # a training batch of 4096 windows of 24 rows, one discrete field, fp32 master table -> bf16 operand of a product
        dict(name="embed_fwd field", op="embed_fwd", n=98304, vocab=500, dim=128, table=F32, out=B16, pad=0.0),
        # a prompt batch, right-padded
        dict(name="embed_fwd prompt", op="embed_fwd", n=32768, vocab=65536, dim=2048, table=B16, out=B16, pad=0.05),
        # ---- gradient of the lookup
        # the reference's batch: 100 windows of 24 rows, a field of 50 values
        dict(name="embed_bwd small", op="embed_bwd", n=2400, vocab=50, dim=128, dout=F32, pad=0.0),
        # 4096 windows of 24 rows, a field of 500 values: every row of the table gets hundreds of terms
        dict(name="embed_bwd field", op="embed_bwd", n=98304, vocab=500, dim=128, dout=F32, pad=0.0),
        # a large vocabulary: most of the work is the table's own gradient
        dict(name="embed_bwd vocab", op="embed_bwd", n=32768, vocab=65536, dim=2048, dout=B16, pad=0.05),
        # ---- distillation
        # validation pass over a small vocabulary: the loss alone
        dict(name="distill loss", op="distill", rows=512, vocab=32001, k=32, dtype=F32, grad=False, tau=2.0, pad=0.1),
        # the categorical head of a column of 48 values, training: many short rows
        dict(name="distill heads", op="distill", rows=98304, vocab=48, k=8, dtype=F32, grad=True, tau=1.5, pad=0.0),
        # a language-model head in training
        dict(name="distill train", op="distill", rows=4096, vocab=131072, k=64, dtype=B16, grad=True, tau=1.0, pad=0.1),
        # ---- draw
        # one request's next token: latency
        dict(name="sample one", op="sample", rows=1, vocab=32000, dtype=B16, per_row=False, top_k=50, top_p=0.95, min_p=0.02, temp=0.8, gap=0),
        # codes of a generated table's column: many short rows, cut out of a wider matrix of heads
        dict(name="sample heads", op="sample", rows=98304, vocab=48, dtype=F32, per_row=False, top_k=0, top_p=0.9, min_p=0.0, temp=1.0, gap=22),
        # a serving batch, every request with its own settings
        dict(name="sample batch", op="sample", rows=256, vocab=131072, dtype=B16, per_row=True, top_k=64, top_p=0.95, min_p=0.05, temp=0.9, gap=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "distill", "sample"])
    dt = rng.choice([F32, B16])
    if op in ("embed_fwd", "embed_bwd"):
        n, vocab = _log(rng, 1, 131072), _log(rng, 2, 131072)
        dim = _log(rng, 16, 4096)
        if rng.random() < 0.7:
            dim = -(-dim // 8) * 8            # most models' widths; the others are odd
        dim = max(16, min(dim, (1 << 26) // n, (1 << 27) // vocab))
        pad = rng.choice([0.0, 0.05, 0.3])
        if op == "embed_fwd":
            return dict(op=op, n=n, vocab=vocab, dim=dim, table=dt, out=rng.choice([F32, B16]), pad=pad)
        return dict(op=op, n=n, vocab=vocab, dim=dim, dout=dt, pad=pad)
    if op == "distill":
        rows, vocab = _log(rng, 1, 98304), _log(rng, 8, 131072)
        rows = max(1, min(rows, (1 << 28) // vocab))
        return dict(op=op, rows=rows, vocab=vocab, k=min(vocab, _log(rng, 1, 128)), dtype=dt, grad=rng.random() < 0.7,
                    tau=round(rng.uniform(0.5, 4.0), 3), pad=rng.choice([0.0, 0.1]))
    rows, vocab = _log(rng, 1, 98304), _log(rng, 2, 131072)
    rows = max(1, min(rows, (1 << 25) // vocab))
    return dict(op=op, rows=rows, vocab=vocab, dtype=dt, per_row=rng.random() < 0.5, top_k=rng.choice([0, 1, 20, 64, 300]),
                top_p=rng.choice([1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.02, 0.1]),
                temp=rng.choice([0.0, 0.6, 1.0, 1.7]), gap=rng.choice([0, 0, 8, 5]))


def _tokens(case, g):
    """Tokens as a text or a field has them: the share of the v-th most frequent falls like 1 / v; some are padding (-1)."""
    n, v = case["n"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    tok = (((v + 1.0) ** u).floor().long() - 1).clamp_(0, v - 1)
    if case["pad"]:
        tok[n - int(n * case["pad"]):] = -1
    return tok


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f32 = dict(device="cuda", dtype=torch.float32)
    op = case["op"]
    s = dict(case=case, op=op)
    if op == "embed_fwd":
        s["tokens"] = _tokens(case, g)
        s["table"] = torch.randn(case["vocab"], case["dim"], generator=g, **f32).mul_(0.02).to(getattr(torch, case["table"]))
        s["out"] = torch.empty(case["n"], case["dim"], device="cuda", dtype=getattr(torch, case["out"]))
        s["scale"] = math.sqrt(case["dim"])
    elif op == "embed_bwd":
        s["tokens"] = _tokens(case, g)
        s["dout"] = torch.randn(case["n"], case["dim"], generator=g, **f32).to(getattr(torch, case["dout"]))
        s["dtable"] = torch.empty(case["vocab"], case["dim"], **f32)
        s["scale"] = math.sqrt(case["dim"])
    elif op == "distill":
        rows, v, k, dt = case["rows"], case["vocab"], case["k"], getattr(torch, case["dtype"])
        logits = torch.empty(rows, v, device="cuda", dtype=dt)
        step = max(1, (1 << 26) // v)
        for lo in range(0, rows, step):
            part = torch.randn(min(step, rows - lo), v, generator=g, **f32)
            logits[lo:lo + step] = part.mul_(2.5).to(dt)
        s["logits"] = logits
        # the teacher's largest logits: indices a random odd stride apart (now and then one comes twice), descending values;
        # the last entry of every fourth row is missing where there are several, and the share `pad` of the rows counts nothing
        start = torch.randint(0, v, (rows, 1), generator=g, device="cuda")
        step = 2 * torch.randint(0, max(1, v // 2), (rows, 1), generator=g, device="cuda") + 1
        s["index"] = (start + step * torch.arange(k, device="cuda")) % v
        s["value"] = torch.randn(rows, k, generator=g, **f32).mul_(2.0).add_(6.0).sort(1, descending=True)[0].contiguous()
        if k > 1:
            s["index"][::4, k - 1] = -1
        w = torch.rand(rows, generator=g, **f32).add_(0.5)
        if case["pad"]:
            w[rows - int(rows * case["pad"]):] = 0.0
        s["weight"] = w
        s["loss"] = torch.empty(rows, **f32)
        s["dlogits"] = torch.empty(rows, v, device="cuda", dtype=dt) if case["grad"] else None
        s["grad_scale"] = 1.0 / rows
    else:
        rows, v, dt = case["rows"], case["vocab"], getattr(torch, case["dtype"])
        wide = torch.randn(rows, v + case["gap"], generator=g, **f32).mul_(2.5)
        peak = torch.randint(0, v, (rows, min(4, v)), generator=g, device="cuda")
        wide.scatter_add_(1, peak, torch.rand(rows, min(4, v), generator=g, **f32) * 8.0)
        s["logits"] = wide.to(dt)[:, :v]
        s["u"] = torch.rand(rows, generator=g, **f32)
        s["out"] = torch.empty(rows, dtype=torch.int64, device="cuda")
        par = dict(temperature=case["temp"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        if case["per_row"]:
            # every request its own: around the case's values
            def jit(x, lo, hi):
                return (x * (lo + (hi - lo) * torch.rand(rows, generator=g, **f32))).contiguous()
            par = dict(temperature=jit(case["temp"], 0.7, 1.3), top_k=jit(float(case["top_k"]), 0.3, 1.7).ceil().int(),
                       top_p=jit(case["top_p"], 0.9, 1.0), min_p=jit(case["min_p"], 0.2, 1.8))
        s["par"] = par
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _embed_fwd(s):
    tok, table = s["tokens"], s["table"]
    fine = (tok >= 0) & (tok < table.shape[0])
    row = table[torch.where(fine, tok, 0)].float() * s["scale"]
    return torch.where(fine[:, None], row, 0.0).to(s["out"].dtype)


def _embed_bwd(s):
    tok, dout, (v, d) = s["tokens"], s["dout"], s["dtable"].shape
    fine = (tok >= 0) & (tok < v)
    # long sums in parts of about 16 terms a row of the table, which are added at the end
    parts = -(-tok.numel() // (16 * v))
    at = torch.where(fine, tok, 0) + v * (torch.arange(tok.numel(), device=tok.device) % parts)
    grad = torch.zeros(parts * v, d, device=dout.device)
    grad.index_add_(0, at, torch.where(fine[:, None], dout.float(), 0.0))
    return (grad.view(parts, v, d).sum(0) if parts > 1 else grad) * s["scale"]


def _distill(s):
    x, idx, tau, w = s["logits"].float() / s["case"]["tau"], s["index"], s["case"]["tau"], s["weight"]
    v = x.shape[1]
    fine = (idx >= 0) & (idx < v)
    at = torch.where(fine, idx, 0)
    m = x.max(1, keepdim=True)[0]
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    t = torch.where(fine, s["value"] / tau, -math.inf)
    t = t - t.max(1, keepdim=True)[0]
    e = t.exp()
    total = e.sum(1, keepdim=True)
    q, logq = e / total, t - total.log()
    loss = (w * tau * tau) * torch.where(q > 0, q * (logq - (x.gather(1, at) - lse)), 0.0).sum(1)
    if s["dlogits"] is None:
        return loss
    d = (x - lse).exp().scatter_add_(1, at, torch.where(fine, -q, 0.0))
    return loss, (d * (w * (tau * s["grad_scale"]))[:, None]).to(s["dlogits"].dtype)


def _column(p, rows):
    """A setting as a column of 64-bit values, whether it is one number or a tensor."""
    if isinstance(p, torch.Tensor):
        return p.double()[:, None]
    return torch.full((rows, 1), float(p), dtype=torch.float64, device="cuda")


def _sample(s):
    # in 64 bits: the answer is an index, decided by sums that may lie next to u times the whole
    logits, par = s["logits"], s["par"]
    rows, v = logits.shape
    temp, k, p, minp = (_column(par[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    top, order = logits.float().sort(dim=1, descending=True, stable=True)
    x = (top.double() - top[:, :1].double()) / torch.where(temp > 0, temp, 1.0)
    w = x.exp()
    rank = torch.arange(v, device=logits.device)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(1) - w
    w = torch.where((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0), w, 0.0)
    w = torch.where((minp <= 0) | (x >= torch.where(minp > 0, minp, 1.0).clamp(max=1.0).log()), w, 0.0)
    w = torch.where((temp > 0) | (rank == 0), w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    run_sum = by_index.cumsum(1)
    u = s["u"].double()[:, None]
    return (run_sum <= u * run_sum[:, -1:]).sum(1).clamp_(max=v - 1)


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        from timeautodiff_amd import ops
        if op == "embed_fwd":
            ops.token_embed_fwd(s["tokens"], s["table"], s["out"], scale=s["scale"])
            return s["out"]
        if op == "embed_bwd":
            ops.token_embed_bwd(s["tokens"], s["dout"], s["dtable"], scale=s["scale"], accumulate=False)
            return s["dtable"]
        if op == "distill":
            ops.distill_loss(s["logits"], s["index"], s["value"], s["loss"], temperature=s["case"]["tau"], row_weight=s["weight"],
                             grad_scale=s["grad_scale"], dlogits=s["dlogits"])
            return s["loss"] if s["dlogits"] is None else (s["loss"], s["dlogits"])
        ops.sample_tokens(s["logits"], s["u"], s["out"], **s["par"])
        return s["out"]
    if op == "embed_fwd":
        return _embed_fwd(s)
    if op == "embed_bwd":
        return _embed_bwd(s)
    if op == "distill":
        return _distill(s)
    return _sample(s)


def work(case):
    op = case["op"]
    size = {F32: 4, B16: 2}
    if op == "embed_fwd":
        n, d = case["n"], case["dim"]
        # distinct rows of the table: about as many as there are tokens, or all of them
        return dict(bytes=n * 8 + min(n, case["vocab"]) * d * size[case["table"]] + n * d * size[case["out"]], flops=n * d)
    if op == "embed_bwd":
        n, d = case["n"], case["dim"]
        return dict(bytes=n * 8 + n * d * size[case["dout"]] + case["vocab"] * d * 4, flops=n * d)
    if op == "distill":
        rows, v, k = case["rows"], case["vocab"], case["k"]
        e = size[case["dtype"]]
        return dict(bytes=rows * v * e * (2 if case["grad"] else 1) + rows * (k * 12 + 8), flops=rows * v * (6 if case["grad"] else 3))
    rows, v = case["rows"], case["vocab"]
    return dict(bytes=rows * v * size[case["dtype"]] + rows * (4 + 8), flops=rows * v * 4)


# ---------------------------------------------------------------------------------------------- from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed_fwd":
        tab = torch.cat([s["table"].double(), s["table"].new_zeros(1, case["dim"]).double()])
        tok = s["tokens"].clone()
        tok[(tok < 0) | (tok >= case["vocab"])] = case["vocab"]
        return tab.index_select(0, tok) * s["scale"]
    if op == "embed_bwd":
        v, d = case["vocab"], case["dim"]
        tok = s["tokens"].clone()
        tok[(tok < 0) | (tok >= v)] = v
        return torch.zeros(v + 1, d, dtype=torch.float64, device="cuda").index_add_(0, tok, s["dout"].double())[:v] * s["scale"]
    if op == "distill":
        tau, v, rows = case["tau"], case["vocab"], case["rows"]
        loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
        grad = torch.empty(rows, v, dtype=torch.float64, device="cuda") if case["grad"] else None
        step = max(1, (1 << 26) // v)
        for lo in range(0, rows, step):
            z = s["logits"][lo:lo + step].double() / tau
            idx, val, w = s["index"][lo:lo + step], s["value"][lo:lo + step].double() / tau, s["weight"][lo:lo + step].double()
            ok = ((idx >= 0) & (idx < v)).double()
            q = torch.softmax(torch.where(ok > 0, val, -math.inf), 1)
            logp = torch.log_softmax(z, 1)
            at = idx.clamp(0, v - 1)
            kl = torch.xlogy(q, q) - q * logp.gather(1, at)
            loss[lo:lo + step] = w * tau ** 2 * (kl * ok).sum(1)
            if grad is not None:
                target = torch.zeros_like(z).scatter_add_(1, at, q * ok)
                grad[lo:lo + step] = (logp.exp() - target) * (w * tau * s["grad_scale"])[:, None]
        return loss if grad is None else (loss, grad)
    # the cut by thresholds on the sorted values, the answer by a search in the running sum
    rows, v, par = case["rows"], case["vocab"], s["par"]
    temp, k, p, minp = (_column(par[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    answer = torch.empty(rows, dtype=torch.int64, device="cuda")
    step = max(1, (1 << 24) // v)
    for lo in range(0, rows, step):
        z = s["logits"][lo:lo + step].double()
        at = slice(lo, min(rows, lo + step))
        t = torch.where(temp[at] > 0, temp[at], 1.0)
        place = (-z).argsort(dim=1, stable=True)
        lead = z.gather(1, place)
        e = torch.exp((lead - lead[:, :1]) / t)
        kept = torch.where(k[at] <= 0, v, k[at]).clamp(max=v).long()
        mass = e.cumsum(1)
        whole = mass.gather(1, kept - 1)
        by_p = (mass < p[at] * whole).sum(1, keepdim=True) + 1
        kept = torch.where(p[at] >= 1, kept, torch.minimum(kept, by_p))
        by_m = ((lead - lead[:, :1]) / t >= torch.log(minp[at].clamp(1e-300, 1.0))).sum(1, keepdim=True)
        kept = torch.minimum(kept, by_m)
        kept = torch.where(temp[at] > 0, kept, 1)
        where = place.argsort(dim=1)          # each index's place in the order
        c = torch.where(where < kept, torch.exp((z - lead[:, :1]) / t), 0.0).cumsum(1)
        answer[at] = torch.searchsorted(c, s["u"][at].double()[:, None] * c[:, -1:], right=True)[:, 0].clamp(max=v - 1)
    return answer
