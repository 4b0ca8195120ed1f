"""float64 restatement of the token family: embedding lookup and gradient, distillation loss and gradient, token draw.
Written from the definitions; no counterpart in the reference."""
import numpy as np


def embed_fwd(tokens, table, scale):
    tok = np.asarray(tokens).reshape(-1)
    out = np.zeros((tok.size, table.shape[1]))
    fine = (tok >= 0) & (tok < table.shape[0])
    out[fine] = table.astype(np.float64)[tok[fine]] * scale
    return out


def embed_bwd(tokens, dout, vocab, scale):
    """(gradient, sum of |terms|, number of terms) per row of the table."""
    tok = np.asarray(tokens).reshape(-1)
    fine = (tok >= 0) & (tok < vocab)
    d = dout.astype(np.float64)[fine]
    grad = np.zeros((vocab, dout.shape[1]))
    size = np.zeros((vocab, dout.shape[1]))
    np.add.at(grad, tok[fine], d)
    np.add.at(size, tok[fine], np.abs(d))
    return grad * scale, size * abs(scale), np.bincount(tok[fine], minlength=vocab)


def _softmax(x):
    m = x.max()
    e = np.exp(x - m)
    return e / e.sum()


def distill(logits, index, value, tau, weight, grad_scale):
    """(loss [rows], gradient [rows, V]); rows that count nothing are zero."""
    x = logits.astype(np.float64)
    rows, V = x.shape
    loss, grad = np.zeros(rows), np.zeros((rows, V))
    for r in range(rows):
        w = 1.0 if weight is None else float(weight[r])
        ok = (index[r] >= 0) & (index[r] < V) & (value[r] > -np.inf)
        if w == 0.0 or not ok.any() or not (x[r] > -np.inf).any():
            continue
        q = _softmax(value[r][ok].astype(np.float64) / tau)
        z = x[r] / tau
        m = z.max()
        logp = z - m - np.log(np.exp(z - m).sum())
        on = q > 0
        loss[r] = w * tau ** 2 * np.sum(q[on] * (np.log(q[on]) - logp[index[r][ok][on]]))
        target = np.zeros(V)
        np.add.at(target, index[r][ok], q)
        grad[r] = grad_scale * w * tau * (np.exp(logp) - target)
    return loss, grad


def kept(row, T, top_k, top_p, min_p):
    """(weights of the kept tokens by index, the smallest relative distance of a decision from its border)."""
    x = row.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    V = x.size
    if m == -np.inf:
        return None, np.inf
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        w = np.zeros(V)
        w[order[0]] = 1.0
        return w, np.inf
    with np.errstate(invalid="ignore"):
        t = np.where(x == m, 0.0, (x - m) / T)
    t = np.where(x == -np.inf, -np.inf, np.where(np.isnan(t), -np.inf, t))
    w = np.exp(t)
    near = np.inf
    w_s, t_s = w[order], t[order]
    if 0 < top_k < V:
        w_s[top_k:] = 0.0
    if top_p < 1:
        before = np.cumsum(w_s) - w_s
        line = top_p * w_s.sum()
        live = w_s > 0
        out = live & ~(before < line)
        out[0] = False
        near = min(near, np.abs(before[live][1:] - line).min() / w_s.sum()) if live.sum() > 1 else near
        w_s = np.where(out, 0.0, w_s)
    if min_p > 0:
        line = np.log(min(min_p, 1.0))
        away = np.abs(t_s[t_s < 0] - line)
        near = min(near, away.min()) if away.size and min_p < 1 else near
        w_s = np.where(t_s >= line, w_s, 0.0)
    back = np.zeros(V)
    back[order] = w_s
    return back, near


def sample(row, u, T, top_k, top_p, min_p):
    """(token, distance of the closest decision from its border, relative)."""
    w, near = kept(row, T, top_k, top_p, min_p)
    if w is None:
        return -1, np.inf
    cum = np.cumsum(w)
    u = 0.0 if not u > 0 else float(u)
    if u >= 1:
        return int(np.nonzero(w)[0][-1]), near
    at = np.unique(cum[cum < cum[-1]])
    if at.size and u > 0:
        near = min(near, np.abs(at - u * cum[-1]).min() / cum[-1])
    return int(np.searchsorted(cum, u * cum[-1], side="right")), near
