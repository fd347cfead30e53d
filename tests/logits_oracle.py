"""Plain 64-bit statements of the operators on logits and beams (numpy), and the
error bounds the GPU tests hold the kernels to.

Bounds count roundings. One fp32 rounding is U = 2^-24 of the value, one bf16
rounding 2^-8. A sum over V terms in fp32 that is split over at least 32
threads and joined as a tree rounds each term at most V / 32 + 16 times; the
exponential and the logarithm are within 4 U of their value, and an argument
a = (x - m) / tau is itself rounded three times, which moves exp(a) by 3 |a| U
of its value.
"""
import numpy as np

U = 2.0 ** -24
BF16 = 2.0 ** -8
FMAX = np.finfo(np.float32).max


def canon(x):
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    return np.minimum(x, float(FMAX)) + 0.0


def logsumexp(x, axis=-1):
    m = np.max(x, axis=axis, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore"):
        return np.squeeze(m, axis) + np.log(np.exp(x - m).sum(axis=axis))


def logsoftmax(x):
    d = x - x.max()
    return d - np.log(np.exp(d).sum())


def lse_bound(lse, vocab):
    return (3 * np.abs(np.where(np.isfinite(lse), lse, 0)) + vocab / 32 + 40) * U


def topk(z, k, tau):
    z = canon(z)
    idx = np.argsort(-z, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(z, idx, 1)
    idx = np.where(top > -np.inf, idx, -1)
    return top, idx, logsumexp(z / tau)


def distill(z, t_idx, t_val, tau, soft, hard, scale, t_lse=None, targets=None, weight=None):
    """(row_loss, dlogits, bound of row_loss, bound of dlogits without the
    rounding to the logits' type), row by row from the definition."""
    n, v = z.shape
    z = np.asarray(z, np.float64)
    loss, grad = np.zeros(n), np.zeros((n, v))
    bl, bg = np.zeros(n), np.zeros((n, v))
    c = v / 32 + 40
    for r in range(n):
        w = 1.0 if weight is None else float(weight[r])
        if w == 0.0 or np.all(z[r] == -np.inf):
            continue
        use = (t_idx[r] >= 0) & (t_idx[r] < v)
        ids, t = t_idx[r][use], t_val[r][use].astype(np.float64) / tau
        if t_lse is not None:
            logp = t - float(t_lse[r])
        else:
            logp = logsoftmax(t) if np.any(t > -np.inf) else np.full(t.shape, -np.inf)
        p = np.exp(logp)
        # relative to the largest logit first: z / tau - lse would lose every
        # digit of lse - max where the logits are as large as -3e38
        lq = logsoftmax(z[r] / tau)
        q = np.exp(lq)
        a = np.where(np.isfinite(z[r]), (z[r].max() - z[r]) / tau, 0.0)
        with np.errstate(invalid="ignore"):
            kl = np.where(p > 0, p * (logp - lq[ids]), 0.0).sum()
        sp = np.zeros(v)
        np.add.at(sp, ids, p)
        big = np.abs(t[np.isfinite(t)]).max(initial=0.0) + (abs(float(t_lse[r])) if t_lse is not None else 0.0)
        g = soft * tau * (p.sum() * q - sp)
        fin = np.where(np.isfinite(lq[ids]), np.abs(lq[ids]), 0.0)
        fip = np.where(np.isfinite(logp), np.abs(logp), 0.0)
        bl[r] = abs(soft) * tau * tau * ((p * ((fin + fip) * (c + 8 * big) + c + 8 * big)).sum()
                                         + 1) * U
        bg[r] = abs(soft) * tau * (p.sum() * q * (c + 8 * big + 4 * a) + sp * (c + 8 * big)) * U
        l = soft * tau * tau * kl
        if hard and targets[r] >= 0 and targets[r] < v:
            l1 = logsoftmax(z[r])
            l += -hard * l1[targets[r]]
            q1 = np.exp(l1)
            hot = np.arange(v) == targets[r]
            g += hard * (q1 - hot)
            bl[r] += abs(hard) * (abs(l1[targets[r]]) * 4 + c) * U
            bg[r] += abs(hard) * (q1 * (c + 4 * a * tau) + hot) * U
        loss[r], grad[r] = w * l, scale * w * g
        bl[r] = abs(w) * (bl[r] + abs(l) * 4 * U)
        bg[r] = abs(scale * w) * (bg[r] + np.abs(g) * 4 * U)
    # beyond the largest fp32 number a loss rounds to infinity
    over = np.abs(loss) > float(FMAX)
    loss[over] = np.sign(loss[over]) * np.inf
    return loss, grad, bl, bg


def select(z, scores, beams, eos=-1, finished=None):
    """(scores, tokens, parents, finished, smallest gap between two candidates
    that differ, among the chosen ones and the first one left out)."""
    z = canon(z)
    m, v = z.shape
    b = m // beams
    s = canon(scores)
    with np.errstate(invalid="ignore"):
        t = (s[:, None] + z) - logsumexp(z)[:, None]
    t = np.where((z == -np.inf) | (s[:, None] == -np.inf), -np.inf, t)
    done = np.zeros(m, bool) if finished is None else np.asarray(finished) != 0
    t[done] = -np.inf
    t[done, eos] = s[done]
    out_s, tok, par, fin = (np.zeros(m), np.zeros(m, np.int64), np.zeros(m, np.int64),
                            np.zeros(m, np.int64))
    gap = np.inf
    for g in range(b):
        flat = t[g * beams:(g + 1) * beams].reshape(-1)
        o = np.argsort(-flat, kind="stable")[:beams + 1]
        near = flat[o][np.isfinite(flat[o])]
        d = -np.diff(near)
        if np.any(d > 0):
            gap = min(gap, d[d > 0].min())
        for j in range(beams):
            live = j < len(o) and flat[o[j]] > -np.inf
            i = g * beams + j
            out_s[i] = flat[o[j]] if live else -np.inf
            par[i] = o[j] // v if live else j
            tok[i] = o[j] % v if live else max(eos, 0)
            fin[i] = done[g * beams + par[i]] or tok[i] == eos
    return out_s, tok, par, fin, gap


def backtrack(tokens, parents, scores, beams, eos, alpha):
    t, m = tokens.shape
    seq, length = np.zeros((m, t), np.int64), np.zeros(m, np.int64)
    rank = np.zeros(m)
    for g in range(m // beams):
        rows = []
        for j in range(beams):
            a, path = j, []
            for i in range(t - 1, -1, -1):
                path.append(tokens[i, g * beams + a])
                p = parents[i, g * beams + a]
                a = p if 0 <= p < beams else a
            path = path[::-1]
            n = path.index(eos) + 1 if eos >= 0 and eos in path else t
            path[n:] = [eos] * (t - n)
            rows.append((canon(scores[g * beams + j]) / float(n) ** float(np.float32(alpha)),
                         path, n))
        order = sorted(range(beams), key=lambda j: (-rows[j][0], j))
        for r, j in enumerate(order):
            rank[g * beams + r], seq[g * beams + r], length[g * beams + r] = rows[j]
    return seq, length, rank
