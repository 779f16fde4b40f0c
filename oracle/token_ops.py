"""The losses over rows of logits (style_transfer_amd.token_losses) in 64 bits, a row at a time on the CPU: test
infrastructure, written from the formulas.  No counterpart in the reference: parity unpinned."""
from __future__ import annotations

import math

import torch


def row(x, tau):
    """(log q, q, entropy) of one row of logits; (all -inf, 0, 0) for a row of -inf only."""
    z = x.double() / tau
    m = z.max()
    if m == -math.inf:
        return z, torch.zeros_like(z), 0.0
    log_q = z - m - (z - m).exp().sum().log()
    q = log_q.exp()
    return log_q, q, float(-(q * log_q.clamp(min=-1e300)).sum())


def token_logprobs(x, labels, tau=1.0, ignore=-100):
    """logp [N], entropy [N], log q [N, V], q [N, V] of x [N, V]; ignored rows are 0."""
    n, vocab = x.shape
    logp, h = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    log_q, q = torch.zeros(n, vocab, dtype=torch.float64), torch.zeros(n, vocab, dtype=torch.float64)
    for r in range(n):
        t = int(labels[r])
        if t == ignore:
            continue
        log_q[r], q[r], h[r] = row(x[r], tau)
        logp[r] = log_q[r, t] if 0 <= t < vocab else math.nan
    return logp, h, log_q, q


def row_gradient(labels, tau, h, log_q, q, a, b, ignore=-100):
    """d / dx of sum a[r] logp[r] + b[r] entropy[r]."""
    g = torch.zeros_like(q)
    for r in range(q.shape[0]):
        t = int(labels[r])
        if t == ignore or not bool(q[r].any()):
            continue
        g[r] = -a[r] * q[r] - b[r] * q[r] * (log_q[r].clamp(min=-1e300) + h[r])
        g[r, t] += a[r]
    return g / tau


def sequences_of(labels, cu=None):
    """[(start, end)] in rows of the flattened labels."""
    if cu is None:
        count, length = labels.shape
        return [(s * length, (s + 1) * length) for s in range(count)]
    return [(int(cu[s]), int(cu[s + 1])) for s in range(len(cu) - 1)]


def preference(x, labels, seqs, ref=None, beta=0.1, kind="sigmoid", smoothing=0.0, average=False, ignore=-100):
    """loss, rewards [2 P], gradient [N, V]."""
    logp, h, log_q, q = token_logprobs(x, labels, 1.0, ignore)
    pairs = len(seqs) // 2
    counts = [[r for r in range(s, e) if int(labels[r]) != ignore] for s, e in seqs]
    per = [1.0 / max(1, len(c)) if average else 1.0 for c in counts]
    ratio = [float(logp[c].sum()) * w - (float(ref[i]) if ref is not None else 0.0) for i, (c, w) in enumerate(zip(counts, per))]
    a = torch.zeros_like(logp)
    loss = 0.0
    for i in range(pairs):
        gap = ratio[i] - ratio[i + pairs]
        z = beta * gap
        if kind == "sigmoid":
            soft = lambda v: max(v, 0.0) + math.log1p(math.exp(-abs(v)))  # noqa: E731
            sig = lambda v: 1 / (1 + math.exp(-v)) if v > -700 else 0.0  # noqa: E731
            loss += (1 - smoothing) * soft(-z) + (smoothing * soft(z) if smoothing else 0.0)      # z may be +inf
            slope = beta * (smoothing * sig(z) - (1 - smoothing) * sig(-z))
        elif kind == "ipo":
            loss += (gap - 0.5 / beta) ** 2
            slope = 2 * (gap - 0.5 / beta)
        else:
            loss += max(0.0, 1 - z)
            slope = -beta if z < 1 else 0.0
        for c, w, sign in ((counts[i], per[i], 1), (counts[i + pairs], per[i + pairs], -1)):
            for r in c:
                a[r] += sign * slope * w / pairs
    return loss / pairs, torch.tensor(ratio, dtype=torch.float64) * beta, row_gradient(labels, 1.0, h, log_q, q, a, torch.zeros_like(a), ignore)


def policy(x, labels, seqs, old, adv, ref=None, low=0.2, high=0.2, kl=0.0, ent=0.0, tau=1.0, per_sequence=False, ignore=-100):
    """loss, [surrogate, KL, entropy, clipped share], gradient [N, V]; adv: one value a row."""
    logp, h, log_q, q = token_logprobs(x, labels, tau, ignore)
    counts = [[r for r in range(s, e) if int(labels[r]) != ignore] for s, e in seqs]
    w = torch.zeros_like(logp)
    if per_sequence:
        held = sum(len(c) > 0 for c in counts)
        for c in counts:
            w[c] = 1.0 / held / max(1, len(c))
    else:
        total = sum(len(c) for c in counts)
        for c in counts:
            w[c] = 1.0 / max(1, total)
    a, b = torch.zeros_like(logp), torch.zeros_like(logp)
    stats = [0.0] * 4
    for c in counts:
        for r in c:
            ratio, adv_r, weight = math.exp(float(logp[r]) - float(old[r])), float(adv[r]), float(w[r])
            held = min(max(ratio, 1 - low), 1 + high)
            stats[0] += weight * -min(ratio * adv_r, held * adv_r)
            clipped = held * adv_r < ratio * adv_r
            stats[3] += weight * clipped
            stats[2] += weight * float(h[r])
            slope = 0.0 if clipped else -adv_r * ratio
            if ref is not None:
                d = float(ref[r]) - float(logp[r])
                stats[1] += weight * (math.expm1(d) - d)
                slope += kl * -math.expm1(d)
            a[r], b[r] = weight * slope, -weight * ent
    loss = stats[0] + kl * stats[1] - ent * stats[2]
    return loss, torch.tensor(stats, dtype=torch.float64), row_gradient(labels, tau, h, log_q, q, a, b, ignore)


def distill(x, idx, val, mask=None, tau=1.0, tail=False):
    """loss, gradient [N, V]."""
    n, vocab = x.shape
    keep = [True] * n if mask is None else [bool(v) for v in mask]
    total, grad = 0.0, torch.zeros(n, vocab, dtype=torch.float64)
    w = 1.0 / max(1, sum(keep))
    for r in range(n):
        if not keep[r]:
            continue
        log_q, q, _ = row(x[r], tau)
        used = [(int(j), float(v)) for j, v in zip(idx[r], val[r]) if int(j) >= 0]
        if any(j >= vocab for j, _ in used):
            total, grad[r] = math.nan, math.nan
            continue
        if not used:
            continue
        if tail:
            log_p = [v for _, v in used]
        else:
            top = max([v for _, v in used], default=-math.inf)
            z = math.log(sum(math.exp((v - top) / tau) for _, v in used)) if top > -math.inf else 0.0
            log_p = [(v - top) / tau - z if top > -math.inf else -math.inf for _, v in used]
        p = [math.exp(v) for v in log_p]
        each = sum(pk * (lk - float(log_q[j])) for pk, lk, (j, _) in zip(p, log_p, used) if pk > 0)
        listed = {j for j, _ in used}
        off = [j for j in range(vocab) if j not in listed]
        mass = sum(p)
        rest = max(0.0, 1 - mass) if tail and off else 0.0
        g = q * (mass + rest)
        for pk, (j, _) in zip(p, used):
            g[j] -= pk
        if rest > 0:
            zoff = log_q[off]
            top = float(zoff.max())
            log_rest = top + math.log(float((zoff - top).exp().sum())) if top > -math.inf else -math.inf
            each += rest * (math.log(rest) - log_rest)
            if top > -math.inf:
                g[off] -= rest * (zoff - log_rest).exp()
        total += tau ** 2 * w * each
        if bool(q.any()):
            grad[r] = tau * w * g
    return total, grad
