"""The vocabulary operators from their definitions, in 64 bits on the CPU, and
the error bounds that the 32-bit kernels are held to."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
             torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
# Half the distance between the smallest numbers of the type.
SMALLEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25,
            torch.bfloat16: 2.0 ** -134, torch.float64: 0.0}


def lookup(table, tokens, scale):
    t = table.double().cpu()
    ids = tokens.long().cpu()
    ok = (ids >= 0) & (ids < t.shape[0])
    out = torch.zeros(tuple(ids.shape) + (t.shape[1],), dtype=torch.float64)
    out[ok] = t[ids[ok]] * scale
    return out


def lookup_bound(want, dtype):
    """One product in 32 bits and one rounding to the type."""
    h = HALF_STEP[dtype]
    return want.abs() * (h + 2.0 ** -23) + SMALLEST[dtype]


def gradient(grad, tokens, rows, scale, start=None):
    """Returns the gradient and the sum of the terms' sizes for the bound."""
    g = grad.double().cpu().reshape(-1, grad.shape[-1])
    ids = tokens.long().cpu().reshape(-1)
    ok = (ids >= 0) & (ids < rows)
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    times = torch.zeros(rows, dtype=torch.float64)
    out.index_add_(0, ids[ok], g[ok] * scale)
    size.index_add_(0, ids[ok], g[ok].abs() * abs(scale))
    times.index_add_(0, ids[ok], torch.ones(int(ok.sum()),
                                            dtype=torch.float64))
    if start is not None:
        out += start.double().cpu()
    return out, size, times


def gradient_bound(want, size, times, dtype, start=None):
    """m terms cost at most m additions of 32 bits (each within 2^-24 of a
    partial sum, which is at most the sum of the sizes), the scaling one
    rounding, adding to what was there one more, and the output one."""
    b = size * (times[:, None] + 1) * 2.0 ** -24 * 1.001
    if start is not None:
        b = b + (want.abs() + size) * 2.0 ** -24
    return b + want.abs() * HALF_STEP[dtype] * 1.001 + SMALLEST[dtype]


def distill(logits, tokens, teacher, weights, temperature):
    """Loss, gradient and their bounds, row by row."""
    x = logits.double().cpu().numpy()
    ids = tokens.long().cpu().numpy()
    t = teacher.double().cpu().numpy()
    n, vocab = x.shape
    w = np.ones(n) if weights is None else weights.double().cpu().numpy()
    T = float(temperature)
    loss, grad = np.zeros(n), np.zeros((n, vocab))
    loss_bound, grad_bound = np.zeros(n), np.zeros((n, vocab))
    u = 2.0 ** -24
    for i in range(n):
        used = (ids[i] >= 0) & (ids[i] < vocab)
        if w[i] == 0 or not used.any():
            continue
        j, tk = ids[i][used], t[i][used] / T
        if tk.max() == -np.inf or x[i].max() == -np.inf:
            continue
        with np.errstate(divide="ignore", invalid="ignore"):
            s = x[i] / T
            zs = s.max() - s                      # distances, in nats
            e = np.exp(-zs)
            log_q = -zs - np.log(e.sum())
            q = np.exp(log_q)
            zt = tk.max() - tk
            et = np.exp(-zt)
            log_p = -zt - np.log(et.sum())
            p = np.exp(log_p)
            term = np.where(p > 0, p * (log_p - log_q[j]), 0.0)
        loss[i] = T * T * term.sum()
        grad[i] = q
        np.subtract.at(grad[i], j, p)
        grad[i] *= w[i] * T
        # A weight 2^((x - m) c): the difference, c = log2(e) / T (a division
        # of a rounded constant) and their product are rounded (4 u of an
        # exponent of z log2(e), so 4 u z of the weight), the instruction is
        # within 2 units = 4 u, and weights pass from one maximum to another
        # (the same again, once in a thread's run and 10 times in the trees,
        # of distances that add up to z). A sum adds its longest chain:
        # vocab additions of a thread at the very most / 32 lanes of the
        # smallest block, and 16 steps of the trees.
        dead = ~np.isfinite(zs)
        zs_ = np.where(dead, 0.0, zs)
        each = (8 * zs_ + 44) * u
        mass = (q * each).sum() + (vocab / 32 + 16) * u
        zt_ = np.where(np.isfinite(zt), zt, 0.0)
        mass_t = (p * (8 * zt_ + 44) * u).sum() + (len(j) / 32 + 16) * u
        # log p and log q: difference, division, logarithm (1 unit) and
        # subtraction.
        at_q = 4 * u * (zs_[j] + abs(np.log(e.sum())) + 1) + mass
        at_p = 4 * u * (zt_ + abs(np.log(et.sum())) + 1) + mass_t
        rel_p = at_p + 4 * u                      # p = exp(log p)
        inside = np.where(p > 0, np.abs(np.where(np.isfinite(term), term, 0))
                          * (rel_p + (len(j) / 32 + 20) * u)
                          + p * (at_p + at_q + u * (zt_ + zs_[j] + 40)), 0)
        loss_bound[i] = 1.01 * (T * T * inside.sum() + 4 * u * abs(loss[i])
                                if np.isfinite(loss[i]) else 0)
        gb = q * (each + mass + 8 * u)
        np.add.at(gb, j, p * (rel_p + (len(j) + 6) * u))
        h = HALF_STEP[logits.dtype]
        grad_bound[i] = 1.01 * abs(w[i]) * T * gb
        grad_bound[i] += (np.abs(grad[i]) + grad_bound[i]) * h
        # Weights below 2^-126 are zero.
        grad_bound[i] += SMALLEST[logits.dtype] + abs(w[i]) * T * 2.0 ** -125
    return loss, grad, loss_bound, grad_bound


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x: the row in 64 bits; the settings as the 32-bit numbers they are."""
    x = np.asarray(x, dtype=np.float64)
    if x.size == 0 or np.isnan(x).any() or x.max() == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    peak = x.max()

    def weight(values):
        with np.errstate(invalid="ignore"):
            return np.where(values == peak, 1.0,
                            np.exp((values - peak) / temperature))

    order = np.argsort(-x, kind="stable")
    if 0 < top_k < x.size:
        order = order[:top_k]
    w = weight(x[order])
    if top_p < 1:
        sums = np.cumsum(w)
        order = order[:int(np.sum(sums - w < top_p * sums[-1])) or 1]
        w = weight(x[order])
    order = np.sort(order[(w >= min_p) | (w == 1.0)])
    w = weight(x[order])
    sums = np.cumsum(w)
    hit = np.nonzero((w > 0) & (sums > u * sums[-1]))[0]
    return int(order[hit[0]]) if hit.size else int(order[w > 0][-1])


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x = logits.double().cpu().numpy()
    n = x.shape[0]

    def rows(value):
        if isinstance(value, torch.Tensor):
            return value.cpu().numpy()
        return np.full(n, value, np.int32 if isinstance(value, int)
                       else np.float32)

    t, k, p, m = rows(temperature), rows(top_k), rows(top_p), rows(min_p)
    u = uniform.cpu().numpy()
    return torch.tensor([sample_row(x[i], float(u[i]), float(t[i]), int(k[i]),
                                    float(p[i]), float(m[i]))
                         for i in range(n)], dtype=torch.int32)
