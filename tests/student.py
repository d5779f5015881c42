"""Plain float64 forms of the ops a student model needs (top logits, distillation, verification of drafts), and inputs for them."""
import numpy as np

NO_TOKEN = np.uint64((1 << 64) - 1)


def bf16_bits(x):
    """Round to nearest even, as raw bit patterns."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), r)


def bf16_values(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def stored(x, dtype):
    """What the device is given for x, and the float32 values that it then holds."""
    if dtype == "bf16":
        b = bf16_bits(x)
        return b, bf16_values(b)
    x = np.ascontiguousarray(x, np.float32)
    return x, x


def top_logits(x, k, T=1.0):
    """x [rows, C] -> values, indices [rows, k], lse [rows]"""
    x = np.asarray(x, np.float64)
    order = np.empty(x.shape[:1] + (k,), np.int64)
    for r, row in enumerate(x):  # NaN first, then descending, equal ones by index
        order[r] = np.lexsort((np.arange(len(row)), np.where(np.isnan(row), 0.0, -row), ~np.isnan(row)))[:k]
    return np.take_along_axis(x, order, 1), order.astype(np.uint64), lse(x / T)


def lse(z):
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        m0 = np.where(np.isfinite(m), m, 0.0)
        return (m0 + np.log(np.exp(z - m0).sum(1, keepdims=True)))[:, 0]


def distill(x, index, u, t_lse=None, weight=None, T=1.0, loss_div=1.0):
    """x [rows, C], index / u [rows, k] -> row losses [rows], gradient [rows, C], and what their bounds take: probabilities, masses, logarithms"""
    x, u = np.asarray(x, np.float64), np.asarray(u, np.float64)
    rows, C = x.shape
    out, grad = np.zeros(rows), np.zeros((rows, C))
    parts = {"p": np.zeros((rows, C)), "q": np.zeros((rows, C)), "mass": np.zeros(rows), "rest": np.zeros(rows), "p_rest": np.ones(rows), "far": np.zeros(rows),
             "log_quotient": np.zeros(rows), "share": np.zeros((rows, C))}
    for r in range(rows):
        w = 1.0 if weight is None else float(weight[r])
        if w == 0.0:
            continue
        ok = index[r] < C
        at, v = index[r][ok].astype(np.int64), u[r][ok] / T
        if t_lse is None:
            level = lse(v[None])[0] if len(v) and v.max() > -np.inf else 0.0
        else:
            level = float(t_lse[r])
        logq = v - level
        q = np.exp(logq)
        z = (x[r] - (x[r].max() if np.isfinite(x[r].max()) else 0.0)) / T  # near the type's limits a normaliser has no digits for its logarithm
        total = lse(z[None])[0]
        logp = z - total
        p = np.exp(logp)
        some = q > 0
        row = float((q[some] * (logq[some] - logp[at[some]])).sum())
        mass = q.sum()
        outside = np.ones(C, bool)
        outside[at] = False
        some_outside = outside.any() and z[outside].max() > -np.inf  # else there is no p_r, and r counts as 0
        rest = max(0.0, 1.0 - mass) if t_lse is not None and some_outside else 0.0
        g = (mass + rest) * p
        np.subtract.at(g, at, q)
        p_rest = 1.0
        if t_lse is not None and some_outside:
            far = z[outside].max()
            spread = lse(z[outside][None] - far)[0]      # shifted as above
            log_rest = far - total + spread
            p_rest = np.exp(log_rest)
            parts["share"][r, outside] = np.exp(z[outside] - far - spread)
            if rest > 0:
                row += rest * (np.log(rest) - log_rest)
                parts["log_quotient"][r] = abs(np.log(rest) - log_rest)
                g -= rest * parts["share"][r]
        out[r], grad[r] = row * w, g * w / (T * loss_div)
        parts["p"][r], parts["mass"][r], parts["rest"][r], parts["p_rest"][r] = p, mass, rest, p_rest
        np.add.at(parts["q"][r], at, q)
        parts["far"][r] = np.abs(logq[some]).max() if some.any() else 0.0
    return out, grad, parts


def verify(target, draft, tokens, lengths, uniforms):
    """target [B, n + 1, C], draft [B, n, C] or None, tokens [B, n], uniforms [B, n + 1] -> out [B, n + 1], accepted [B]"""
    target = np.asarray(target, np.float64)
    B, n1, C = target.shape
    n = n1 - 1
    out, accepted = np.full((B, n1), NO_TOKEN, np.uint64), np.zeros(B, np.uint64)
    for b in range(B):
        length = n if lengths is None else min(n, int(lengths[b]))
        a = 0
        while a < length:
            d = int(tokens[b, a])
            q = 1.0 if draft is None else (float(draft[b, a, d]) if d < C else 1.0)
            if not (d < C and float(uniforms[b, a]) * q < float(target[b, a, d])):
                break
            out[b, a] = d
            a += 1
        w = np.fmax(target[b, a], 0.0)
        if a < length:
            v = w.copy()
            if draft is not None:
                v = np.fmax(target[b, a] - np.asarray(draft[b, a], np.float64), 0.0)
            elif int(tokens[b, a]) < C:
                v[int(tokens[b, a])] = 0.0
            if v.sum() > 0:
                w = v
        accepted[b] = a
        if w.sum() > 0:
            run = np.cumsum(w)
            j = int(np.searchsorted(run, float(uniforms[b, n]) * run[-1], side="right"))
            out[b, a] = min(j, int(np.nonzero(w)[0][-1]))
    return out, accepted
