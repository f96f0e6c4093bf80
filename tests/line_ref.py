"""What the calls on packed lines' logits compute, restated line by line in numpy: the ruled logits in
float32 with every operation rounded on its own (the definition), probabilities in 64 bits; the
head with adapters in 64 bits."""
from __future__ import annotations

import numpy as np

F = np.float32


def ruled(z, line_at, rules):
    """z [rows, classes] (float16 or float32) -> float32 under the lines' rules; rules: a dict of the
    arrays of crec_rules (absent: no rule)."""
    z = z.astype(np.float32).copy()
    classes = z.shape[1]
    with np.errstate(all="ignore"):
        for i in range(len(line_at) - 1):
            rows = z[line_at[i]:line_at[i + 1]]
            if len(rows) == 0:
                continue
            if "history" in rules:
                h = rules["history"][rules["history_at"][i]:rules["history_at"][i + 1]]
                seen, n = np.unique(h[(h >= 0) & (h < classes)], return_counts=True)
                rep = F(rules["repeat"][i]) if "repeat" in rules else F(1)
                pres = F(rules["presence"][i]) if "presence" in rules else F(0)
                freq = F(rules["frequency"][i]) if "frequency" in rules else F(0)
                v = rows[:, seen]
                rows[:, seen] = np.where(v > 0, v / rep, v * rep) - (n.astype(F) * freq + pres)
            if "bias" in rules:
                b = rules["bias_of"][i] if "bias_of" in rules else 0
                if 0 <= b < len(rules["bias"]):
                    t = rules["bias"][b]
                    rows[:] = np.where(np.isneginf(t), -np.inf, rows + t)
            if "allowed" in rules:
                s = rules["set_of"][i] if "set_of" in rules else 0
                if 0 <= s < len(rules["allowed"]):
                    c = np.arange(classes)
                    rows[:, (rules["allowed"][s][c // 32] >> (c % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return z


def softmax_parts(row):
    """(best, its lowest class, ln of the sum of exp(z - best)) in 64 bits; best -inf where nothing is left."""
    r = row.astype(np.float64)
    best = np.nanmax(r) if not np.isnan(r).all() else -np.inf
    if best == -np.inf:
        return best, 0, 0.0
    return best, int(np.flatnonzero(r == best)[0]), float(np.log(np.exp(r - best).sum()))


def greedy(z, line_at):
    """Ruled logits -> per line (ids, starts, probs float64)."""
    out = []
    for i in range(len(line_at) - 1):
        ids, starts, probs, prev = [], [], [], 0
        for t in range(line_at[i], line_at[i + 1]):
            best, c, ln = softmax_parts(z[t])
            p = np.exp(-ln) if best > -np.inf else 0.0
            if c != 0 and c != prev:
                ids.append(c)
                starts.append(t - line_at[i])
                probs.append(p)
            elif c != 0:
                probs[-1] = max(probs[-1], p)
            prev = c
        out.append((ids, starts, probs))
    return out


def candidates(z, k):
    """Ruled logits [rows, classes] -> (ids [rows, k], logp float64, blank float64)."""
    n = len(z)
    ids, logp, blank = np.full((n, k), -1, np.int32), np.full((n, k), -np.inf), np.full(n, -np.inf)
    for t in range(n):
        best, _, ln = softmax_parts(z[t])
        r = z[t].astype(np.float64)
        base = best if best > -np.inf else 0.0
        blank[t] = r[0] - base - ln
        order = [c for c in np.argsort(-r[1:], kind="stable")[:k] + 1 if r[c] > -np.inf]
        ids[t, :len(order)] = order
        logp[t, :len(order)] = r[order] - base - ln
    return ids, logp, blank


def sum_tolerance(classes):
    """How far a float32 sum of exp(z - best) over the classes may be off, relative to it, in units of the
    rounding 2^-24: a chain of at most 32 adds a lane and 1,024 classes of each of 16 warps, then 10 of
    the joins; exp itself, 2^-22 (4), and its argument, |z - best| roundings twice (a sum of C terms
    weighs |z - best| by at most ln C on average); a final reciprocal."""
    chain = 32 * -(-classes // 16384) + 10
    return (chain + 4 + 2 * np.log(classes + 1) + 2) * 2.0 ** -24


def adapters(x, w, b, sets, line_at, adapter):
    """x [rows, K] float16, w [classes, K] float16, b float32, sets [(A, B, scale)]: the lines' logits in 64 bits,
    and for each the sum of the products' magnitudes (what roundings are relative to)."""
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    z = x64 @ w64.T + b.astype(np.float64)
    mag = np.abs(x64) @ np.abs(w64).T + np.abs(b.astype(np.float64))
    for i in range(len(line_at) - 1):
        a = adapter[i] if adapter is not None else -1
        if 0 <= a < len(sets):
            A, B, s = sets[a]
            A, B, s = A.astype(np.float64), B.astype(np.float64), float(np.float32(s))
            lo, hi = line_at[i], line_at[i + 1]
            z[lo:hi] += s * (x64[lo:hi] @ A.T) @ B.T
            mag[lo:hi] += abs(s) * (np.abs(x64[lo:hi]) @ np.abs(A).T) @ np.abs(B).T
    return z, mag
