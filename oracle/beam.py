"""Oracle: beam search's selection and the forking of paged sequences, in numpy
float64 and plain Python.

Test infrastructure only (see ``oracle/__init__.py``).

* ``select``: s = score + (x - logsumexp(x)) of every (beam, token), ranked by
  s / max(length, 1) ** penalty, ties to the lower beam, then the lower token; a
  finished beam has one continuation (pad token, its own score and length). NaN
  logits count as -inf, +inf as fp32's largest number.
* ``fork``: sequence after sequence, as the rule is worded: share the parent's
  pages up to its length, then in ascending order copy a page that others hold
  before writing to it and take the lowest free pages for the new rows.
"""
from __future__ import annotations

import numpy as np

PAGE = 64
BIG = float(np.finfo(np.float32).max)


def clean(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, np.float64)
    return np.minimum(np.where(np.isnan(x), -np.inf, x), BIG)


def continuations(logits, scores, lengths, finished, vocab: int, pad: int, penalty: float):
    """One group: logits [K, V] -> (sum, rank) of every continuation [K, V], -inf where there is none."""
    x = clean(logits)
    K = x.shape[0]
    total = np.full((K, vocab), -np.inf)
    rank = np.full((K, vocab), -np.inf)
    for b in range(K):
        s = float(scores[b])
        if np.isnan(s) or s == -np.inf:
            continue
        n = int(lengths[b]) + (0 if finished[b] else 1)
        if finished[b]:
            total[b, pad] = s
        else:
            top = x[b].max()
            if top == -np.inf:
                continue
            with np.errstate(over="ignore"):
                lse = np.log(np.exp(x[b] - top).sum())  # less the maximum, which is too large beside it in some rows
            total[b] = np.where(x[b] > -np.inf, s + ((x[b] - top) - lse), -np.inf)
        rank[b] = total[b] * float(max(n, 1)) ** -penalty
    return total, rank


def select(logits, scores, lengths, finished, groups: int, beams: int, num: int, eos: int, pad: int, penalty: float):
    """logits [groups * beams, V] -> dict of [groups, num] arrays."""
    V = logits.shape[1]
    out = dict(scores=np.full((groups, num), -np.inf), tokens=np.full((groups, num), -1), parents=np.full((groups, num), -1),
               lengths=np.zeros((groups, num), int), finished=np.zeros((groups, num), int),
               sources=np.full((groups, num), -1))
    for g in range(groups):
        rows = slice(g * beams, (g + 1) * beams)
        total, rank = continuations(logits[rows], scores[rows], lengths[rows], finished[rows], V, pad, penalty)
        order = np.argsort(-rank.reshape(-1), kind="stable")
        for i, at in enumerate(order[:num]):
            if not total.reshape(-1)[at] > -np.inf:
                break
            b, t = divmod(int(at), V)
            over = bool(finished[g * beams + b])
            end = over or t == eos
            out["scores"][g, i] = total[b, t]
            out["tokens"][g, i] = t
            out["parents"][g, i] = g * beams + b
            out["lengths"][g, i] = lengths[g * beams + b] + (0 if over else 1)
            out["finished"][g, i] = int(end)
            out["sources"][g, i] = -1 if end else g * beams + b
    return out


def fork(refs, tables, lengths, parents, advance: int, rows: int, absent: int = -1):
    """-> (refs, tables, lengths, copies, missing pages), the inputs left alone."""
    refs = [int(r) for r in refs]
    tables = [[int(p) for p in t] for t in tables]
    n, ld = len(tables), len(tables[0])

    def is_page(p):
        return 0 <= p < len(refs) and p != absent

    L = []
    for i in range(n):
        p = i if parents is None else int(parents[i])
        L.append(min(max(int(lengths[p]) + advance, 0), ld * PAGE) if 0 <= p < n else 0)
    out = []
    for i in range(n):
        p = i if parents is None else int(parents[i])
        have = -(-L[i] // PAGE)
        row = [tables[p][e] if e < have and is_page(tables[p][e]) else absent for e in range(ld)] if 0 <= p < n \
            else [absent] * ld
        out.append(row)
    for t in tables:
        for p in t:
            if is_page(p):
                refs[p] -= 1
    for t in out:
        for p in t:
            if is_page(p):
                refs[p] += 1
    # which sequences copy (the sharing is settled before any page is taken)
    copying = [False] * n
    for i in range(n):
        if rows > 0 and L[i] % PAGE:
            p = out[i][L[i] // PAGE]
            if is_page(p) and refs[p] > 1:
                refs[p] -= 1
                copying[i] = True
    free = [p for p in range(len(refs)) if refs[p] == 0 and p != absent]
    copies, missing = [], 0

    def take():
        nonlocal missing
        if not free:
            missing += 1
            return absent
        p = free.pop(0)
        refs[p] = 1
        return p

    for i in range(n):
        at = L[i] // PAGE
        if copying[i]:
            src = out[i][at]
            out[i][at] = take()
            if out[i][at] != absent:
                copies.append((src, out[i][at], L[i] % PAGE))
        for e in range(-(-L[i] // PAGE), -(-(L[i] + rows) // PAGE)):
            if e < ld:
                out[i][e] = take()
            else:
                missing += 1
    return np.array(refs), np.array(out), np.array(L), copies, missing
