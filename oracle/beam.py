"""Beam search in 64 bits: selection, and what becomes of the pages."""

import numpy as np


def keys(logits, scores, done=None, pad_token=0):
    """``[batch, beams * vocab]``: every continuation's score; -inf where none is offered."""
    batch, beams = scores.shape
    x = np.asarray(logits, np.float64).reshape(batch, beams, -1)
    x = np.where(np.isnan(x), -np.inf, x)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(-1, keepdims=True)
        out = np.asarray(scores, np.float64)[:, :, None] + ((x - m) - np.log(np.exp(x - m).sum(-1, keepdims=True)))
    out = np.where(np.isnan(out), -np.inf, out)
    out[~np.isfinite(m[..., 0])] = -np.inf
    if done is not None:
        out[done] = -np.inf
        b, j = np.nonzero(done)
        out[b, j, pad_token] = np.where(np.isnan(scores[b, j]), -np.inf, scores[b, j])
    return out.reshape(batch, -1)


def select(all_keys, n):
    """Places of the n best, equal ones in order."""
    return np.argsort(-all_keys, axis=1, kind="stable")[:, :n]


def reorder(table, lens, refs, parents, page):
    """``(table, lens, refs, ok, copies)`` after every row became its parent's; ``copies`` lists
    ``(from, to)`` pages."""
    rows, cols = table.shape
    n_pages = len(refs)
    new, new_len, ok, need = np.full_like(table, -1), np.zeros_like(lens), np.ones(rows, np.int32), {}
    for i, p in enumerate(parents):
        if not 0 <= p < rows:
            continue
        heir = p == i or (parents[p] != p and not np.any(parents[:i] == p))
        if heir:
            new[i], new_len[i] = table[p], lens[p]
            continue
        whole = int(lens[p]) // page
        part = lens[p] % page > 0
        if not 0 <= lens[p] <= cols * page or (part and not 0 <= table[p][whole] < n_pages):
            ok[i] = 0
            continue
        new[i, :whole], new_len[i] = table[p][:whole], lens[p]
        if part:
            need[i] = int(table[p][whole])
    # counts change by what entries change
    refs = refs.copy()
    for before, sign in ((table, -1), (new, 1)):
        for i in range(rows):
            for pg in before[i]:
                if 0 <= pg < n_pages:
                    refs[pg] += sign
    free = list(np.nonzero(refs == 0)[0])
    copies = []
    given_up = []
    for i, src in need.items():
        if not free:
            ok[i], new_len[i] = 0, 0
            given_up.append(i)
            continue
        to = int(free.pop(0))
        new[i, new_len[i] // page] = to
        refs[to] = 1
        copies.append((src, to))
    for i in given_up:
        for pg in new[i]:
            if 0 <= pg < n_pages:
                refs[pg] -= 1
        new[i] = -1
    return new, new_len, refs, ok, copies
