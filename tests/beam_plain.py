"""Beam search in 64 bits on numpy: the choice and the reordering."""
from __future__ import annotations

import numpy as np


def scores_of(x, base):
    """Scores [beams][vocab] of logits x, float64; -infinity where there is no continuation."""
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        s = base[:, None] + ((x - top) - np.log(np.exp(x - top).sum(-1, keepdims=True)))
    s[np.isnan(s)] = -np.inf
    s[~(base > -np.inf)] = -np.inf
    return s


def choose(x, base, keep, ended=None, end=-1):
    """One text: logits [beams][vocab] and scores [beams] as float64 -> (scores, parents, tokens, ended), and the
    score after the last one kept (or -infinity)."""
    beams, vocab = x.shape
    s = scores_of(x, base)
    if ended is not None:
        for i in np.nonzero(ended)[0]:
            s[i] = -np.inf
            if base[i] > -np.inf:
                s[i, end] = base[i]
    flat = s.reshape(-1)
    at = np.arange(beams * vocab)
    order = np.lexsort((at, -x.reshape(-1), at // vocab, -flat))  # ties: the lower beam, the larger logit, the lower token
    order = order[flat[order] > -np.inf]
    near, order = order[:keep + 1], order[:keep]
    out = [np.full(keep, -np.inf), np.minimum(np.arange(keep), beams - 1), np.full(keep, -1), np.zeros(keep, np.uint8)]
    n = len(order)
    out[0][:n], out[1][:n], out[2][:n] = flat[order], order // vocab, order % vocab
    was = np.zeros(beams, bool) if ended is None else np.asarray(ended, bool)
    out[3][:n] = (out[2][:n] == end) | was[out[1][:n]]
    return out, flat[near]


def reorder(parents, table, lengths, spare, beams, page, pages):
    """(rows' parents, table_out, spare_out, copies [(from page, to page, tokens)]) in plain steps."""
    rows = len(table)
    frm, out, left, copies = np.arange(rows), table.copy(), spare.copy(), []
    for r in range(rows):
        if 0 <= parents[r] < beams:
            frm[r] = r // beams * beams + parents[r]
        f = frm[r]
        if f == r:
            continue
        full, part = divmod(max(int(lengths[f]), 0), page)
        out[r, :full] = table[f, :full]
        if part and full < table.shape[1]:
            if not 0 <= table[f, full] < pages:
                out[r, full] = table[f, full]
                continue
            out[r, full], left[r] = spare[r], table[r, full]
            if 0 <= spare[r] < pages:
                copies.append((table[f, full], spare[r], part))
    return frm, out, left, copies
