"""Policy sampling in float64 -- TEST INFRASTRUCTURE ONLY (the oracle).

Restates, one row at a time and in NumPy, what ``onyx_policy_sample``, ``onyx_policy_probs``
and ``onyx_spec_sample`` define (include/onyx_b200.h): weights ``exp((v - max) / T)`` of the
valid ids (+inf ids share the mass alone; T = 0 keeps the first maximum), ids ranked by value
with the lowest first among equals, top-k, top-p over the top-k mass, min-p against the
largest weight; the draw walks the kept ids in id order. With top_k = 0 and min_p = 0 the
kept set is that of ``oracle.sampling.kept_weights`` (the reference's
``_filtered_reference_weights``, onyx_cuda/src/onyx_cuda/selection.py).
"""

from __future__ import annotations

import math

import numpy as np

from .sampling import unpack_mask

STATUS_EMPTY_MASK = 1
STATUS_ALL_NEG_INF = 2
STATUS_NAN_IN_SUPPORT = 4
STATUS_BAD_POLICY = 32


def policy_ok(policy) -> bool:
    t, k, p, m = (float(x) for x in policy)
    return (0.0 <= t < math.inf and 0.0 <= k < math.inf and k == math.floor(k)
            and 0.0 < p <= 1.0 and 0.0 <= m <= 1.0)


def kept_weights(values, valid, policy) -> tuple[int, np.ndarray]:
    """(status, float64 weights of every id: 0 where it is not kept)."""
    values = np.asarray(values, dtype=np.float64)
    out = np.zeros(values.size)
    if not policy_ok(policy):
        return STATUS_BAD_POLICY, out
    t, k, p, m = (float(x) for x in policy)
    ids = np.flatnonzero(valid)
    if ids.size == 0:
        return STATUS_EMPTY_MASK, out
    v = values[ids]
    if np.isnan(v).any():
        return STATUS_NAN_IN_SUPPORT, out
    top = v.max()
    if top == -math.inf:
        return STATUS_ALL_NEG_INF, out
    if t == 0.0:
        out[ids[int(np.argmax(v))]] = 1.0
        return 0, out
    if top == math.inf:
        ids = ids[v == math.inf]
        v = np.zeros(ids.size)
        w = np.ones(ids.size)
    else:
        with np.errstate(over="ignore"):  # a tiny temperature: -inf, weight 0
            w = np.exp(np.where(v == top, 0.0, (v - top) / t))
    order = np.argsort(-v, kind="stable")
    if k:
        order = order[: int(min(k, order.size))]
    if p < 1.0:
        cum = np.cumsum(w[order])
        order = order[: int(np.argmax(cum >= p * cum[-1])) + 1]
    order = order[w[order] >= m]
    out[ids[order]] = w[order]
    return 0, out


def choose(weights: np.ndarray, u: float) -> int:
    """First id, in id order, whose cumulative weight exceeds u times the total."""
    ids = np.flatnonzero(weights > 0.0)
    cum = np.cumsum(weights[ids])
    past = np.flatnonzero(cum > u * cum[-1])
    return int(ids[past[0]] if past.size else ids[-1])


def _valid(masks, row, vocab):
    return np.ones(vocab, bool) if masks is None else unpack_mask(masks[row], vocab)


def sample(values, masks, policies, uniforms) -> tuple[np.ndarray, np.ndarray]:
    """values [B, V], masks [B, W] or None, policies [B, 4], uniforms [B]."""
    rows, vocab = np.shape(values)
    ids, status = np.full(rows, -1, np.int32), np.zeros(rows, np.uint32)
    for r in range(rows):
        st, w = kept_weights(values[r], _valid(masks, r, vocab), policies[r])
        if not 0.0 <= float(uniforms[r]) < 1.0:
            st = STATUS_BAD_POLICY
        status[r] = st
        if not st:
            ids[r] = choose(w, float(uniforms[r]))
    return ids, status


def probs(values, masks, policies) -> tuple[np.ndarray, np.ndarray]:
    """float64 probabilities [B, V] and status."""
    rows, vocab = np.shape(values)
    out, status = np.zeros((rows, vocab)), np.zeros(rows, np.uint32)
    for r in range(rows):
        status[r], w = kept_weights(values[r], _valid(masks, r, vocab), policies[r])
        if not status[r]:
            out[r] = w / w.sum()
    return out, status


def spec(values, masks, drafts, policies, uniforms, draft_probs=None, draft_lens=None,
         drawn_from=None):
    """values [B, G+1, V], masks [B, G+1, W] or None, drafts [B, G], policies [B, 4],
    uniforms [B, G+1], draft_probs [B, G, V] or None, draft_lens [B] or None. Entry b's token
    was drawn from the weights that the dict `drawn_from`, if given, gets under b."""
    batch, g1, vocab = np.shape(values)
    taken, token = np.zeros(batch, np.int32), np.full(batch, -1, np.int32)
    status = np.zeros(batch, np.uint32)
    for b in range(batch):
        n = g1 - 1 if draft_lens is None else int(draft_lens[b])
        last = float(uniforms[b, g1 - 1])
        if not 0 <= n < g1 or not 0.0 <= last < 1.0:
            status[b] = STATUS_BAD_POLICY
            continue
        i = 0
        while True:
            u = float(uniforms[b, i]) if i < n else 0.0
            st, w = kept_weights(values[b, i],
                                 _valid(None if masks is None else masks[b], i, vocab),
                                 policies[b])
            if not 0.0 <= u < 1.0:
                st = STATUS_BAD_POLICY
            if st:
                status[b] = st
                break
            if i == n:
                drawn, token[b] = w, choose(w, last)
                break
            p, d = w / w.sum(), int(drafts[b, i])
            inside = 0 <= d < vocab
            if draft_probs is None:
                q = np.zeros(vocab)
                if inside:
                    q[d] = 1.0
            else:
                q = np.asarray(draft_probs[b, i], np.float64)
                q = np.where(q > 0.0, q, 0.0)
            if inside and u * q[d] < p[d]:
                i += 1
                continue
            rest = np.maximum(p - q, 0.0)
            drawn = rest if rest.sum() > 0.0 else w
            token[b] = choose(drawn, last)
            break
        if drawn_from is not None and not status[b]:
            drawn_from[b] = drawn
        taken[b] = i
    return taken, token, status
