"""Float64 definitions of the operators of bounded contexts, on the CPU: what a row sees under a window with sinks, attention of
new tokens over pages under it, the weight that each key got, and the eviction of the keys of least weight."""
import math

import torch

from . import anchor as oa


def visible(window=None, sinks=0):
    """(nq, nk) -> (nq, nk): query i, at position p = i + nk - nq, sees key j <= p if j > p - window or j < sinks."""
    def seen(nq, nk):
        p, j = torch.arange(nq)[:, None] + (nk - nq), torch.arange(nk)[None]
        return (j <= p) if window is None else (j <= p) & ((j > p - window) | (j < sinks))
    return seen


def attention(q, k, v, cu_q, cu_k=None, scale=None, dy=None, window=None, sinks=0):
    return oa.attention(q, k, v, cu_q, cu_k, scale, dy, visible(window, sinks))


def weights(q, k, lse, cu_q, cu_k=None, scale=None, window=None, sinks=0):
    """Of each sequence (H_kv, keys): the sum of exp(scale q.k - lse) over the rows that see a key and the heads that share its head."""
    q, k, lse = (t.detach().cpu().double() for t in (q, k, lse))
    cu_q = [int(x) for x in cu_q]
    cu_k = cu_q if cu_k is None else [int(x) for x in cu_k]
    H, KV = q.shape[1], k.shape[1]
    scale, out = 1 / math.sqrt(q.shape[2]) if scale is None else scale, []
    for i0, i1, j0, j1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        seen, w = visible(window, sinks)(i1 - i0, j1 - j0), torch.zeros(KV, j1 - j0, dtype=torch.float64)
        for h in range(H):
            z = q[i0:i1, h] @ k[j0:j1, h * KV // H].T * scale - lse[h, i0:i1, None]
            w[h * KV // H] += torch.where(seen, torch.exp(z), torch.zeros_like(z)).sum(0)
        out.append(w)
    return out


def tree_attention(q, k, v, k_pages, v_pages, page_table, context_lens, cu, parents=None, scale=None, window=None, sinks=0):
    """(y, sum of p |v|, [each stream's (H_kv, context + new tokens) weights]): each stream's new tokens over its pages and their
    ancestors; a token is at the context's length plus its depth."""
    q, k, v, kp, vp = (t.detach().cpu().double() for t in (q, k, v, k_pages, v_pages))
    H, KV, P = q.shape[1], k.shape[1], kp.shape[2]
    G, scale = H // KV, 1 / math.sqrt(q.shape[2]) if scale is None else scale
    y, bound, w = torch.zeros_like(q), torch.zeros_like(q), []
    cu = [int(x) for x in cu]
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        L, n = int(context_lens[b]), hi - lo
        pages = [int(x) for x in page_table[b][:-(-L // P)]]
        kc, vc = (x[pages].transpose(1, 2).reshape(-1, KV, q.shape[2])[:L] for x in (kp, vp))
        seen, depth = torch.zeros(n, L + n, dtype=torch.bool), []
        for i in range(n):
            up = i - 1 if parents is None else int(parents[lo + i])
            depth.append(depth[up] + 1 if up >= 0 else 0)
            here, j = L + depth[i], i
            while j >= 0:
                seen[i, L + j] = window is None or depth[i] - depth[j] < window or L + depth[j] < sinks
                j = j - 1 if parents is None else int(parents[lo + j])
            at = torch.arange(L)
            seen[i, :L] = True if window is None else (at > here - window) | (at < sinks)
        got = torch.zeros(KV, L + n, dtype=torch.float64)
        for h in range(H):
            kk, vv = torch.cat([kc[:, h // G], k[lo:hi, h // G]]), torch.cat([vc[:, h // G], v[lo:hi, h // G]])
            kk, vv = (torch.where(seen.any(0)[:, None], t, torch.zeros_like(t)) for t in (kk, vv))  # what nobody sees may be anything
            p, _ = oa.softmax(q[lo:hi, h] @ kk.T * scale, seen)
            y[lo:hi, h], bound[lo:hi, h] = p @ vv, p @ vv.abs()
            got[h // G] += p.sum(0)
        w.append(got)
    return y, bound, w


def evict(weights, positions, length, keep, settled=0, evicted=0, sinks=0, recent=0):
    """One head's (moves [(from, to)], weights, positions) of `length` cached places cut to min(length, keep), lists in and out.
    Place j holds position positions[j] if j < settled, else j + evicted.  First stay the positions below `sinks`, then the last
    `recent` of all length + evicted, then the largest weights (those that are no positive numbers count as 0), of equals the
    lowest places; the kept ones from the new length on take the given-up ones' places before it, both in order."""
    at = [positions[j] if j < settled else j + evicted for j in range(length)]
    n = min(length, keep)

    def rank(j):
        w = weights[j]
        return (3, 0.0) if at[j] < sinks else (2, 0.0) if at[j] >= length + evicted - recent else (1, w if w > 0 else 0.0)

    kept = set(sorted(range(length), key=lambda j: (-rank(j)[0], -rank(j)[1], j))[:n])
    moves = list(zip((j for j in range(n, length) if j in kept), (j for j in range(n) if j not in kept)))
    weights, positions = list(weights), list(positions)
    positions[:n] = at[:n]
    for src, dst in moves:
        weights[dst], positions[dst] = weights[src], at[src]
    return moves, weights, positions
