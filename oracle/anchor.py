"""Float64 definitions of the softmax anchor layers' operators, on the CPU: attention over packed sequences with its
gradients, rotary positions, and attention of new tokens over pages.

Each also gives what its roundings can do to a bf16 or fp32 implementation, from the sums of absolute values: a weight that
is rounded by a relative u moves y_i by at most u sum_j p_ij |v_j|, and so on (`bounds`)."""
import math

import torch


def _visible(nq: int, nk: int) -> torch.Tensor:
    """(nq, nk): query i sees keys j <= i + nk - nq."""
    return torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)


def softmax(z: torch.Tensor, seen: torch.Tensor):
    """(weights, log of the sum of exponentials) over the seen entries of each row; a row without any has weights 0."""
    z = z.masked_fill(~seen, -math.inf)
    top = z.max(dim=-1, keepdim=True).values if z.shape[-1] else torch.full((*z.shape[:-1], 1), -math.inf, dtype=z.dtype)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z - top)
    s = e.sum(dim=-1, keepdim=True)
    return torch.where(s > 0, e / s, torch.zeros_like(e)), (torch.log(s) + top).squeeze(-1)


def attention(q, k, v, cu_q, cu_k=None, scale=None, dy=None, visible=_visible):
    """{"y", "lse" (H, tokens)} and, with dy, {"dq", "dk", "dv"}; under "bounds" for each the sums that rounding errors scale
    with ({name: (of rounded weights, of rounded dy . y)}).  `visible`: which keys queries see, of their numbers."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    cu_q = [int(x) for x in cu_q]
    cu_k = cu_q if cu_k is None else [int(x) for x in cu_k]
    H, KV = q.shape[1], k.shape[1]
    G, scale = H // KV, 1 / math.sqrt(q.shape[2]) if scale is None else scale
    r = dict(y=torch.zeros_like(q), lse=torch.full((H, q.shape[0]), -math.inf, dtype=torch.float64))
    b = dict(y=torch.zeros_like(q))
    if dy is not None:
        dy = dy.detach().cpu().double()
        r.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        b.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    most = 0.0
    for i0, i1, j0, j1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        seen = visible(i1 - i0, j1 - j0)
        for h in range(H):
            e = h // G
            qq, kk, vv = q[i0:i1, h], k[j0:j1, e], v[j0:j1, e]
            p, lse = softmax(qq @ kk.T * scale, seen)
            if p.numel():
                most = max(most, float((qq.abs() @ kk.abs().T).max()) * scale)
            y = p @ vv
            r["y"][i0:i1, h], r["lse"][h, i0:i1], b["y"][i0:i1, h] = y, lse, p @ vv.abs()
            if dy is not None:
                g = dy[i0:i1, h]
                dp = g @ vv.T
                delta = (g * y).sum(1, keepdim=True)
                ds = p * (dp - delta)
                # ds rounded once; delta from a y that was rounded; p and dp exact to fp32
                slack = ds.abs() + p * ((g.abs() * y.abs()).sum(1, keepdim=True))
                r["dq"][i0:i1, h] = ds @ kk * scale
                r["dk"][j0:j1, e] += ds.T @ qq * scale
                r["dv"][j0:j1, e] += p.T @ g
                b["dq"][i0:i1, h] = slack @ kk.abs() * scale
                b["dk"][j0:j1, e] += slack.T @ qq.abs() * scale
                b["dv"][j0:j1, e] += p.T @ g.abs()
    r["bounds"], r["most"] = b, most
    return r


def rotary(x, positions, inv_freq, interleaved=False, magnitude=1.0, inverse=False):
    x, f = x.detach().cpu().double(), inv_freq.detach().cpu().double()
    rot = 2 * f.shape[0]
    t = positions.detach().cpu().double()[:, None] * f[None]
    c, s = (torch.cos(t) * magnitude)[:, None], (torch.sin(t) * magnitude)[:, None] * (-1 if inverse else 1)
    y = x.clone()
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def tree_attention(q, k, v, k_pages, v_pages, page_table, context_lens, cu, parents=None, scale=None):
    """(y, sum of p |v|): each stream's new tokens over its pages and their ancestors."""
    q, k, v, kp, vp = (t.detach().cpu().double() for t in (q, k, v, k_pages, v_pages))
    H, KV, P = q.shape[1], k.shape[1], kp.shape[2]
    G, scale = H // KV, 1 / math.sqrt(q.shape[2]) if scale is None else scale
    y, bound = torch.zeros_like(q), torch.zeros_like(q)
    cu = [int(x) for x in cu]
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        L, n = int(context_lens[b]), hi - lo
        pages = [int(x) for x in page_table[b][:-(-L // P)]]
        kc = kp[pages].transpose(1, 2).reshape(-1, KV, q.shape[2])[:L]
        vc = vp[pages].transpose(1, 2).reshape(-1, KV, q.shape[2])[:L]
        seen = torch.zeros(n, L + n, dtype=torch.bool)
        seen[:, :L] = True
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, L + j] = True
                j = j - 1 if parents is None else int(parents[lo + j])
        for h in range(H):
            kk, vv = torch.cat([kc[:, h // G], k[lo:hi, h // G]]), torch.cat([vc[:, h // G], v[lo:hi, h // G]])
            z = q[lo:hi, h] @ kk.T * scale
            p, _ = softmax(z, seen)
            vv = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv)) if not torch.isfinite(vv).all() else vv
            y[lo:hi, h], bound[lo:hi, h] = p @ vv, p @ vv.abs()
    return y, bound
