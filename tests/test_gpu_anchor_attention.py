"""Packed causal attention and its gradients (kdn_attn_fwd, kdn_attn_bwd) against the float64 definition.

Tolerances, element by element, from the roundings alone.  bf16 (u = 2^-8): the weights and the output are rounded once
each, so y is within 2 u sum p |v|; dv within 2 u sum p |dy|; dk and dq have ds rounded (u |ds|), dy . y formed from a
rounded y (u p sum |dy| |y|) and the result rounded.  fp32 (u = 2^-24): a score is a sum of d products within d u of its
absolute sum, which the exponential turns into that relative error of a weight, and the sums over n rows add n u."""
import pytest
import torch

from kdn import anchor
from oracle import anchor as oa

DEV = "cuda:0"


def make(lens_q, lens_k, H, KV, d, dtype, seed=0, spread=1.0, grad=True):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(lens_q), sum(lens_k)
    q, k, v, dy = (torch.randn(n, h, d, generator=g).mul(s).to(dtype) for n, h, s in
                   ((nq, H, spread), (nk, KV, spread), (nk, KV, 1.0), (nq, H, 1.0)))
    cu = [torch.tensor([0] + list(torch.tensor(x).cumsum(0).tolist()) if x else [0], dtype=torch.int64) for x in (lens_q, lens_k)]
    return q, k, v, dy, cu[0], cu[1]


def unit(dtype, d, n, most):
    """The factor of the bounds: twice the rounding unit, or fp32's sums (see above) with two units for the exponentials."""
    return 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * ((d + 4) * (1 + most) + n + 8)


def close(got, want, bound, f, what):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    # the output's own rounding, and what a sum of exact terms loses in fp32
    slack = f * (bound + want.abs()) + 2.0 ** -24 * 64 * bound + 1e-30
    over = (got - want).abs() - slack
    assert float(over.max() if over.numel() else 0) <= 0, (what, float(((got - want).abs() / slack).max()))


def check(lens_q, lens_k=None, H=4, KV=2, d=64, dtype=torch.bfloat16, spread=1.0, scale=None, seed=0, low=True):
    q, k, v, dy, cq, ck = make(lens_q, lens_q if lens_k is None else lens_k, H, KV, d, dtype, seed, spread)
    dev = [t.to(DEV) for t in (q, k, v, dy, cq, ck)]
    cks = None if lens_k is None else dev[5]
    y, lse, rest = anchor.attention_forward(*dev[:3], dev[4], cks, scale, return_lse=True, return_low=True)
    dq, dk, dv = anchor.attention_backward(*dev[:3], y, lse, dev[3], dev[4], cks, scale, rest if low else None)
    want = oa.attention(q, k, v, cq, None if lens_k is None else ck, scale, dy)
    n = max([1, *lens_q]) * (H // KV) + max([1, *(lens_k or lens_q)])
    f = unit(dtype, d, n, want["most"])
    b = want["bounds"]
    close(y, want["y"], b["y"], f, "y")
    live = torch.isfinite(want["lse"])
    assert torch.equal(torch.isneginf(lse.cpu()), ~live)
    if live.any():
        err = (lse.cpu().double() - want["lse"])[live].abs().max()
        assert float(err) <= 2.0 ** -24 * ((d + 4) * (1 + want["most"]) + n + 8), float(err)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        # fp32's weights carry their own relative error into every term (the same factor); bf16's bound has it in 2 u
        close(got, want[name], b[name], 2 * f, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [33, 31, 32], [63, 64, 65], [127, 128, 129], [300, 5]])
def test_lengths(lens, d, dtype):
    check(lens, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV", [(1, 1), (3, 3), (6, 2), (8, 1), (16, 4), (5, 1)])
def test_head_groups(H, KV):
    check([70, 141], H=H, KV=KV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens_q,lens_k", [([5], [200]), ([200], [5]), ([130, 70], [0, 70]), ([0, 40], [33, 40]), ([64], [65]), ([129], [1]),
                                           ([1, 1], [700, 0])])
def test_own_key_lengths_and_empty_rows(lens_q, lens_k, dtype):
    check(lens_q, lens_k, dtype=dtype)


@pytest.mark.gpu
def test_many_short_sequences():
    check([(7 * i) % 23 for i in range(150)], H=2, KV=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [60, 115])
def test_enough_rows_for_fewer_waves_a_row(n, d, dtype):
    """8700 and 17000 rows of 4 heads: two waves a row, and one (the others here have too few rows for that)."""
    check([(37 * i) % 301 for i in range(n)], H=4, KV=4, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_longer(d):
    check([1111], H=2, KV=1, d=d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wide_scores(dtype):
    """Scores of hundreds: one weight near 1, the running maximum moving often."""
    check([260], spread=6.0, dtype=dtype)


@pytest.mark.gpu
def test_scale():
    check([100], scale=0.5)


@pytest.mark.gpu
def test_without_the_low_part():
    check([100, 3], low=False)


@pytest.mark.gpu
def test_low_part():
    """y and its low part together are the unrounded result, to the low part's own rounding, 2^-16 of y: what is left is the
    weights' rounding, 2^-8 sum p |v|."""
    q, k, v, dy, cu, _ = make([90], [90], 4, 2, 64, torch.bfloat16)
    y, lse, low = anchor.attention_forward(*(t.to(DEV) for t in (q, k, v)), cu.to(DEV), return_lse=True, return_low=True)
    assert float((low.float().abs() - 2.0 ** -8 * y.float().abs()).max()) <= 0
    want = oa.attention(q, k, v, cu)
    off = (y.double() + low.double()).cpu() - want["y"]
    assert float((off.abs() - (2.0 ** -8 + 2.0 ** -18) * want["bounds"]["y"] - 2.0 ** -15 * want["y"].abs()).max()) <= 0
    assert anchor.attention_forward(*(t.float().to(DEV) for t in (q, k, v)), cu.to(DEV), return_lse=True, return_low=True)[2] is None


@pytest.mark.gpu
def test_strided_views_and_other_layouts():
    lens = [77, 130]
    q, k, v, dy, cu, _ = make(lens, lens, 4, 2, 64, torch.bfloat16)
    cu = cu.to(DEV)
    plain = anchor.attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), cu)
    fused = torch.cat([q, k, v], dim=1).to(DEV).split([4, 2, 2], dim=1)
    assert torch.equal(anchor.attention_forward(*fused, cu), plain)
    major = [t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # heads outermost
    assert torch.equal(anchor.attention_forward(*major, cu), plain)
    odd = torch.empty(207, 4, 68, dtype=torch.bfloat16, device=DEV)[..., 2:66]  # rows that start off 16 bytes: copied
    odd.copy_(q)
    assert torch.equal(anchor.attention_forward(odd, k.to(DEV), v.to(DEV), cu), plain)
    out = torch.zeros(207, 8, 64, dtype=torch.bfloat16, device=DEV)
    anchor.attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), cu, out=out[:, ::2])
    assert torch.equal(out[:, ::2], plain) and not out[:, 1::2].any()
    one_key = k[:, :1].to(DEV).expand(-1, 2, -1)  # a broadcast head
    same = anchor.attention_forward(q.to(DEV), one_key.contiguous(), v.to(DEV), cu)
    assert torch.equal(anchor.attention_forward(q.to(DEV), one_key, v.to(DEV), cu), same)


@pytest.mark.gpu
def test_other_sequences_and_padding_do_not_reach_a_row():
    lens = [50, 64, 90]
    q, k, v, dy, cu, _ = make(lens, lens, 4, 2, 64, torch.bfloat16)
    pad = 13
    grow = lambda t: torch.cat([t, torch.full((pad, *t.shape[1:]), float("nan"), dtype=t.dtype)]).to(DEV)  # noqa: E731
    q2, k2, v2, dy2 = map(grow, (q, k, v, dy))
    bad = slice(50, 114)
    for t in (q2, k2, v2, dy2):
        t[bad] = float("inf")
    y, lse = anchor.attention_forward(q2, k2, v2, cu.to(DEV), return_lse=True)
    grads = anchor.attention_backward(q2, k2, v2, y, lse, dy2, cu.to(DEV))
    y0, lse0 = anchor.attention_forward(*(t.to(DEV) for t in (q, k, v)), cu.to(DEV), return_lse=True)
    grads0 = anchor.attention_backward(*(t.to(DEV) for t in (q, k, v)), y0, lse0, dy.to(DEV), cu.to(DEV))
    for a, b in ((y, y0), *zip(grads, grads0)):
        assert torch.equal(a[:50], b[:50]) and torch.equal(a[114:204], b[114:204])
        assert not a[204:].any()  # rows past the last sequence: zeros
    assert torch.isneginf(lse[:, 204:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 100, 150])
def test_values_of_unseen_keys_do_not_reach_a_row(n, d, dtype):
    """A few values infinite or NaN: a row has them only where it sees their keys, everything else stays a number.  (n sequences
    of 240 tokens and four heads: four, two and one wave to a row.)"""
    q, k, v, dy, cu, _ = make([240] * n, [240] * n, 4, 2, d, dtype)
    clean = v.clone()
    inf, nan = float("inf"), float("nan")
    rare = torch.zeros(240, 2, d, dtype=torch.float64)  # in the first and the last sequence
    for at, e, x, value in ((37, 0, 3, inf), (70, 0, 3, inf), (70, 0, 40, -inf), (101, 0, 3, -inf), (130, 1, d - 1, nan), (239, 1, 0, inf), (0, 1, 7, -inf)):
        rare[at, e, x] = value
    dirty = torch.isnan(rare) | (rare != 0)
    for b in {0, n - 1}:
        v[240 * b:240 * (b + 1)][dirty] = rare[dirty].to(dtype)
        clean[240 * b:240 * (b + 1)][dirty] = 0
    y = anchor.attention_forward(*(t.to(DEV) for t in (q, k, v, cu))).cpu().double()
    some = [0, n - 1, n // 2]
    pick = lambda t: torch.cat([t[240 * b:240 * (b + 1)] for b in some])  # noqa: E731
    got = pick(y).view(3, 240, 4, d)
    want = oa.attention(pick(q), pick(k), pick(clean), torch.arange(4) * 240)
    extra = rare.cumsum(0).repeat_interleave(2, 1)  # what a row has seen: infinities that meet are no number
    reached = torch.isnan(extra) | (extra != 0)
    for i, b in enumerate(some):
        g = got[i].clone()
        if b in (0, n - 1):
            assert torch.equal(torch.isnan(g), torch.isnan(extra)) and torch.equal(torch.isinf(g), torch.isinf(extra))
            assert torch.equal(g[torch.isinf(extra)], extra[torch.isinf(extra)])
            g[reached] = want["y"].view(3, 240, 4, d)[i][reached]
        close(g, want["y"].view(3, 240, 4, d)[i], want["bounds"]["y"].view(3, 240, 4, d)[i], unit(dtype, d, 480, want["most"]), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unseen_keys_that_are_no_numbers(dtype):
    """NaN and infinite keys and values from token 100 on: the rows before are what they are without them, the rows after NaN."""
    q, k, v, dy, cu, _ = make([180], [180], 4, 2, 64, dtype)
    want = oa.attention(q[:100], k[:100], v[:100], torch.tensor([0, 100]))
    k[100], k[101:], v[100:] = float("nan"), float("inf"), float("nan")
    y, lse = anchor.attention_forward(*(t.to(DEV) for t in (q, k, v, cu)), return_lse=True)
    close(y[:100], want["y"], want["bounds"]["y"], unit(dtype, 64, 200, want["most"]), "y")
    assert torch.isfinite(lse[:, :100]).all() and torch.isnan(y[100:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_bits_every_time(dtype):
    lens = [300, 17]
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make(lens, lens, 8, 2, 128, dtype))
    first = None
    for _ in range(3):
        y, lse = anchor.attention_forward(q, k, v, cu, return_lse=True)
        now = (y, lse, *anchor.attention_backward(q, k, v, y, lse, dy, cu))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32: along a direction, (f(x + h u) - f(x - h u)) / 2h with h = 2^-6: the differences' own error, h^2/6 of the third
    derivative and the forward's rounding over h, stays under 2^-9 of the gradient's size for these sizes."""
    lens = [37, 70]
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make(lens, lens, 4, 2, 64, torch.float32, seed=3))
    y, lse = anchor.attention_forward(q, k, v, cu, return_lse=True)
    grads = anchor.attention_backward(q, k, v, y, lse, dy, cu)
    g = torch.Generator().manual_seed(9)
    h = 2.0 ** -6
    for i, grad in enumerate(grads):
        u = torch.randn(grad.shape, generator=g).to(DEV)
        xs = [q, k, v]
        f = []
        for s in (h, -h):
            ys = list(xs)
            ys[i] = xs[i] + s * u
            f.append(float((anchor.attention_forward(*ys, cu).double() * dy.double()).sum()))
        slope, want = (f[0] - f[1]) / (2 * h), float((grad.double() * u.double()).sum())
        assert abs(slope - want) <= 2.0 ** -9 * float(grad.norm()) * float(u.norm()) / grad.numel() ** 0.5, (i, slope, want)


@pytest.mark.gpu
def test_autograd_and_uniform_batches():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(3, 45, h, 64, generator=g).to(DEV, torch.bfloat16).requires_grad_(True) for h in (4, 2, 2))
    y = anchor.attention(q, k, v)
    dy = torch.randn(y.shape, generator=g).to(DEV, torch.bfloat16)
    y.backward(dy)
    cu = torch.arange(0, 4 * 45, 45, device=DEV)
    flat = [t.detach().reshape(-1, *t.shape[2:]) for t in (q, k, v)]
    y2, lse, low = anchor.attention_forward(*flat, cu.int(), return_lse=True, return_low=True)
    grads = anchor.attention_backward(*flat, y2, lse, dy.reshape(y2.shape), cu, low=low)
    assert torch.equal(y.detach().reshape(y2.shape), y2)
    for t, want in zip((q, k, v), grads):
        assert torch.equal(t.grad.reshape(want.shape), want)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    lens = [129, 40]
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make(lens, lens, 4, 2, 64, torch.bfloat16))
    y0, lse0 = anchor.attention_forward(q, k, v, cu, return_lse=True)
    g0 = anchor.attention_backward(q, k, v, y0, lse0, dy, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y1, lse1 = anchor.attention_forward(q, k, v, cu, return_lse=True)
        g1 = anchor.attention_backward(q, k, v, y1, lse1, dy, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y0, y1) and all(torch.equal(a, b) for a, b in zip(g0, g1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, lse2 = anchor.attention_forward(q, k, v, cu, return_lse=True)
        g2 = anchor.attention_backward(q, k, v, y2, lse2, dy, cu)
    for r in range(3):
        q.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        y3, lse3 = anchor.attention_forward(q, k, v, cu, return_lse=True)
        g3 = anchor.attention_backward(q, k, v, y3, lse3, dy, cu)
        assert torch.equal(y2, y3) and all(torch.equal(a, b) for a, b in zip(g2, g3)), r


@pytest.mark.gpu
def test_empty_calls():
    z = torch.zeros(0, 4, 64, device=DEV, dtype=torch.bfloat16)
    cu = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert anchor.attention_forward(z, z, z, cu).shape == (0, 4, 64)
    q = torch.ones(5, 4, 64, device=DEV, dtype=torch.bfloat16)
    y, lse = anchor.attention_forward(q, z, z, torch.tensor([0, 5], device=DEV), torch.tensor([0, 0], device=DEV), return_lse=True)
    assert not y.any() and torch.isneginf(lse).all()
    dq, dk, dv = anchor.attention_backward(q, z, z, y, lse, q, torch.tensor([0, 5], device=DEV), torch.tensor([0, 0], device=DEV))
    assert not dq.any() and dk.shape == (0, 4, 64)


@pytest.mark.gpu
def test_refusals():
    q = torch.zeros(8, 4, 64, device=DEV, dtype=torch.bfloat16)
    cu = torch.tensor([0, 8], device=DEV)
    with pytest.raises(ValueError):
        anchor.attention(q, q[:, :3], q[:, :3], cu)       # 4 heads over 3
    with pytest.raises(ValueError):
        anchor.attention(q, q.float(), q, cu)             # mixed types
    with pytest.raises(ValueError):
        anchor.attention(q, q[:4], q[:4], cu)             # other keys without their offsets
    with pytest.raises(ValueError):
        anchor.attention(q, q, q)                         # packed without offsets
    with pytest.raises(ValueError):
        anchor.attention(q, q, q, cu, scale=0.0)
    with pytest.raises(ValueError):
        anchor.attention(q, q, q, cu.float())
    with pytest.raises(ValueError):
        anchor.attention(q, q, q, cu, out=torch.empty(8, 4, 66, device=DEV, dtype=torch.bfloat16)[..., 1:65])
    with pytest.raises(TypeError):
        anchor.attention(q.half(), q.half(), q.half(), cu)
    with pytest.raises(RuntimeError):
        anchor.attention(q[..., :32].contiguous(), q[..., :32].contiguous(), q[..., :32].contiguous(), cu)  # d = 32
    with pytest.raises(RuntimeError):
        anchor.attention(q.cpu(), q.cpu(), q.cpu(), cu)
