"""Attention that sees a sliding window and sinks, over packed prompts, and its gradients (kdn_attn_window_fwd, _bwd) against the
float64 definition.  The tolerances are those of the attention without a window, from its roundings alone: bf16 (u = 2^-8) rounds
the weights and the output once each, ds once more in the gradients; fp32 (u = 2^-24) has a score's d products, which the exponential
turns into a weight's relative error, and the sums over n rows."""
import pytest
import torch

from kdn import anchor
from oracle import bounded as ob

DEV = "cuda:0"


def make(lens_q, lens_k, H, KV, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(lens_q), sum(lens_k)
    q, k, v, dy = (torch.randn(n, h, d, generator=g).to(dtype) for n, h in ((nq, H), (nk, KV), (nk, KV), (nq, H)))
    return q, k, v, dy, torch.tensor([0, *lens_q]).cumsum(0), torch.tensor([0, *lens_k]).cumsum(0)


def close(got, want, bound, f, what):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    slack = f * (bound + want.abs()) + 2.0 ** -24 * 64 * bound + 1e-30
    over = (got - want).abs() - slack
    assert float(over.max() if over.numel() else 0) <= 0, (what, float(((got - want).abs() / slack).max()))


def check(lens_q, lens_k=None, window=40, sinks=4, H=4, KV=2, d=64, dtype=torch.bfloat16, scale=None, seed=0):
    q, k, v, dy, cq, ck = make(lens_q, lens_q if lens_k is None else lens_k, H, KV, d, dtype, seed)
    dev = [t.to(DEV) for t in (q, k, v, dy, cq, ck)]
    cks, how = None if lens_k is None else dev[5], dict(window=window, sinks=sinks)
    y, lse, low = anchor.attention_forward(*dev[:3], dev[4], cks, scale, return_lse=True, return_low=True, **how)
    grads = anchor.attention_backward(*dev[:3], y, lse, dev[3], dev[4], cks, scale, low, **how)
    want = ob.attention(q, k, v, cq, None if lens_k is None else ck, scale, dy, window, sinks)
    n = max([1, *lens_q]) * (H // KV) + max([1, *(lens_k or lens_q)])
    f = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * ((d + 4) * (1 + want["most"]) + n + 8)
    b = want["bounds"]
    close(y, want["y"], b["y"], f, "y")
    live = torch.isfinite(want["lse"])
    assert torch.equal(torch.isneginf(lse.cpu()), ~live)
    if live.any():
        err = (lse.cpu().double() - want["lse"])[live].abs().max()
        assert float(err) <= 2.0 ** -24 * ((d + 4) * (1 + want["most"]) + n + 8), float(err)
    for name, got in zip(("dq", "dk", "dv"), grads):
        close(got, want[name], b[name], 2 * f, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (31, 0), (32, 33), (33, 64), (64, 1), (65, 100), (127, 128), (128, 5)])
def test_windows(window, sinks, d, dtype):
    check([300, 1, 5, 0, 129], window=window, sinks=sinks, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV", [(1, 1), (6, 2), (8, 1), (16, 4)])
def test_head_groups(H, KV):
    check([70, 241], H=H, KV=KV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(3, 2), (50, 0), (64, 70)])
@pytest.mark.parametrize("lens_q,lens_k", [([5], [200]), ([200], [5]), ([130, 70], [0, 70]), ([0, 140], [33, 140]), ([64], [165]), ([229], [101]),
                                           ([1, 1], [700, 0]), ([500], [760])])
def test_own_key_lengths_and_empty_rows(lens_q, lens_k, window, sinks, dtype):
    check(lens_q, lens_k, window=window, sinks=sinks, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("sinks", [0, 4, 150, 256, 257, 400])
def test_rows_far_behind_the_sinks(sinks, dtype, d):
    """More than one segment of far rows to a sequence, their first inside a segment."""
    check([2500, 1100, 40], window=100, sinks=sinks, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype", [(40, torch.bfloat16), (70, torch.bfloat16), (40, torch.float32)])
def test_waves_with_rows_of_their_own(heads, dtype):
    """Batches large enough that two waves share 32 rows, and that none do (their number goes by rows and heads)."""
    check([1250, 700], window=130, sinks=4, H=heads, KV=heads // 2 if heads == 40 else heads, d=64, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,d,dtype", [(10, 64, torch.bfloat16), (10, 64, torch.float32), (20, 64, torch.bfloat16), (10, 128, torch.bfloat16),
                                           (20, 128, torch.bfloat16), (10, 128, torch.float32), (36, 128, torch.float32)])
def test_batches_between(heads, d, dtype):
    """Two waves to 32 rows, or one, at sizes between the smallest and those above, with rows far behind the sinks."""
    check([1350, 600], window=70, sinks=5, H=heads, KV=heads // 2, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [4, 24])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 4), (6, 1), (3, 0), (28, 4)])
def test_few_keys_in_bf16_are_as_exact_as_many(window, sinks, d, heads):
    """Where one of a few keys has nearly all the weight: dq and dk are off by their own rounding and that of ds, two independent ones.
    One is, at the root mean square, 2^-8 / sqrt(3) of the value over its mantissa m, of which 1 / m^2 is 0.541 in the mean where values
    are spread evenly over their logarithm: 0.00166.  Few rows have most of the norm: 5 % more."""
    q, k, v, dy, cu, _ = make([700, 41], [700, 41], heads, heads // 2, d, torch.bfloat16)
    want = ob.attention(q, k, v, cu, dy=dy, window=window, sinks=sinks)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(anchor.attention(*leaves, cu.to(DEV), window=window, sinks=sinks), leaves, dy.to(DEV))
    for name, a in zip(("dq", "dk"), got):
        assert float((a.cpu().double() - want[name]).norm() / want[name].norm()) < 1.05 * 2 ** 0.5 * 2.0 ** -8 * (0.541 / 3) ** 0.5, name


@pytest.mark.gpu
def test_many_short_sequences():
    check([(7 * i) % 23 for i in range(150)], window=6, sinks=2, H=2, KV=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_window_over_everything_is_none(dtype):
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make([200, 77], [200, 77], 4, 2, 64, dtype))
    plain = anchor.attention_forward(q, k, v, cu, return_lse=True, return_low=True)
    grads = anchor.attention_backward(q, k, v, *plain[:2], dy, cu, low=plain[2])
    for window, sinks in ((200, 0), (277, 0), (2 ** 40, 2 ** 70), (100, 100), (1, 276), (1, 10 ** 9)):
        got = anchor.attention_forward(q, k, v, cu, return_lse=True, return_low=True, window=window, sinks=sinks)
        again = anchor.attention_backward(q, k, v, *got[:2], dy, cu, low=got[2], window=window, sinks=sinks)
        for a, b in zip((*plain[:2], *grads), (*got[:2], *again)):
            assert float((a.double() - b.double()).norm() / a.double().norm()) < (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,heads", [(64, 4), (128, 4), (64, 60), (128, 60), (64, 160), (128, 160)])
def test_what_a_row_does_not_see_may_be_no_number(d, heads, dtype):
    """Keys and values that lie before a row's window and behind the sinks: NaN and infinities there leave the row as it was."""
    n, window, sinks = 300, 50, 3
    q, k, v, _, cu, _ = make([n], [n], heads, heads // 2, d, dtype)
    clean = anchor.attention(*(t.to(DEV) for t in (q, k, v, cu)), window=window, sinks=sinks).cpu()
    k[100], v[100], v[20, :, 7], v[150, 0, 9] = float("nan"), float("inf"), float("-inf"), float("nan")
    got = anchor.attention(*(t.to(DEV) for t in (q, k, v, cu)), window=window, sinks=sinks).cpu()
    seen = ob.visible(window, sinks)(n, n)
    touched = seen[:, 100] | seen[:, 20] | seen[:, 150]
    f = 4 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18  # two results, each off by two roundings at most
    assert float((got[~touched].double() - clean[~touched].double()).abs().max()) <= f * float(v[torch.isfinite(v)].abs().max())
    assert torch.isfinite(got[~touched]).all()
    assert torch.isneginf(got[20:70, :, 7]).all() and torch.isnan(got[100:150]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_autograd_is_the_formula_and_padding_is_zero(dtype):
    lens = [90, 33]
    q, k, v, dy, cu, _ = make(lens, lens, 4, 2, 64, dtype)
    pad = 17
    wide = [torch.cat([t, torch.full((pad, *t.shape[1:]), 3.0, dtype=dtype)]) for t in (q, k, v, dy)]
    leaves = [t.to(DEV).requires_grad_(True) for t in wide[:3]]
    y = anchor.attention(*leaves, cu.to(DEV), window=20, sinks=2)
    got = torch.autograd.grad(y, leaves, wide[3].to(DEV))
    n = sum(lens)
    assert not y[n:].any() and not any(g[n:].any() for g in got)
    tight = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    z = anchor.attention(*tight, cu.to(DEV), window=20, sinks=2)
    assert torch.equal(z, y[:n])
    for a, b in zip(torch.autograd.grad(z, tight, dy.to(DEV)), got):
        assert float((a - b[:n]).double().norm()) <= 2.0 ** -7 * float(a.double().norm())
    uniform = anchor.attention(*(t[:90].view(2, 45, *t.shape[1:]).to(DEV) for t in (q, k, v)), window=20, sinks=2)
    both = anchor.attention(*(t[:90].to(DEV) for t in (q, k, v)), torch.tensor([0, 45, 90], device=DEV), window=20, sinks=2)
    assert torch.equal(uniform.view(90, 4, 64), both)


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32: a step of h along random directions; the loss's third derivative and its rounding bound the difference's error."""
    lens = [70, 33]
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make(lens, lens, 4, 2, 64, torch.float32))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(anchor.attention(*leaves, cu, window=9, sinks=3), leaves, dy)
    for i, g in enumerate(grads):
        u = torch.randn_like(g)
        u /= u.norm()
        loss = []
        for h in (1e-2, -1e-2):
            args = [q, k, v]
            args[i] = args[i] + h * u
            loss.append(float((anchor.attention(*args, cu, window=9, sinks=3).double() * dy.double()).sum()))
        want = float((g.double() * u.double()).sum())
        # sum of 26368 terms near 1 with relative error 2^-20 each: 2^-20 sqrt(26368) / 2h = 0.008; h^2 of a unit direction is 1e-4
        assert abs((loss[0] - loss[1]) / 2e-2 - want) < 0.02 + 1e-3 * abs(want)


@pytest.mark.gpu
def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    q, k, v, dy, cu, _ = (t.to(DEV) for t in make([700, 1300], [700, 1300], 8, 2, 128, torch.bfloat16))
    how = dict(window=200, sinks=4)

    def both():
        y, lse, low = anchor.attention_forward(q, k, v, cu, return_lse=True, return_low=True, **how)
        return (y, *anchor.attention_backward(q, k, v, y, lse, dy, cu, low=low, **how))

    want = both()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        there = both()
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(want, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a, b) for a, b in zip(want, both()))


@pytest.mark.gpu
def test_refusals():
    q, k, v, _, cu, _ = (t.to(DEV) for t in make([8], [8], 4, 2, 64, torch.bfloat16))
    for how in (dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=-1)):
        with pytest.raises(ValueError):
            anchor.attention(q, k, v, cu, **how)
    for how in (dict(window=2.5), dict(window=4, sinks=1.0)):
        with pytest.raises(TypeError):
            anchor.attention(q, k, v, cu, **how)
    with pytest.raises(RuntimeError):
        leaf = q.clone().requires_grad_(True)
        g, = torch.autograd.grad(anchor.attention(leaf, k, v, cu, window=4).float().sum(), leaf, create_graph=True)
        g.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("how", [dict(), dict(window=9, sinks=2)])
def test_gradients_of_more_rows_than_a_grid_counts(how):
    """8.4 million rows of 32 heads, sixteen to a workgroup, are past 32 bits of work-items: sequences alike have gradients alike."""
    n, seqs, H, d = 64, 2 ** 17 + 64, 32, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    one = [torch.randn(n, 1, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    k, v = (t.repeat(seqs, 1, 1) for t in one)
    q, dy = (torch.randn(1, H, d, generator=g, device=DEV).to(torch.bfloat16).expand(n * seqs, H, d) for _ in range(2))
    cu = torch.arange(seqs + 1, device=DEV) * n
    y, lse = anchor.attention_forward(q, k, v, cu, return_lse=True, **how)
    few = anchor.attention_backward(q[:8 * n], k[:8 * n], v[:8 * n], y[:8 * n], lse[:, :8 * n], dy[:8 * n], cu[:9], **how)
    got = anchor.attention_backward(q, k, v, y, lse, dy, cu, **how)
    for a, b in zip(got, few):
        part = a.view(seqs, n, *a.shape[1:])
        assert float(b.float().norm()) > 0 and bool((part[-1] == part[0]).all()) and bool((part[2 ** 16:2 ** 16 + 64] == part[:1]).all())
        assert float((part[:8].float() - b.view(8, n, *b.shape[1:]).float()).norm()) < 2.0 ** -6 * float(b.float().norm())  # roundings of bf16
