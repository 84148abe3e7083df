"""The weight that each key of a batch of prompts got (kdn_attn_weights) against the float64 definition.  A term is the exponential
of an fp32 score (d products, off by d 2^-24 of their absolute sum, at most `most`) less lse: relative 2^-24 ((d + 4) (1 + most)), and a
sum of n of them adds n 2^-24, whatever the inputs' type (they are exact in the products)."""
import pytest
import torch

from kdn import anchor
from kdn.bounded import attention_weights
from oracle import bounded as ob

DEV = "cuda:0"


def make(lens_q, lens_k, H, KV, d, dtype, window=None, sinks=0, seed=0):
    """Queries, keys, offsets, and lse of the rows as the attention before left it."""
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(sum(n), h, d, generator=g).to(dtype) for n, h in ((lens_q, H), (lens_k, KV)))
    cq, ck = (torch.tensor([0, *n]).cumsum(0) for n in (lens_q, lens_k))
    lse = ob.attention(q, k, k, cq, ck, window=window, sinks=sinks)["lse"].float()
    return q, k, lse, cq, ck


def check(lens_q, lens_k=None, H=4, KV=2, d=64, dtype=torch.bfloat16, window=None, sinks=0, add=False, seed=0):
    lens_k = lens_q if lens_k is None else lens_k
    q, k, lse, cq, ck = make(lens_q, lens_k, H, KV, d, dtype, window, sinks, seed)
    spare = max(lens_k) + 3
    w = torch.full((len(lens_k), KV, spare), 0.5, device=DEV)
    args = [t.to(DEV) for t in (q, k, lse)]
    got = attention_weights(*args, w, cq.to(DEV), None if lens_k is lens_q else ck.to(DEV), window=window, sinks=sinks, add=add)
    assert got is w
    want = ob.weights(q, k, lse, cq, ck, window=window, sinks=sinks)
    most = 40.0  # of sum |q| |k| scale, for normal values at these widths
    u = 2.0 ** -24 * ((d + 4) * (1 + most) + max([1, *lens_q]) * (H // KV) + 8)
    for b, (nq, nk) in enumerate(zip(lens_q, lens_k)):
        x = want[b]
        if add and nk > nq:
            x[:, :nk - nq] += 0.5
        row = w[b].cpu().double()
        assert torch.equal(row[:, nk:], torch.full_like(row[:, nk:], 0.5))
        assert torch.isfinite(row).all()
        assert float(((row[:, :nk] - x).abs() - u * x).max() if nk else 0) <= 2.0 ** -40, (b, float((row[:, :nk] - x).abs().max()))
    return args, w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [33, 31, 32], [63, 64, 65], [255, 256, 257], [700, 5]])
def test_lengths(lens, d, dtype):
    check(lens, d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("lens_q,lens_k", [([5], [200]), ([200], [5]), ([130, 70], [0, 70]), ([0, 40], [33, 40]), ([64], [765]), ([1, 1], [700, 1])])
def test_the_last_rows_and_pieces(lens_q, lens_k, add, dtype):
    check(lens_q, lens_k, add=add, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 3), (33, 64), (65, 100), (300, 5)])
def test_windows(window, sinks, d, dtype):
    check([900, 1, 129], d=d, dtype=dtype, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV", [(1, 1), (6, 2), (8, 1), (16, 4)])
def test_head_groups(H, KV):
    check([70, 341], H=H, KV=KV)


@pytest.mark.gpu
def test_many_sequences():
    check([(7 * i) % 23 for i in range(150)], H=2, KV=1)


@pytest.mark.gpu
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,H,KV,d", [(9, 8, 4, 64), (120, 8, 4, 64), (1, 4, 4, 128), (400, 16, 4, 128)])
def test_few_rows_over_many_keys(rows, H, KV, d, add):
    """Rows that stay in LDS while the keys pass: sequences of many and of no rows and keys, more rows than LDS holds among them."""
    lens_k = [(37 * i) % 400 for i in range(66)] + [3000]
    check([min(rows * (i % 3) // 2, n + 5) if i != 40 else rows for i, n in enumerate(lens_k)], lens_k, H=H, KV=KV, d=d, add=add)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128)])
@pytest.mark.parametrize("lens_q,lens_k,window,sinks", [([2600], [2600], 100, 5), ([2100, 20, 1900], [2100, 20, 1900], 33, 300), ([1500], [1700], 1, 1),
                                                       ([1500], [1300], 70, 257), ([0, 3000, 0], [50, 2999, 0], 64, 64)])
def test_rows_far_behind_the_sinks(lens_q, lens_k, window, sinks, dtype, d):
    check(lens_q, lens_k, d=d, dtype=dtype, window=window, sinks=sinks, add=sinks == 1)


@pytest.mark.gpu
def test_one_workgroup_to_a_tile_of_keys():
    """So many keys that no two workgroups share a tile's rows."""
    check([40, 30], [9000, 8000], H=32, KV=32, d=64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_with_the_attention_before_it(dtype):
    """lse as the kernel gives it: every row's weights sum to one, so that all of them sum to the rows that see a key."""
    lens, H, KV = [300, 77], 8, 2
    q, k, _, cu, _ = make(lens, lens, H, KV, 64, dtype)
    q, k, cu = q.to(DEV), k.to(DEV), cu.to(DEV)
    for how in (dict(), dict(window=50, sinks=3)):
        _, lse = anchor.attention_forward(q, k, k, cu, return_lse=True, **how)
        w = torch.empty(2, KV, 300, device=DEV)
        attention_weights(q, k, lse, w, cu, **how)
        for b, n in enumerate(lens):
            total = w[b, :, :n].double().sum(-1)
            assert float((total - n * (H // KV)).abs().max()) <= 2.0 ** -24 * (68 * 41 * 2 + n * 4) * n * (H // KV)


@pytest.mark.gpu
def test_slots_places_strides_and_padding():
    lens, KV = [90, 40, 300], 2
    q, k, lse, cq, _ = make(lens, lens, 4, KV, 64, torch.bfloat16)
    _, want = check(lens)
    pad = torch.full((7, 4, 64), 3.0, dtype=torch.bfloat16)
    fused = torch.cat([torch.cat([q, k], 1), torch.cat([pad, pad[:, :KV]], 1)]).to(DEV)
    wide = torch.cat([lse, torch.zeros(4, 7)], 1).to(DEV)
    table = torch.zeros(5, 3, KV, 120, device=DEV)
    attention_weights(fused[:, :4], fused[:, 4:], wide, table[:, 1], cq.to(DEV), slots=torch.tensor([3, 9, 0], device=DEV))
    assert torch.equal(table[3, 1, :, :90], want[0, :, :90]) and torch.equal(table[0, 1], want[2, :, :120])
    rest = table.clone()
    rest[3, 1, :, :90], rest[0, 1] = 0, 0
    assert not rest.any()


@pytest.mark.gpu
def test_what_a_row_does_not_see_may_be_no_number():
    q, k, lse, cq, ck = make([100], [300], 4, 2, 64, torch.bfloat16)
    k[200 + 60:] = float("nan")  # the first 60 rows see the keys before it
    lse[:, 60:] = 0
    w = torch.zeros(1, 2, 300, device=DEV)
    q[60:] = 0
    attention_weights(*(t.to(DEV) for t in (q, k, lse)), w, cq.to(DEV), ck.to(DEV))
    assert torch.isfinite(w[..., :260]).all() and torch.isnan(w[..., 260:]).all()


@pytest.mark.gpu
def test_the_same_bits_on_another_stream_and_in_a_graph():
    (q, k, lse), w = check([500, 40], [700, 1300], H=8, KV=2, d=128)
    cq, ck = (torch.tensor([0, *n], device=DEV).cumsum(0) for n in ([500, 40], [700, 1300]))
    other, there = torch.cuda.Stream(), torch.full_like(w, 0.5)
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        attention_weights(q, k, lse, there, cq, ck)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(w, there)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention_weights(q, k, lse, there, cq, ck)
    for _ in range(3):
        there.fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, there)


@pytest.mark.gpu
def test_refusals():
    q, k, lse, cq, ck = (t.to(DEV) for t in make([8], [8], 4, 2, 64, torch.bfloat16))
    w = torch.zeros(1, 2, 8, device=DEV)
    ok = dict(q=q, k=k, lse=lse, weights=w, cu_seqlens=cq)
    for bad in (dict(lse=lse[:2]), dict(lse=lse.double()), dict(weights=w[:, :1]), dict(weights=w.double()), dict(weights=w.expand(3, 2, 8)),
                dict(k=k[:5]), dict(k=k.float()), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(cu_seqlens_k=ck[:1]),
                dict(q=q.clone().requires_grad_(True)), dict(slots=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(weights=w.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            attention_weights(**{**ok, **bad})
    assert not w.any()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("add", [False, True])
def test_long_pieces_among_single_rows(d, add):
    """A few sequences with far more rows than the others, one of them behind the 64th, one without keys and one that is the last."""
    lens_k = [(91 * i) % 500 + 60 for i in range(80)]
    lens_q = [min(1, n) for n in lens_k]
    for b, rows, keys in ((3, 400, 520), (9, 300, 0), (70, 700, 700), (79, 130, 900)):
        lens_q[b], lens_k[b] = rows, keys
    check(lens_q, lens_k, H=32 if d == 128 else 64, KV=32, d=d, add=add)


@pytest.mark.gpu
def test_long_pieces_are_walked_by_many_workgroups():
    """One piece of a prompt among decoding streams: in one call at most four times as long as the two kinds in calls of their own
    (when its keys' tiles were the stretch of two workgroups a head, thirteen times)."""
    H, KV, d, keys, rows, streams = 32, 8, 128, 4096, 4096, 63
    g = torch.Generator(device=DEV).manual_seed(0)
    make_bf16 = lambda n, h: torch.randn(n, h, d, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731

    def took(lens_q):
        q, k = make_bf16(sum(lens_q), H), make_bf16(keys * len(lens_q), KV)
        lse = torch.full((H, sum(lens_q)), 9.0, device=DEV)
        cq, ck = (torch.tensor([0, *n], device=DEV).cumsum(0) for n in (lens_q, [keys] * len(lens_q)))
        w = torch.zeros(len(lens_q), KV, keys, device=DEV)
        times = []
        for _ in range(6):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            attention_weights(q, k, lse, w, cq, ck, add=True)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert took([1] * 20 + [rows] + [1] * (streams - 20)) < 4 * (took([1] * streams) + took([rows]))
