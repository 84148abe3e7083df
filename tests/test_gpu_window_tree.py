"""Attention of new tokens over pages under a window with sinks, and the weights that the keys got (kdn_tree_attn_bounded) against
the float64 definition.  y's tolerances are those of the attention over pages without a window: twice bf16's rounding unit of
sum p |v|, or fp32's sums.  A weight is a sum of exponentials of fp32 scores (d products, off by d 2^-24 of their absolute
sum, at most 40) over lse: relative 2^-24 (d + 4) 41 and the sum's own, whatever the inputs' type."""
import pytest
import torch

from kdn import anchor
from oracle import bounded as ob

DEV = "cuda:0"


def make(lens, new, H, KV, d, P, dtype, seed=0, poison=True):
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype) for h in (H, KV, KV))
    counts = [-(-x // P) for x in lens]
    total = max(1, sum(counts)) + 2
    kp, vp = (torch.randn(total, KV, P, d, generator=g).to(dtype) for _ in range(2))
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max([1, *counts])), -7, dtype=torch.int32)
    used = 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(order[used:used + c], dtype=torch.int32)
        used += c
        if poison and c and lens[b] % P:  # what lies behind a stream's last token may be anything
            kp[order[used - 1], :, lens[b] % P:] = float("nan")
            vp[order[used - 1], :, lens[b] % P:] = float("inf")
    parents = torch.tensor([int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for m in new for i in range(m)], dtype=torch.int32)
    return q, k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32), torch.tensor([0, *new]).cumsum(0), parents


def check(lens, new, H=8, KV=2, d=64, P=16, dtype=torch.bfloat16, tree=False, weights=False, window=None, sinks=0, seed=0, **kw):
    args = make(lens, new, H, KV, d, P, dtype, seed)
    *dev, parents = (t.to(DEV) for t in args)
    how = dict(window=window, sinks=sinks)
    spare = max(lens) + max(new) + 3
    w = torch.full((len(lens), KV, spare), 0.25, device=DEV) if weights else None
    if weights:
        kw["max_new"] = max(new)
    y = anchor.tree_attention(*dev, parents=parents if tree else None, weights=w, **how, **kw)
    want, bound, got_w = ob.tree_attention(*args[:8], args[8] if tree else None, **how)
    most = 40.0  # of sum |q| |k| scale, for normal values at these widths
    f = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * ((d + 4) * (1 + most) + max(lens) + 72)
    got = y.cpu().double()
    assert torch.isfinite(got).all()
    slack = f * (bound + want.abs()) + 2.0 ** -18 * bound
    assert float(((got - want).abs() - slack).max()) <= 0, float(((got - want).abs() / slack).max())
    if weights:
        u = 2.0 ** -24 * ((d + 4) * (1 + most) + 40)
        for b, (L, n) in enumerate(zip(lens, new)):
            ww = got_w[b]
            ww[:, :L] += 0.25
            if n == 0:
                ww[:] = 0.25
            row = w[b].cpu().double()
            assert torch.equal(row[:, L + n:], torch.full_like(row[:, L + n:], 0.25))
            assert float(((row[:, :L + n] - ww).abs() - u * (1 + ww)).max() if L + n else 0) <= 0
    return dev, parents, y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (2, 0), (16, 16), (33, 4), (64, 40), (200, 0), (129, 300)])
def test_single_tokens(window, sinks, d, dtype):
    check([0, 1, 17, 31, 32, 33, 200, 201, 700], [1] * 9, d=d, dtype=dtype, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [[2, 8], [1, 0, 5], [33, 7], [64, 1], [20, 64, 32]])
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (40, 42), (70, 4), (150, 64)])
def test_trees_and_runs(new, tree, window, sinks, dtype):
    check([40, 300, 0][:len(new)], new, dtype=dtype, tree=tree, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,KV,new", [(4, 4, 1), (16, 1, 3), (33, 1, 2), (8, 1, 64)])
def test_head_groups_and_pages(H, KV, new, d):
    for P in (16, 64):
        check([520, 77], [new, max(1, new - 1)], H=H, KV=KV, d=d, P=P, window=100, sinks=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 20])
def test_many_chunks_and_bounds_from_the_host(new, dtype):
    """A window over several chunks, contexts that are longer than it and not; a wide bound and a workspace of the caller's."""
    lens = [5000, 2100, 900, 3]
    dev, parents, y = check(lens, [new] * 4, tree=True, dtype=dtype, window=2000, sinks=70)
    held = torch.empty(anchor.tree_workspace_bytes(4, 8, 2, 64, dtype, 16, 5008, 64, window=2000, sinks=70), dtype=torch.uint8, device=DEV)
    again = anchor.tree_attention(*dev, parents=parents, max_new=64, workspace=held, window=2000, sinks=70)
    assert float((again.double() - y.double()).norm() / y.double().norm()) < (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18)
    assert held.nbytes < anchor.tree_workspace_bytes(4, 8, 2, 64, dtype, 16, 5008, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 12])
def test_a_window_over_everything_is_none(new):
    dev, parents, y = check([500, 33], [new] * 2, tree=True, max_new=new, max_context=500)
    for how in (dict(window=512 + 12), dict(window=2 ** 50, sinks=2 ** 70), dict(window=3, sinks=600)):
        assert torch.equal(anchor.tree_attention(*dev, parents=parents, max_new=new, max_context=500, **how), y)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 9, 40])
def test_what_no_token_sees_may_be_no_number(new):
    """Keys before the window and behind the sinks, those of their tiles among them."""
    lens, window, sinks, P = [400, 203], 70, 5, 16
    args = make(lens, [new] * 2, 8, 2, 64, P, torch.bfloat16)
    want, bound, _ = ob.tree_attention(*args[:8], window=window, sinks=sinks)
    for b, L in enumerate(lens):
        for j in range(sinks, L - window + 1):
            page, at = int(args[5][b, j // P]), j % P
            args[3][page, :, at], args[4][page, :, at] = float("nan"), float("inf")
    got = anchor.tree_attention(*(t.to(DEV) for t in args[:8]), window=window, sinks=sinks).cpu().double()
    slack = 2 * 2.0 ** -8 * (bound + want.abs()) + 2.0 ** -18 * bound
    assert float(((got - want).abs() - slack).max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("how", [dict(), dict(window=60, sinks=3)])
def test_weights_of_tokens(how, d, dtype):
    check([0, 1, 31, 32, 33, 255, 1300], [1] * 7, d=d, dtype=dtype, weights=True, **how)
    check([40, 700, 0, 129], [3, 0, 8, 1], H=8, KV=2, d=d, dtype=dtype, weights=True, **how)
    check([300, 10], [32, 5], H=2, KV=2, d=d, dtype=dtype, weights=True, **how)


@pytest.mark.gpu
def test_weights_over_many_chunks_and_slots():
    """Streams in rows of a larger table, some in none; strides; a row that is too short."""
    lens, H, KV = [5000, 2100, 700, 33], 32, 4
    args = make(lens, [1] * 4, H, KV, 64, 32, torch.bfloat16)
    dev = [t.to(DEV) for t in args[:8]]
    _, _, want = ob.tree_attention(*args[:8])
    table = torch.zeros(6, 3, KV, 5001, device=DEV)
    slots = torch.tensor([4, -1, 0, 6], dtype=torch.int32, device=DEV)
    y = anchor.tree_attention(*dev, weights=table[:, 1], slots=slots, max_new=1)
    assert torch.equal(y, anchor.tree_attention(*dev, weights=torch.zeros(4, KV, 5100, device=DEV), max_new=1))
    u = 2.0 ** -24 * (68 * 41 + 40)
    for b, row in ((0, 4), (2, 0)):
        assert float(((table[row, 1, :, :lens[b] + 1].cpu().double() - want[b]).abs() - u * want[b]).max()) <= 2.0 ** -40
    rest = table.clone()
    rest[4, 1], rest[0, 1] = 0, 0
    assert not rest.any() and not table[0, 1, :, 701:].any()
    short = torch.zeros(4, KV, 600, device=DEV)
    anchor.tree_attention(*dev, weights=short, max_new=1)
    assert float(((short[0].cpu().double() - want[0][:, :600]).abs() - u * want[0][:, :600]).max()) <= 2.0 ** -40


@pytest.mark.gpu
def test_weights_add_up_over_steps_in_a_graph_and_on_another_stream():
    lens = [300, 45]
    dev = [t.to(DEV) for t in make(lens, [1, 1], 8, 2, 128, 16, torch.bfloat16)[:8]]
    once = torch.zeros(2, 2, 320, device=DEV)
    y = anchor.tree_attention(*dev, weights=once, window=200, sinks=4, max_context=300, max_new=1)
    other, w = torch.cuda.Stream(), torch.zeros_like(once)
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        z = anchor.tree_attention(*dev, weights=w, window=200, sinks=4, max_context=300, max_new=1)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(y, z) and torch.equal(w, once)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = anchor.tree_attention(*dev, weights=w, window=200, sinks=4, max_context=300, max_new=1)
    for steps in range(2, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, z)
        for b, L in enumerate(lens):
            assert torch.equal(w[b, :, L:], once[b, :, L:])  # the new token's is set
            assert torch.allclose(w[b, :, :L], steps * once[b, :, :L], rtol=2.0 ** -21, atol=0)


@pytest.mark.gpu
def test_padded_rows_are_zeros_and_streams_without_tokens_keep_their_weights():
    args = make([50, 20, 300], [1, 0, 2], 8, 2, 64, 16, torch.bfloat16)
    q, k, v = (torch.cat([t[:1], t, t[:3]]) for t in args[:3])
    cu = args[7] + 1
    w = torch.full((3, 2, 400), 0.5, device=DEV)
    y = anchor.tree_attention(*(t.to(DEV) for t in (q, k, v, *args[3:7], cu)), weights=w, max_new=2, out=torch.full_like(q, 9.0).to(DEV))
    assert not y[:1].any() and not y[4:].any() and y[1:4].any()
    assert bool((w[1] == 0.5).all())


@pytest.mark.gpu
def test_refusals():
    *dev, parents = (t.to(DEV) for t in make([40], [2], 8, 2, 64, 16, torch.bfloat16))
    w = torch.zeros(1, 2, 64, device=DEV)
    for bad in (dict(window=0), dict(window=4, sinks=-1), dict(weights=w, parents=parents), dict(weights=w.double()), dict(weights=w[:, :1]),
                dict(weights=w.cpu()), dict(weights=w.expand(2, 2, 64)), dict(weights=w.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(weights=w.clone().requires_grad_(True)), dict(weights=w[:, :1].expand(1, 2, 64), max_new=2), dict(weights=w, slots=torch.zeros(2, dtype=torch.int32, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            anchor.tree_attention(*dev, **bad)
    with pytest.raises(RuntimeError):  # 64 new tokens of 4 heads are more than 32 rows
        anchor.tree_attention(*dev, weights=w, max_new=64)
    assert not w.any()
    before = w._version
    anchor.tree_attention(*dev, weights=w, max_new=2)
    assert w._version > before


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 8])
@pytest.mark.parametrize("window,sinks", [(2000, 70), (1200, 900), (130, 2000)])
def test_weights_in_a_window_over_many_chunks(window, sinks, new, d, dtype):
    """Contexts longer than the window and not; where the window's keys follow the sinks', inside the first chunk and inside later ones."""
    check([5000, 2100, 900, 3], [new, max(1, new - 3), new, 1], d=d, dtype=dtype, weights=True, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("streams,KV,window", [(70, 8, 900), (100, 8, 900), (97, 8, 5000)])
def test_large_batches_in_a_window(streams, KV, window, dtype):
    """More workgroups than run at a time, in one chunk a context and in several; with weights, and a token more for some streams."""
    g = torch.Generator().manual_seed(streams)
    lens = torch.randint(0, 2 * window, (streams,), generator=g).tolist()
    lens[3] = 2 * window
    for weights in (False, True):
        check(lens, [1 + (b % 5 == 0) for b in range(streams)], H=KV, KV=KV, dtype=dtype, weights=weights, window=window, sinks=4)


@pytest.mark.gpu
def test_a_stream_more_than_the_gpu_has_room_for_is_no_second_round():
    """65 streams of eight key heads, a window of 16000, at most a quarter longer than 64, whose workgroups run all at once (in chunks of a
    whole window half as long again)."""
    H, KV, d, P, window = 32, 8, 128, 64, 16000

    def took(streams):
        each = -(-(window + 2000) // P)
        kp, vp = (torch.zeros(streams * each, KV, P, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        table = torch.arange(streams * each, dtype=torch.int32, device=DEV).view(streams, each)
        q, k = (torch.ones(streams, h, d, dtype=torch.bfloat16, device=DEV) for h in (H, KV))
        lens = torch.full((streams,), window + 2000, dtype=torch.int32, device=DEV)
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            anchor.tree_attention(q, k, k, kp, vp, table, lens, max_context=window + 2000, window=window, sinks=4)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert took(65) < 1.25 * took(64)
