"""Eviction from the pages by weight (kdn_evict) against the definition: whole numbers and moved bits, equal to the last one."""
import pytest
import torch

from kdn.bounded import evict
from oracle import bounded as ob

DEV = "cuda:0"


def make(lens, layers=1, KV=2, d=64, P=16, dtype=torch.bfloat16, seed=0, zeros=0.1):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // P) for n in lens]
    pages = sum(counts) + 2
    slab = torch.randn(pages, layers, 2, KV, P, d, generator=g).to(dtype)
    order, used = torch.randperm(pages, generator=g).tolist(), 0
    table = torch.full((len(lens), max([1, *counts])), -9, dtype=torch.int32)
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(order[used:used + c], dtype=torch.int32)
        used += c
    room = max(lens) + 5
    w = torch.exp(2 * torch.randn(len(lens), layers, KV, room, generator=g))
    w[torch.rand(w.shape, generator=g) < zeros] = 0
    w[torch.rand(w.shape, generator=g) < 0.1] = 1.0  # equals
    return slab, table, w, g


def places(slab, table, b, n, P):
    """(layers, 2, KV, n, d): a stream's first n places."""
    pages = table[b, :-(-n // P)].long()
    x = slab[pages].permute(1, 2, 3, 0, 4, 5)
    return x.reshape(*x.shape[:3], -1, x.shape[-1])[..., :n, :]


def check(lens, keep, settled=None, evicted=None, sinks=0, recent=0, slots=None, w=None, max_len=None, **kw):
    P, layers, KV = kw.get("P", 16), kw.get("layers", 1), kw.get("KV", 2)
    slab, table, weights, g = make(lens, **kw)
    if w is not None:
        weights = w(weights)
    B, room = len(lens), weights.shape[-1]
    gone = [0] * B if evicted is None else evicted
    pos = torch.randint(0, 1000, weights.shape, generator=g).to(torch.int32)
    for b in range(B):  # distinct positions of the settled places
        n = settled[b] if settled else 0
        if n:
            pos[b, ..., :n] = torch.rand(layers, KV, n + gone[b], generator=g).argsort(-1)[..., :n].to(torch.int32)
    rows = list(range(B)) if slots is None else slots
    table_w = torch.full((max(rows) + 2, layers, KV, room), 7.0)
    table_p = torch.full((max(rows) + 2, layers, KV, room), 7, dtype=torch.int32)
    for b, r in enumerate(rows):
        if r >= 0:
            table_w[r], table_p[r] = weights[b], pos[b]
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    dev = [t.to(DEV) for t in (slab, table_w, table_p)]
    if layers == 1:  # a single layer's views
        views = dev[0][:, 0, 0], dev[0][:, 0, 1], dev[1][:, 0], dev[2][:, 0]
    else:
        views = dev[0][:, :, 0], dev[0][:, :, 1], dev[1], dev[2]
    evict(*views[:2], table.to(DEV), ints(lens), ints(keep), *views[2:], ints(settled), ints(evicted), sinks=sinks, recent=recent,
          slots=ints(rows), max_len=max_len)
    got = [t.cpu() for t in dev]
    want = [slab.clone(), table_w.clone(), table_p.clone()]
    for b, r in enumerate(rows):
        if r < 0:
            continue
        for layer in range(layers):
            for e in range(KV):
                moves, ww, pp = ob.evict(weights[b, layer, e].tolist(), pos[b, layer, e].tolist(), lens[b], keep[b], settled[b] if settled else 0,
                                         gone[b], sinks, recent)
                want[1][r, layer, e] = torch.tensor(ww)
                want[2][r, layer, e] = torch.tensor(pp, dtype=torch.int32)
                for src, dst in moves:
                    want[0][table[b, dst // P], layer, :, e, dst % P] = slab[table[b, src // P], layer, :, e, src % P]
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))  # the bits: NaNs among them


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128)])
@pytest.mark.parametrize("lens,keep", [([1, 2, 0], [1, 1, 5]), ([17, 64, 65, 200], [16, 1, 64, 100]), ([1025, 1024, 1023], [1024, 1000, 0])])
def test_lengths(lens, keep, dtype, d):
    check(lens, keep, dtype=dtype, d=d)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 32, 256])
@pytest.mark.parametrize("layers,KV", [(3, 2), (1, 5), (2, 1)])
def test_layers_heads_and_pages(layers, KV, P):
    check([300, 90], [120, 89], layers=layers, KV=KV, P=P)


@pytest.mark.gpu
@pytest.mark.parametrize("sinks,recent", [(4, 0), (0, 30), (4, 30), (300, 5), (5, 2 ** 40), (2 ** 63, 0), (200, 200)])
def test_what_is_held(sinks, recent):
    """More than are kept, too: then the sinks stay first, the lowest places of them."""
    check([300, 90, 40], [120, 60, 39], sinks=sinks, recent=recent)
    check([300, 90, 40], [120, 60, 39], [100, 90, 7], [1000, 3, 0], sinks=sinks, recent=recent)


@pytest.mark.gpu
def test_cut_again():
    """Streams cut before, their places' positions in any order; more settled than are kept, and nothing to cut."""
    check([300, 300, 50], [200, 100, 60], [150, 250, 20], [40, 100000, 9], sinks=4, recent=16)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16384, 16385, 40001])
def test_long_caches(n):
    """Within the ranks that LDS holds, one more, and far more."""
    check([n], [n // 3], KV=1, sinks=4, recent=100)
    check([n, 77], [n - 1, 70], KV=1, zeros=0.9)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0.0, 1.0, float("nan"), -1.0, float("inf")])
def test_equal_weights_and_no_numbers(fill):
    """All alike: the lowest places stay; infinities above all numbers, NaN and negative ones as zeros."""
    check([2000, 70], [700, 69], w=lambda w: torch.full_like(w, fill))

    def some(w):
        w[..., ::3] = fill
        return w

    check([2000, 70], [700, 69], w=some)


@pytest.mark.gpu
def test_neighbouring_floats():
    """Ranks that differ in their last bits alone, and the smallest numbers."""
    check([500, 300], [100, 299], w=lambda w: (1.0 + torch.randint(0, 40, w.shape) * 2.0 ** -23))
    check([500, 300], [100, 299], w=lambda w: torch.randint(0, 40, w.shape) * 2.0 ** -149)


@pytest.mark.gpu
def test_slots():
    check([100, 200, 50], [60, 100, 20], slots=[4, -1, 0])


@pytest.mark.gpu
def test_the_same_slot_twice_stays_inside():
    """Not allowed, and harmless: other tensors are as they were."""
    slab, table, w, _ = make([300, 300])
    w[0, 0] = torch.arange(305.)
    guard = torch.full((3, 2, 305), 5.0, device=DEV)
    guard[1] = w[0, 0].to(DEV)
    pos = torch.zeros(3, 2, 305, dtype=torch.int32, device=DEV)
    dev = slab.to(DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    evict(dev[:, 0, 0], dev[:, 0, 1], table.to(DEV), ints(300, 300), ints(100, 150), guard, pos, slots=ints(1, 1))
    assert bool((guard[0] == 5).all()) and bool((guard[2] == 5).all()) and not pos[0].any() and not pos[2].any()


@pytest.mark.gpu
def test_lengths_and_pages_out_of_range():
    """Lengths past the bound are cut to it; page numbers outside the pool are their nearest page's."""
    slab, table, w, _ = make([300, 90])
    pos = torch.zeros(w[:, 0].shape, dtype=torch.int32, device=DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table[0, 3] = 2 ** 30
    for max_len in (None, 64):
        evict(*(slab.to(DEV)[:, 0, i] for i in (0, 1)), table.to(DEV), ints(2 ** 31 - 1, -5), ints(50, -7), w[:, 0].to(DEV), pos,
              ints(-3, 2 ** 31 - 1), ints(-1, 7), max_len=max_len)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    lens, keep = [1300, 700], [600, 600]
    slab, table, w, _ = make(lens, layers=2, d=128)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    first = [t.to(DEV) for t in (slab, w, torch.zeros(w.shape, dtype=torch.int32))]

    def cut(state):
        evict(state[0][:, :, 0], state[0][:, :, 1], tab, L, K, *state[1:], sinks=4, recent=64, max_len=1300)

    tab, L, K = table.to(DEV), ints(lens), ints(keep)
    want = [t.clone() for t in first]
    cut(want)
    there = [t.clone() for t in first]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        cut(there)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(want, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cut(there)
    for _ in range(3):
        for a, b in zip(there, first):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, there))


@pytest.mark.gpu
def test_refusals():
    slab, table, w, _ = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in make([40, 30], layers=2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    pos = torch.zeros(w.shape, dtype=torch.int32, device=DEV)
    ok = dict(k_pages=slab[:, :, 0], v_pages=slab[:, :, 1], page_table=table, lens=ints(40, 30), keep=ints(20, 20), weights=w, positions=pos)
    before = slab.clone()
    for bad in (dict(v_pages=slab[:, :1, 1]), dict(v_pages=slab[:, :, 1].float()), dict(page_table=table.long()), dict(lens=ints(40)),
                dict(keep=ints(1, 2, 3)), dict(weights=w[:, :1]), dict(weights=w.double()), dict(positions=pos.long()), dict(positions=pos[..., :9]),
                dict(sinks=-1), dict(recent=-1), dict(max_len=-1), dict(weights=w[:1], positions=pos[:1]), dict(k_pages=slab[:, 0, 0]),
                dict(k_pages=slab[:, :, 0].transpose(3, 4)), dict(weights=w.clone().requires_grad_(True)), dict(settled=ints(1)),
                dict(k_pages=slab[:, :, 0, :, :, 1:], v_pages=slab[:, :, 1, :, :, 1:]), dict(lens=torch.tensor([40, 30]))):
        with pytest.raises((ValueError, RuntimeError)):
            evict(**{**ok, **bad})
    assert torch.equal(slab, before)


@pytest.mark.gpu
def test_rows_that_lie_on_one_another_are_refused():
    """Expanded pages: a move into one would be a move into several, in no order."""
    slab, table, w, _ = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in make([40, 30], layers=2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    pos = torch.zeros(w.shape, dtype=torch.int32, device=DEV)
    k, v = slab[:, :, 0], slab[:, :, 1]
    before = slab.clone()
    for one in (k[:1], k[:, :1], k[:, :, :1], k[:, :, :, :1]):
        for pages in ((one.expand(k.shape), v), (v, one.expand(k.shape))):
            with pytest.raises(ValueError, match="lie on one another"):
                evict(*pages, table, ints(40, 30), ints(20, 20), w, pos)
    with pytest.raises(ValueError, match="lie on one another"):
        evict(k[:, 0, :1].expand(k[:, 0].shape), v[:, 0], table, ints(40, 30), ints(20, 20), w[:, 0], pos[:, 0])
    assert torch.equal(slab, before) and not pos.any()
    one = slab[:, :1, 0], slab[:, :1, 1]  # a single entry's stride may be any
    evict(*(t.as_strided(t.shape, (t.stride(0), 0, *t.stride()[2:]), t.storage_offset()) for t in one), table, ints(40, 30), ints(20, 20), w[:, :1], pos[:, :1])


@pytest.mark.gpu
def test_more_moves_than_one_grid_counts():
    """65 streams, 32 layers, eight heads, room for 32768 places: 17 million workgroups, whose work-items are past 32 bits; the places that
    there are, 40 of each head, are few."""
    streams, layers, KV, d, P, L, keep, room = 65, 32, 8, 128, 16, 40, 20, 32768
    slab = torch.randn(3 * streams, layers, 2, KV, P, d, device=DEV).to(torch.bfloat16)
    table = torch.zeros(streams, room // P, dtype=torch.int32, device=DEV)
    table[:, :3] = torch.arange(3 * streams, device=DEV).view(streams, 3)
    w = torch.zeros(streams, layers, KV, room, device=DEV)
    w[..., :L] = torch.arange(L, device=DEV) + 1.0  # the latest stay
    pos = torch.zeros(w.shape, dtype=torch.int32, device=DEV)
    rows = lambda: slab[table[:, :3].long()].permute(0, 2, 3, 4, 1, 5, 6).reshape(streams, layers, 2, KV, 3 * P, d)  # noqa: E731
    before = rows().clone()
    ints = lambda x: torch.full((streams,), x, dtype=torch.int32, device=DEV)  # noqa: E731
    evict(slab[:, :, 0], slab[:, :, 1], table, ints(L), ints(keep), w, pos, max_len=room)
    assert torch.equal(rows()[..., :keep, :], before[..., L - keep:L, :])
    assert bool((w[..., :keep] == w[0, 0, 0, L - keep:L]).all()) and bool((pos[..., :keep] == torch.arange(L - keep, L, device=DEV)).all())
