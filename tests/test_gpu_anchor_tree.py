"""Attention of new tokens over pages (kdn_tree_attn) against the float64 definition; tolerances as for the prompts'
attention: twice bf16's rounding unit of sum p |v| (weights and output), or fp32's sums."""
import pytest
import torch

from kdn import anchor
from oracle import anchor as oa

DEV = "cuda:0"


def make(lens, new, H, KV, d, P, dtype, seed=0, spare=0, poison=True):
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype) for h in (H, KV, KV))
    counts = [-(-x // P) for x in lens]
    total = max(1, sum(counts)) + 2
    kp, vp = (torch.randn(total, KV, P, d, generator=g).to(dtype) for _ in range(2))
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max([1, *counts]) + spare), -7, dtype=torch.int32)
    used = 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(order[used:used + c], dtype=torch.int32)
        used += c
        if poison and c and lens[b] % P:  # what lies behind a stream's last token may be anything
            kp[order[used - 1], :, lens[b] % P:] = float("nan")
            vp[order[used - 1], :, lens[b] % P:] = float("inf")
    parents = torch.tensor([int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for m in new for i in range(m)], dtype=torch.int32)
    cu = torch.tensor([0, *new]).cumsum(0)
    return q, k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32), cu, parents


def check(lens, new, H=8, KV=2, d=64, P=16, dtype=torch.bfloat16, tree=True, seed=0, spare=0, **kw):
    args = make(lens, new, H, KV, d, P, dtype, seed, spare)
    *dev, parents = (t.to(DEV) for t in args)
    y = anchor.tree_attention(*dev, parents=parents if tree else None, **kw)
    want, bound = oa.tree_attention(*args[:8], args[8] if tree else None, kw.get("scale"))
    most = 40.0  # of sum |q| |k| scale, for normal values at these widths
    f = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * ((d + 4) * (1 + most) + max(lens) + 72)
    got = y.cpu().double()
    assert torch.isfinite(got).all()
    slack = f * (bound + want.abs()) + 2.0 ** -18 * bound
    assert float(((got - want).abs() - slack).max()) <= 0, float(((got - want).abs() / slack).max())
    return dev, parents, y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[0], [1, 15, 16, 17], [31, 32, 33], [255, 256, 257, 0], [1300, 3]])
def test_single_tokens(lens, d, dtype):
    check(lens, [1] * len(lens), d=d, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [[2, 8], [1, 0, 5], [33, 7], [64, 1], [20, 64, 32]])
@pytest.mark.parametrize("tree", [True, False])
def test_trees_and_runs(new, tree, dtype):
    check([40, 300, 0][:len(new)], new, dtype=dtype, tree=tree)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,KV,new", [(4, 4, 1), (4, 4, 40), (16, 1, 1), (16, 1, 3), (32, 1, 1), (33, 1, 2), (8, 1, 64), (64, 1, 64)])
def test_head_groups(H, KV, new, d):
    check([520, 77], [new, max(1, new - 1)], H=H, KV=KV, d=d)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 32, 64, 256])
def test_page_sizes(P):
    check([300, 5, 1024], [1, 3, 1], P=P, spare=3)
    check([300, 5, 1024], [17, 3, 40], P=P, spare=3)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20])
def test_bounds_from_the_host(new):
    """The chunks of a wider table, of tight bounds, and of a workspace that the caller holds: the same up to their sums' order."""
    lens = [2000, 700, 1]
    dev, parents, y = check(lens, [new] * 3, max_context=2000, max_new=new)
    wide = torch.cat([dev[5], torch.full((3, 2000), 2 ** 30, dtype=torch.int32, device=DEV)], dim=1)  # never read: past the contexts
    check_same = anchor.tree_attention(*dev[:5], wide, *dev[6:], parents=parents, max_new=64)
    assert float((check_same.double() - y.double()).norm() / y.double().norm()) < 2.0 ** -8
    n = anchor.tree_workspace_bytes(5, 8, 2, 64, torch.bfloat16, 16, 4096, new)
    held = torch.empty(n, dtype=torch.uint8, device=DEV)
    again = anchor.tree_attention(*dev, parents=parents, max_context=2000, max_new=new, workspace=held)
    assert torch.equal(again, y)


@pytest.mark.gpu
def test_many_streams_use_one_launch_size():
    check([(37 * i) % 211 for i in range(130)], [1 + i % 3 for i in range(130)], H=4, KV=2)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 7])
def test_longest_chunks(new):
    """Streams enough for chunks of 2048 keys, one of them with three: one token, and 7 (56 rows to a key head)."""
    check([4100, 2049, 2048] + [3] * 297, [new] * 300, H=16, KV=2, P=256)


@pytest.mark.gpu
def test_pages_in_other_layouts():
    lens, new = [100, 37], [1, 4]
    q, k, v, kp, vp, table, ctx, cu, par = (t.to(DEV) for t in make(lens, new, 8, 2, 64, 16, torch.bfloat16))
    y = anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, parents=par)
    both = torch.stack([kp, vp], dim=1)  # one slab, keys and values of a page together
    assert torch.equal(anchor.tree_attention(q, k, v, both[:, 0], both[:, 1], table, ctx, cu, parents=par), y)
    tok = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]  # tokens before heads
    assert torch.equal(anchor.tree_attention(q, k, v, *tok, table, ctx.long(), cu.int(), parents=par.long()), y)
    fused = torch.cat([q, k, v], dim=1).split([8, 2, 2], dim=1)
    assert torch.equal(anchor.tree_attention(*fused, kp, vp, table, ctx, cu, parents=par), y)


@pytest.mark.gpu
def test_bad_parents_and_page_numbers_stay_inside():
    """A parent that is no earlier token hangs its token on the context; a page number outside the pool reads some page."""
    lens, new = [40], [5]
    args = make(lens, new, 8, 2, 64, 16, torch.bfloat16, poison=False)
    dev = [t.to(DEV) for t in args]
    good = torch.tensor([-1, 0, -1, -1, 3], dtype=torch.int32, device=DEV)
    bad = torch.tensor([9, 0, 2, -5, 3], dtype=torch.int32, device=DEV)
    assert torch.equal(anchor.tree_attention(*dev[:8], parents=bad), anchor.tree_attention(*dev[:8], parents=good))
    dev[5][0, 1] = 2 ** 30
    assert torch.isfinite(anchor.tree_attention(*dev[:8], parents=good)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("KV", [8, 2])
def test_siblings_that_are_no_numbers(KV, d, dtype):
    """Draft 3 with NaN keys and values, draft 4 with an infinite value: they reach themselves and what hangs on them, nobody else.
    A context that ends with an infinite value gives its infinity.  (Few rows to a key head, and many.)"""
    lens, new = [0, 33, 300], [12, 9, 12]
    args = make(lens, new, 8, KV, d, 16, dtype)
    q, k, v, kp, vp, table, cl, cu, _ = args
    parents = torch.tensor([-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 2, 8] + [-1, 0, 0, 0, 1, 2, 3, 4, 5] + [-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 2, 8],
                           dtype=torch.int32)
    tree = lambda *a: anchor.tree_attention(*(t.to(DEV) for t in a), parents=parents.to(DEV)).cpu().double()  # noqa: E731
    want, bound = oa.tree_attention(*args[:8], parents)
    last = int(table[2, 299 // 16])
    for b, lo in enumerate((0, 12, 21)):
        k[lo + 3], v[lo + 3] = float("nan"), float("nan")
        v[lo + 4, :, 5] = float("inf")
    vp[last, :, 299 % 16, 6] = float("-inf")
    got = tree(*args[:8])
    f = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * ((d + 4) * 41 + 300 + 72)
    slack = f * (bound + want.abs()) + 2.0 ** -18 * bound
    for lo, n in ((0, 12), (12, 9), (21, 12)):
        for i in range(n):
            up, j = set(), i
            while j >= 0:
                up.add(j)
                j = int(parents[lo + j])
            y, special = got[lo + i], {}
            if 3 in up:
                assert torch.isnan(y).all()
                continue
            if 4 in up:
                special[5] = float("inf")
            if lo == 21:
                special[6] = float("-inf")
            keep = torch.ones(d, dtype=torch.bool)
            for x, value in special.items():
                assert (y[:, x] == value).all(), (lo, i, x)
                keep[x] = False
            assert torch.isfinite(y[:, keep]).all(), (lo, i)
            assert float(((y - want[lo + i]).abs() - slack[lo + i])[:, keep].max()) <= 0, (lo, i)


@pytest.mark.gpu
def test_far_pages_pass_32_bits():
    """A slab over 4 GiB: its last pages lie at offsets past 2^32 bytes and 2^31 elements."""
    P, KV, d = 64, 4, 128
    pages = (1 << 31) // (P * KV * d) + 64
    kp = torch.zeros(pages, KV, P, d, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(1)
    small = torch.randn(4, 2, KV, P, d, generator=g).to(torch.bfloat16)
    kp[-4:] = small[:, 0].to(DEV)
    kp[-8:-4] = small[:, 1].to(DEV)
    q, k, v = (torch.randn(1, h, d, generator=g).to(DEV, torch.bfloat16) for h in (8, 4, 4))
    ctx = torch.tensor([200], dtype=torch.int32, device=DEV)
    near = anchor.tree_attention(q, k, v, small[:, 0].contiguous().to(DEV), small[:, 1].contiguous().to(DEV),
                                 torch.arange(4, dtype=torch.int32, device=DEV)[None], ctx)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device=DEV)[None]
    back, fwd = kp[:-4], kp[4:]  # two views of the slab whose pages of one number are four apart
    got = anchor.tree_attention(q, k, v, fwd, back, table - 4, ctx)
    assert torch.equal(got, near)
    rows = (table[0].long() * P + 5).to(DEV)
    new = torch.randn(4, KV, d, generator=g).to(DEV, torch.bfloat16)
    anchor.page_append(new, new, kp, kp, rows)
    assert torch.equal(kp[-4:, :, 5], new)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    lens, new = [600, 300], [1, 4]
    q, k, v, kp, vp, table, ctx, cu, par = (t.to(DEV) for t in make(lens, new, 8, 2, 64, 16, torch.bfloat16))
    y = anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, parents=par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, parents=par)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, parents=par)
    for r in range(3):
        ctx.sub_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, parents=par)), r


@pytest.mark.gpu
def test_refusals():
    q, k, v, kp, vp, table, ctx, cu, par = (t.to(DEV) for t in make([20], [2], 8, 2, 64, 16, torch.bfloat16))
    with pytest.raises(ValueError):
        anchor.tree_attention(q, k, v, kp, vp, table, ctx)                      # two tokens of one stream without offsets
    with pytest.raises(ValueError):
        anchor.tree_attention(q, k, v, kp, vp, table.long(), ctx, cu)
    with pytest.raises(ValueError):
        anchor.tree_attention(q, k, v, kp.float(), vp, table, ctx, cu)
    with pytest.raises(ValueError):
        anchor.tree_attention(q, k, v, kp[:, :1], vp[:, :1], table, ctx, cu)
    with pytest.raises(RuntimeError):
        anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, max_new=65)
    with pytest.raises(RuntimeError):
        anchor.tree_attention(q, k, v, kp[:, :, :8].contiguous(), vp[:, :, :8].contiguous(), table, ctx, cu)  # pages of 8
    deep = torch.zeros(1, 100, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        anchor.tree_attention(q, k, v, kp, vp, deep, ctx, cu, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
