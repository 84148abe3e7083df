"""Pages on the device (kdn_page_copy, kdn_page_append) and the pool's bookkeeping with them: bits, exactly."""
import pytest
import torch

from kdn import anchor

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((40, 2, 2, 16, 64), torch.bfloat16), ((40, 1, 3, 16, 128), torch.float32), ((1200, 8), torch.bfloat16),
                                         ((30, 5000, 8), torch.bfloat16)])
def test_copy(shape, dtype):
    g = torch.Generator().manual_seed(0)
    host = torch.randn(shape, generator=g).to(dtype)
    order = torch.randperm(shape[0], generator=g)
    n = shape[0] // 2 - 1  # more than a launch's list for the largest
    pairs = torch.stack([order[:n], order[n:2 * n]], dim=1).int()
    slab = host.to(DEV)
    anchor.page_copy(slab, pairs)
    host[order[n:2 * n]] = host[order[:n]]
    assert torch.equal(slab.cpu(), host)
    anchor.page_copy(slab, [])
    anchor.page_copy(slab, [(0, 1)])
    host[1] = host[0]
    assert torch.equal(slab.cpu(), host)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,P,KV", [(64, 16, 1), (128, 32, 3)])
def test_append(d, P, KV, dtype):
    g = torch.Generator().manual_seed(1)
    slab = torch.randn(12, 2, 2, KV, P, d, generator=g).to(dtype)
    dev = slab.to(DEV)
    n = 5 * P
    rows = torch.randperm(12 * P, generator=g)[:n]
    rows[3], rows[7], rows[9] = -1, 12 * P, 1 << 40  # padding, and past the slab: skipped
    k, v = torch.randn(n, 2 * KV, d, generator=g).to(dtype).split([KV, KV], dim=1)
    anchor.page_append(k.to(DEV), v.to(DEV), dev[:, 1, 0], dev[:, 1, 1], rows.to(DEV))
    for i, r in enumerate(rows.tolist()):
        if 0 <= r < 12 * P:
            slab[r // P, 1, 0, :, r % P], slab[r // P, 1, 1, :, r % P] = k[i], v[i]
    assert torch.equal(dev.cpu(), slab)
    anchor.page_append(k[:0].to(DEV), v[:0].to(DEV), dev[:, 1, 0], dev[:, 1, 1], rows[:0].to(DEV))


@pytest.mark.gpu
def test_pool_keeps_every_streams_tokens():
    """Random opens, forks, writes, truncations, closes and compactions: what each stream reads back is what it wrote."""
    P, d = 16, 64
    pool = anchor.PagePool(60, P, 12)
    slab = torch.full((60, 2, 1, P, d), -1.0, device=DEV)
    g = torch.Generator().manual_seed(4)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    held, stamp = {}, 0
    for step in range(150):
        do = draw(10)
        s = sorted(held)[draw(len(held))] if held else None
        if s is None or (do == 0 and len(held) < 10):
            held[pool.open()] = []
        elif do == 1 and len(held) < 10:
            held[pool.fork(s)] = list(held[s])
        elif do == 2:
            pool.close(s)
            del held[s]
        elif do == 3:
            keep = draw(len(held[s]) + 1)
            pool.truncate(s, keep)
            held[s] = held[s][:keep]
        elif do == 4:
            anchor.page_copy(slab, pool.compact())
            used = {int(x) for t in held if held[t] for x in pool.table([t])[0]}
            assert used == set(range(pool.used))
        else:
            n = 1 + draw(40)
            first = len(held[s])
            free = pool.free
            try:
                anchor.page_copy(slab, pool.extend(s, n))
            except RuntimeError:
                assert pool.free == free and pool.length(s) == first  # refused for want of pages: nothing changed
                continue
            new = torch.arange(stamp, stamp + n, dtype=torch.float32)
            stamp += n
            kv = new[:, None, None].expand(n, 1, d).contiguous().to(DEV)
            anchor.page_append(kv, -kv, slab[:, 0], slab[:, 1], pool.rows(s, first, n).to(DEV))
            held[s] += new.tolist()
        if step % 10 == 9:
            for t, want in held.items():
                rows = pool.rows(t, 0, len(want)).to(DEV)
                assert slab[:, 0][rows // P, 0, rows % P, 0].tolist() == want
                assert slab[:, 1][rows // P, 0, rows % P, d - 1].tolist() == [-x for x in want]
    for s in list(held):
        pool.close(s)
    assert pool.free == 60


@pytest.mark.gpu
def test_refusals():
    slab = torch.zeros(8, 2, 16, 64, device=DEV)
    with pytest.raises(RuntimeError):
        anchor.page_copy(slab, [(0, 8)])
    with pytest.raises(RuntimeError):
        anchor.page_copy(slab, [(0, 1), (2, 1)])   # one target twice
    with pytest.raises(RuntimeError):
        anchor.page_copy(slab, [(0, 1), (1, 2)])   # a target that is a source
    with pytest.raises(ValueError):
        anchor.page_copy(slab[:, :1], [(0, 1)])
    with pytest.raises(RuntimeError):
        anchor.page_copy(torch.zeros(4, 3, device=DEV), [(0, 1)])  # pages of 12 bytes
    k = torch.zeros(2, 1, 64, device=DEV)
    rows = torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        anchor.page_append(k, k, slab[:, :1], slab[:, :1], rows[:1])
    with pytest.raises(ValueError):
        anchor.page_append(k, k, slab, slab, rows)  # two heads in the pages
    with pytest.raises(ValueError):
        anchor.page_append(k.bfloat16(), k.bfloat16(), slab[:, :1], slab[:, :1], rows)
