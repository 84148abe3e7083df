"""Bounded contexts as they are used: anchor layers with a window over pages that slide, and layers whose steps weigh the cached keys
that the pool then cuts; against whole prompts, and against attention over the tokens that were kept."""
import pytest
import torch

from kdn import anchor
from layers import AnchorAttentionLayer
from oracle import bounded as ob
from serving import HybridMemoryPool

DEV = "cuda:0"


def make(dtype=torch.float32, heads=4, kv=2, d_head=64, layers=2, pages=200, queries=None, **kw):
    torch.manual_seed(0)
    net = [AnchorAttentionLayer(heads * d_head, heads, kv, rotary_dim=32, **kw).to(DEV, dtype) for _ in range(layers)]
    pool = HybridMemoryPool(8, 512, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device=DEV, anchor_layers=layers, anchor_heads=kv,
                            anchor_dim=d_head, anchor_pages=pages, anchor_dtype=dtype, anchor_queries=queries)
    return net, pool


def step(net, pool, plan, x, weigh=False, **kw):
    for i, layer in enumerate(net):
        x = x + layer.step(x, plan, *pool.anchor_pages(i), weights=pool.anchor_weights(i) if weigh else None, **kw)
    return x


def same(a, b, dtype=torch.float32):
    """Two orders of the same fp32 sums through two layers: some hundred roundings of 2^-24 on values near 1."""
    err = float((a.float() - b.float()).norm() / b.float().norm())
    assert err < (2.0 ** -16 if dtype == torch.float32 else 2.0 ** -5), err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(20, 0), (70, 4), (33, 20)])
def test_windows_slide(window, sinks, dtype):
    """A prompt, tokens, a piece and a run; the pages between sinks and window are freed as they go."""
    net, pool = make(dtype, window=window, sinks=sinks)
    lens = [(150, 1, 1, 100, 9, 1), (30, 1, 1, 80, 40, 1)]
    xs = [torch.randn(sum(n), 256, device=DEV).to(dtype) for n in lens]
    with torch.no_grad():
        want = []
        for x in xs:
            y = x[None]
            for layer in net:
                y = y + layer(y)
            want.append(y[0])
        streams, done = [pool.allocate_stream(0) for _ in lens], [0, 0]
        for new in zip(*lens):
            plan = pool.anchor_plan(streams, new)
            got = step(net, pool, plan, torch.cat([x[d:d + n] for x, d, n in zip(xs, done, new)])).split(new)
            for g, w, d, n in zip(got, want, done, new):
                same(g, w[d:d + n], dtype)
            done = [d + n for d, n in zip(done, new)]
            pool.anchor_slide(streams, window, sinks)
            assert all(pool.anchor_tokens(s) < window + sinks + 3 * 16 for s in streams)
    assert pool.anchor_pages_used < (sum(done) // 16) * (0.9 if window < 70 else 1.0)


@pytest.mark.gpu
def test_a_tree_of_drafts_in_a_window():
    net, pool = make(window=3, sinks=1)
    n = 45
    path = torch.randn(1, n + 4, 256, device=DEV)
    x = torch.stack([path[0, n], path[0, n + 1], torch.randn(256, device=DEV), path[0, n + 2], path[0, n + 3]])
    with torch.no_grad():
        y = path
        for layer in net:
            y = y + layer(y)
        s = pool.allocate_stream(n)
        step(net, pool, pool.anchor_plan([s], [n]), path[0, :n])
        pool.anchor_slide([s], 3, 1)
        plan = pool.anchor_plan([s], [5], depths=[0, 1, 1, 2, 3])
        for i, layer in enumerate(net):
            r, _, _ = layer.step(x, plan, *pool.anchor_pages(i), parents=torch.tensor([-1, 0, 0, 1, 3], dtype=torch.int32, device=DEV))
            x = x + r
        same(x[[0, 1, 3, 4]], y[0, n:])


@pytest.mark.gpu
def test_training_a_layer_with_a_window():
    """Gradients of a layer's parameters against those of the same function of torch operations in 64 bits."""
    torch.manual_seed(0)
    layer = AnchorAttentionLayer(256, 4, 2, rotary_dim=64, window=9, sinks=2).to(DEV)
    x = torch.randn(2, 40, 256, device=DEV)
    dy = torch.randn_like(x)
    got = torch.autograd.grad(layer(x), list(layer.parameters()), dy)
    wq, wk, wv, wo = (p.detach().double().requires_grad_(True) for p in layer.parameters())
    t = torch.arange(40, device=DEV, dtype=torch.float64)[:, None] * layer.inv_freq(x.device)[None]
    c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]

    def turn(z):
        a, b = z[..., :32], z[..., 32:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    hide = ~ob.visible(9, 2)(40, 40).to(DEV)
    rows = []
    for xb in x.double():
        q, k, v = turn((xb @ wq.T).view(40, 4, 64)), turn((xb @ wk.T).view(40, 2, 64)), (xb @ wv.T).view(40, 2, 64)
        y = [torch.softmax((q[:, h] @ k[:, h // 2].T / 8).masked_fill(hide, -float("inf")), -1) @ v[:, h // 2] for h in range(4)]
        rows.append(torch.cat(y, -1) @ wo.T)
    for a, b in zip(got, torch.autograd.grad(torch.stack(rows), [wq, wk, wv, wo], dy.double())):
        assert float((a.double() - b).norm() / b.norm()) < 2.0 ** -16  # sums of 80 and 256 fp32 products, a few hundred roundings of 2^-24


class Kept:
    """One layer and stream in 64 bits: which positions a head has, their keys, values and weights, in no order."""

    def __init__(self, kv):
        self.k, self.v, self.w = ([{} for _ in range(kv)] for _ in range(3))

    def attend(self, q, k, v, at):
        """The token at position `at` over what is kept and itself; its output; weights are added."""
        H, kv = q.shape[0], len(self.k)
        y = torch.empty_like(q)
        for e in range(kv):
            self.k[e][at], self.v[e][at], self.w[e][at] = k[e], v[e], 0.0
            pos = list(self.k[e])
            kk, vv = torch.stack([self.k[e][p] for p in pos]), torch.stack([self.v[e][p] for p in pos])
            for h in range(e * H // kv, (e + 1) * H // kv):
                p = torch.softmax(kk @ q[h] / q.shape[1] ** 0.5, 0)
                y[h] = p @ vv
                for x, i in zip(p.tolist(), pos):
                    self.w[e][i] += x
        return y

    def cut(self, keep, total, sinks, recent):
        for e in range(len(self.k)):
            order = sorted(self.k[e], key=lambda p: (p >= sinks, p < total - recent, -self.w[e][p], p))
            for p in order[keep:]:
                del self.k[e][p], self.v[e][p], self.w[e][p]


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", [(60,), (40, 20), (57, 3), (30, 5, 25)])
def test_cut_streams_go_on(pieces):
    """A prompt in pieces, weighed; cut to 32; tokens with a cut after each; a fork that goes its own way and is cut, too."""
    net, pool = make(layers=1, queries=4)
    layer, n, more = net[0], sum(pieces), 6
    assert pool.anchor_weights(0).shape == (8, 2, 512)
    x = torch.randn(n + 2 * more, 256, device=DEV)
    with torch.no_grad():
        at = torch.arange(n + more, device=DEV)
        rows = {}
        for name, z in (("a", x[:n + more]), ("b", torch.cat([x[:n], x[n + more:]]))):
            rows[name] = [t.double().cpu() for t in layer._project(z, at)]
        s, done = pool.allocate_stream(0), 0
        for m in pieces:
            step(net, pool, pool.anchor_plan([s], [m]), x[done:done + m], True)
            done += m
        model = {"a": Kept(2), "b": Kept(2)}
        for name, (q, k, v) in rows.items():
            for t in range(n):
                model[name].attend(q[t], k[t], v[t], t)

        def look(stream, m):
            """The pool's weights and positions are the model's; positions of the settled places, the others by their place."""
            L, settled, gone = pool.anchor_tokens(stream), pool._settled[stream], pool._gone[stream]
            for e in range(2):
                pos = pool._positions[stream, 0, e, :settled].tolist() + [j + gone for j in range(settled, L)]
                assert sorted(pos) == sorted(m.k[e])
                w = pool.anchor_weights(0)[stream, e].tolist()
                assert max(abs(w[j] - m.w[e][p]) for j, p in enumerate(pos)) < 60 * 2.0 ** -18  # sums of up to 132 weights
                assert not any(w[L:])

        look(s, model["a"])
        f = pool.fork_stream(s)
        pool.anchor_evict([s, f], 32, sinks=2, recent=5)
        for m in model.values():
            m.cut(32, n, 2, 5)
        for t in range(more):
            plan = pool.anchor_plan([s, f], [1, 1])
            got = layer.step(torch.stack([x[n + t], x[n + more + t]]), plan, *pool.anchor_pages(0), weights=pool.anchor_weights(0))
            for g, (stream, name) in zip(got, ((s, "a"), (f, "b"))):
                q, k, v = (r[n + t] for r in rows[name])
                want = layer.w_out(model[name].attend(q, k, v, n + t).float().to(DEV).view(-1))
                same(g, want)
                look(stream, model[name])
            if t % 2 == 0:
                pool.anchor_evict([s, f], 32, sinks=2, recent=5)
                for m in model.values():
                    m.cut(32, n + t + 1, 2, 5)
        with pytest.raises(ValueError):  # among the kept ones, which lie in no order
            pool.anchor_truncate(s, 20)
        pool.anchor_truncate(s, 32)
        look_w = pool.anchor_weights(0)[s]
        assert not look_w[:, 32:].any() and look_w[:, :32].any()
    pool.release_stream(s)
    pool.release_stream(f)
    assert pool.anchor_pages_used == 0
    again = pool.allocate_stream(0)
    assert not pool.anchor_weights(0)[again].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_pages_stay_as_they_were(dtype):
    """Cutting a fork moves no row of its parent's pages; accepted drafts come without weights, as zeros."""
    net, pool = make(dtype, queries=4)
    x = torch.randn(90, 256, device=DEV).to(dtype)
    with torch.no_grad():
        a = pool.allocate_stream(0)
        step(net, pool, pool.anchor_plan([a], [90]), x, True)
        rows = pool._anchor.rows(pool._anchor_stream[a], 0, 90)
        look = lambda: [pool.anchor_pages(i)[j][rows // 16, :, rows % 16].clone() for i in range(2) for j in range(2)]  # noqa: E731
        before, w = look(), pool.anchor_weights(1)[a].clone()
        b = pool.fork_stream(a)
        pool.anchor_evict([b], 50, sinks=1, recent=4)
        assert all(torch.equal(p, q) for p, q in zip(before, look())) and torch.equal(w, pool.anchor_weights(1)[a])
        plan = pool.anchor_plan([b], [2])
        anchor.page_append(*(torch.randn(2, 2, 64, device=DEV).to(dtype) for _ in range(2)), *pool.anchor_pages(0), plan.rows)
        assert not pool.anchor_weights(0)[b, :, 50:].any()
        nxt = torch.randn(2, 256, device=DEV).to(dtype)
        with torch.no_grad():
            solo = step(net, pool, pool.anchor_plan([a], [1]), nxt[:1], True)
        assert torch.isfinite(solo).all()


@pytest.mark.gpu
def test_many_query_heads_to_a_key_head():
    """More than 32 rows to a key head: a token's step takes the whole keys, and the same weights come of it."""
    net, pool = make(heads=36, kv=1, layers=1, queries=36)
    x = torch.randn(41, 36 * 64, device=DEV)
    with torch.no_grad():
        s, t = pool.allocate_stream(0), pool.allocate_stream(0)
        step(net, pool, pool.anchor_plan([s], [41]), x, True)
        step(net, pool, pool.anchor_plan([t], [40]), x[:40], True)
        step(net, pool, pool.anchor_plan([t], [1]), x[40:], True)
    w = pool.anchor_weights(0)
    assert float((w[s] - w[t]).abs().max()) < 41 * 36 * 2.0 ** -18
    assert abs(float(w[s].double().sum()) - 41 * 36) < 41 * 36 * 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("keep,sinks,recent", [(12, 2, 64), (12, 0, 12), (20, 4, 2 ** 40), (3, 5, 8), (12, 2, 11)])
def test_a_budget_below_sinks_and_recent_keeps_the_latest(keep, sinks, recent):
    """Cut after every token, whatever the weights: the sinks, then the latest tokens, the one just written among them."""
    _, pool = make(layers=2, queries=4)
    s = pool.allocate_stream(0)
    total = 50
    pool.anchor_plan([s], [total])
    pool._weights[s] = torch.rand(pool._weights[s].shape, device=DEV).sort(-1, descending=True).values  # the oldest the largest
    for _ in range(6):
        pool.anchor_evict([s], keep, sinks=sinks, recent=recent)
        first = min(sinks, keep)
        want = [*range(first), *range(total - (keep - first), total)]
        for pos in pool._positions[s, :, :, :keep].flatten(0, 1).tolist():
            assert sorted(pos) == want
        assert pool.anchor_tokens(s) == keep
        pool.anchor_plan([s], [1])
        pool._weights[s, :, :, keep] = 0.1
        total += 1


@pytest.mark.gpu
def test_cutting_clears_the_places_that_streams_had():
    """Those and no others: what a cut costs goes by what it takes away, not by the longest stream that the pool has room for."""
    _, pool = make(layers=2, queries=4)
    a, b, c = (pool.allocate_stream(0) for _ in range(3))
    pool.anchor_plan([a, b, c], [90, 70, 60])
    pool._weights.fill_(5.0)
    w = pool._weights
    pool.anchor_evict([a, b], 50)
    assert not w[a, :, :, 50:90].any() and not w[b, :, :, 50:70].any() and bool((w[[a, b]][..., :50] == 5).all())
    assert bool((w[[a, b]][..., 90:] == 5).all()) and bool((w[c] == 5).all())
    pool.anchor_truncate(c, 20)
    assert not w[c, :, :, 20:60].any() and bool((w[c, :, :, :20] == 5).all()) and bool((w[c, :, :, 60:] == 5).all())
    pool.anchor_truncate(c, 20)
    with pytest.raises(RuntimeError):
        pool.anchor_truncate(c, 21)
    pool.anchor_truncate(c, 0)
    assert not w[c, :, :, :60].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_accepted_drafts_weigh_as_tokens_do(dtype):
    """A tree verified without weights, its accepted path as a run with them: the weights, positions and pages of tokens one by one."""
    net, pool = make(dtype, queries=4)
    n, path, tree = 50, [0, 1, 3], [-1, 0, 0, 1]  # draft 2 is refused
    x = torch.randn(n + 4, 256, device=DEV).to(dtype)
    with torch.no_grad():
        a, b = pool.allocate_stream(0), pool.allocate_stream(0)
        for s in (a, b):
            step(net, pool, pool.anchor_plan([s], [n]), x[:n], True)
        pool.anchor_evict([a, b], 40, sinks=2, recent=4)
        one = torch.cat([step(net, pool, pool.anchor_plan([a], [1]), x[n + t:n + t + 1], True) for t in path])
        drafts, y, before = pool.anchor_plan([b], [4], depths=[0, 1, 1, 2]), x[n:], []
        for i, layer in enumerate(net):
            before.append(y)
            y = y + layer.step(y, drafts, *pool.anchor_pages(i), parents=torch.tensor(tree, dtype=torch.int32, device=DEV), weights=pool.anchor_weights(i))[0]
        same(y[path], one, dtype)
        assert not pool.anchor_weights(0)[b, :, 40:].any()
        plan = pool.anchor_plan([b], [3])
        for i, layer in enumerate(net):
            layer.step(before[i][path], plan, *pool.anchor_pages(i), weights=pool.anchor_weights(i))
        for i in range(2):
            w = pool.anchor_weights(i)
            same(w[b], w[a], dtype)
            assert bool((w[b, :, 40:43] > 0).all())
            rows = [pool._anchor.rows(pool._anchor_stream[s], 0, 43) for s in (a, b)]
            for pages in pool.anchor_pages(i):
                same(*(pages[r // 16, :, r % 16] for r in rows), dtype)
