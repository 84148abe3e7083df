"""The anchor layer, the pool's pages and the recurrent layer together: what a stream gives token by token, in pieces, forked
or verified as a tree, is what one pass over its whole prompt gives."""
import pytest
import torch

from kdn import anchor
from layers import AnchorAttentionLayer, KernelDeltaNetLayer
from serving import HybridMemoryPool

DEV = "cuda:0"


def make(dtype=torch.float32, heads=4, kv=2, d_head=64, layers=2, **kw):
    torch.manual_seed(0)
    net = [AnchorAttentionLayer(heads * d_head, heads, kv, rotary_dim=32, **kw).to(DEV, dtype) for _ in range(layers)]
    pool = HybridMemoryPool(8, 512, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device=DEV, anchor_layers=layers, anchor_heads=kv,
                            anchor_dim=d_head, anchor_pages=80, anchor_dtype=dtype)
    return net, pool


def whole(net, x):
    for layer in net:
        x = x + layer(x)
    return x


def step(net, pool, plan, x, parents=None):
    kept = []
    for i, layer in enumerate(net):
        r = layer.step(x, plan, *pool.anchor_pages(i), parents=parents)
        if not plan.keep:
            r, k, v = r
            kept.append((k, v))
        x = x + r
    return (x, kept) if not plan.keep else x


def same(a, b, dtype=torch.float32):
    """Two orders of the same fp32 sums through two layers: some hundred roundings of 2^-24 on values near 1."""
    err = float((a.float() - b.float()).norm() / b.float().norm())
    assert err < (2.0 ** -16 if dtype == torch.float32 else 2.0 ** -5), err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_then_tokens(dtype):
    net, pool = make(dtype)
    lens, more = [70, 1, 33], 5
    xs = [torch.randn(n + more, 256, device=DEV).to(dtype) for n in lens]
    with torch.no_grad():
        want = [whole(net, x[None])[0] for x in xs]
        streams = [pool.allocate_stream(n) for n in lens]
        plan = pool.anchor_plan(streams, lens)
        got = step(net, pool, plan, torch.cat([x[:n] for x, n in zip(xs, lens)])).split(lens)
        for g, w, n in zip(got, want, lens):
            same(g, w[:n], dtype)
        for t in range(more):
            if t == 2:
                pool.release_stream(pool.fork_stream(streams[0]))
                assert pool.anchor_compact() >= 0
            plan = pool.anchor_plan(streams, [1] * 3)
            got = step(net, pool, plan, torch.stack([x[n + t] for x, n in zip(xs, lens)]))
            for g, w, n in zip(got, want, lens):
                same(g, w[n + t], dtype)
    assert [pool.anchor_tokens(s) for s in streams] == [n + more for n in lens]
    for s in streams:
        pool.release_stream(s)
    assert pool.anchor_pages_used == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", [[100, 100, 7], [30, 64, 64], [65, 1, 90]])
def test_a_prompt_in_pieces(pieces):
    net, pool = make()
    x = torch.randn(sum(pieces), 256, device=DEV)
    s, done = pool.allocate_stream(0), 0
    with torch.no_grad():
        want = whole(net, x[None])[0]
        for n in pieces:
            got = step(net, pool, pool.anchor_plan([s], [n]), x[done:done + n])
            same(got, want[done:done + n])
            done += n


@pytest.mark.gpu
def test_forks_go_their_own_ways():
    net, pool = make()
    x = torch.randn(3, 60, 256, device=DEV)
    x[1:, :37] = x[0, :37]  # one prompt of 37 tokens, three continuations
    with torch.no_grad():
        want = whole(net, x)
        a = pool.allocate_stream(37)
        step(net, pool, pool.anchor_plan([a], [37]), x[0, :37])
        used = pool.anchor_pages_used
        b, c = pool.fork_stream(a), pool.fork_stream(a)
        assert pool.anchor_pages_used == used  # shared
        for t in range(37, 60):
            got = step(net, pool, pool.anchor_plan([a, b, c], [1, 1, 1]), x[:, t])
            same(got, want[:, t])
    assert pool.anchor_pages_used == 2 + 3 * 2  # two full pages of all three, two more each


@pytest.mark.gpu
def test_a_tree_of_drafts_and_what_is_accepted():
    net, pool = make()
    n = 45
    path = torch.randn(1, n + 4, 256, device=DEV)
    wrong = torch.randn(2, 256, device=DEV)
    #  0 - 1 - 3 - 5     the path that will be accepted
    #    \ 2   \ 4       and two that will not
    x = torch.stack([path[0, n], path[0, n + 1], wrong[0], path[0, n + 2], wrong[1], path[0, n + 3]])
    parents, depths = [-1, 0, 0, 1, 1, 3], [0, 1, 1, 2, 2, 3]
    with torch.no_grad():
        want = whole(net, path)[0]
        other = [whole(net, torch.cat([path[:, :n + i], w[None, None]], dim=1))[0, -1] for i, w in ((1, wrong[0]), (2, wrong[1]))]
        s = pool.allocate_stream(n)
        step(net, pool, pool.anchor_plan([s], [n]), path[0, :n])
        plan = pool.anchor_plan([s], [6], depths=depths)
        got, kept = step(net, pool, plan, x, parents=torch.tensor(parents, dtype=torch.int32, device=DEV))
        same(got[[0, 1, 3, 5]], want[n:n + 4])
        same(got[[2, 4]], torch.stack(other))
        assert pool.anchor_tokens(s) == n
        took = torch.tensor([0, 1, 3], device=DEV)  # three are accepted: their keys and values go into the pages
        rows = pool.anchor_plan([s], [3]).rows
        for i, (k, v) in enumerate(kept):
            anchor.page_append(k[took], v[took], *pool.anchor_pages(i), rows)
        got = step(net, pool, pool.anchor_plan([s], [1]), path[0, n + 3:n + 4])
        same(got[0], want[n + 3])


@pytest.mark.gpu
def test_a_step_without_room_changes_nothing():
    net, pool = make()
    a, b = pool.allocate_stream(0), pool.allocate_stream(0)
    x = torch.randn(600, 256, device=DEV)
    with torch.no_grad():
        step(net, pool, pool.anchor_plan([a], [600]), x)
        c = pool.fork_stream(a)
        used = pool.anchor_pages_used
        with pytest.raises(RuntimeError):
            pool.anchor_plan([c, b], [10, 1000])
        assert pool.anchor_tokens(c) == 600 and pool.anchor_tokens(b) == 0 and pool.anchor_pages_used - used <= 1
        more = torch.randn(1, 1, 256, device=DEV)
        want = whole(net, torch.cat([x[None], more], dim=1))[0, -1]
        for s in (a, c):
            same(step(net, pool, pool.anchor_plan([s], [1]), more[0])[0], want)


@pytest.mark.gpu
def test_training_beside_the_recurrent_layer():
    """A hybrid block's gradients against the same block with the attention in float64 autograd."""
    torch.manual_seed(1)
    B, T, H = 2, 70, 4
    lin = KernelDeltaNetLayer(256, H).to(DEV)
    att = AnchorAttentionLayer(256, H, 2, rotary_dim=48, scaling="parts", factor=4.0).to(DEV)
    x = torch.randn(B, T, 256, device=DEV, requires_grad=True)
    h = x + lin(x)[0]
    out = h + att(h)
    dy = torch.randn_like(out)
    out.backward(dy)
    got = [x.grad, *(p.grad for p in att.parameters())]

    ref = AnchorAttentionLayer(256, H, 2, rotary_dim=48, scaling="parts", factor=4.0).double()
    ref.load_state_dict({k: v.cpu().double() for k, v in att.state_dict().items()})
    hr = h.detach().cpu().double().requires_grad_(True)
    q, k, v = (w(hr).view(B, T, -1, 64) for w in (ref.w_q, ref.w_k, ref.w_v))
    f, mag = anchor.rotary_frequencies(48, scaling="parts", factor=4.0)
    z = torch.polar(torch.full((), mag, dtype=torch.float64), torch.arange(T).double()[:, None] * f)[None, :, None]

    def turn(t):
        r = torch.complex(t[..., :24], t[..., 24:48]) * z
        return torch.cat([r.real, r.imag, t[..., 48:]], dim=-1)

    q, k = turn(q), turn(k).repeat_interleave(2, dim=2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / 8
    p = s.masked_fill(~torch.ones(T, T, dtype=torch.bool).tril(), float("-inf")).softmax(-1)
    o = torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(2, dim=2)).reshape(B, T, 256)
    (hr + ref.w_out(o)).backward(dy.cpu().double())
    # the part of dL/dx that comes through the recurrent layer, from the same dL/dh
    want = torch.autograd.grad(x + lin(x)[0], x, hr.grad.float().to(DEV))[0]
    for a, b in zip(got, [want, *(p.grad for p in ref.parameters())]):
        same(a.cpu(), b.cpu())


@pytest.mark.gpu
def test_packed_and_uniform_forward_agree():
    net, _ = make(layers=1)
    x = torch.randn(2, 40, 256, device=DEV)
    with torch.no_grad():
        y = net[0](x)
        packed = net[0](x.reshape(80, 256), torch.tensor([0, 40, 80], device=DEV))
        assert torch.equal(packed.view(y.shape), y)
        short = net[0](x.reshape(80, 256), torch.tensor([0, 40, 61], device=DEV))
        assert torch.equal(short[:40], y[0]) and not short[61:].any()
    with pytest.raises(ValueError):
        AnchorAttentionLayer(256, 8)  # heads of 32
