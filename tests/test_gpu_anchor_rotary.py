"""Rotary positions (kdn_rotary) against the float64 definition.  A result is one product and one fused product and sum in
fp32 of a sine and cosine good to a few units, then one rounding: within (2^-8 for bf16, 8 units of 2^-24 for fp32) of
|a| + |b| times the magnitude."""
import pytest
import torch

from kdn import anchor
from oracle import anchor as oa

DEV = "cuda:0"


def make(n, H, KV, d, dtype, top, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(n, h, d, generator=g).to(dtype) for h in (H, KV))
    return q, k, torch.randint(0, top, (n,), generator=g)


def close(got, x, pos, f, mag, **kw):
    want = oa.rotary(x, pos, f, magnitude=mag, **kw)
    rot = 2 * f.shape[0]
    z = x.double().abs()
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if kw.get("interleaved") else (i, i + rot // 2)
    size = z.clone()
    size[..., a] = size[..., b] = (z[..., a] + z[..., b]) * mag
    unit = 2.0 ** -8 if x.dtype == torch.bfloat16 else 8 * 2.0 ** -24
    over = (got.cpu().double() - want).abs() - unit * size
    assert float(over.max() if over.numel() else 0) <= 0, float((over / size).max())
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])  # the rest is copied


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (128, 128), (128, 96), (128, 16), (64, 2), (64, 6), (128, 30), (128, 8)])
def test_layouts(d, rot, interleaved, dtype):
    q, k, pos = make(37, 6, 2, d, dtype, 131072)
    f, mag = anchor.rotary_frequencies(rot)
    qo, ko = anchor.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), f.to(DEV), interleaved=interleaved)
    close(qo, q, pos, f, mag, interleaved=interleaved)
    close(ko, k, pos, f, mag, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
@pytest.mark.parametrize("inverse", [False, True])
def test_scalings_and_the_inverse(scaling, inverse):
    q, k, pos = make(9, 4, 4, 128, torch.float32, 1 << 40)  # far positions: the angle is formed in 64 bits
    pos = pos % (1 << 22)
    f, mag = anchor.rotary_frequencies(128, scaling=scaling, factor=4.0)
    qo, ko = anchor.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), f.to(DEV), magnitude=mag, inverse=inverse)
    close(qo, q, pos, f, mag, inverse=inverse)
    close(ko, k, pos, f, mag, inverse=inverse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1, 5, 8191, 8193])
def test_token_counts(n):
    q, k, pos = make(n, 2, 1, 64, torch.bfloat16, 10000)
    f, mag = anchor.rotary_frequencies(64)
    qo, ko = anchor.rotary(q.to(DEV), k.to(DEV), pos.to(DEV).int(), f.to(DEV))
    close(qo, q, pos, f, mag)
    close(ko, k, pos, f, mag)


@pytest.mark.gpu
def test_views_in_place_and_q_alone():
    q, k, pos = make(50, 4, 2, 64, torch.bfloat16, 5000)
    f = anchor.rotary_frequencies(32)[0].to(DEV)
    want = anchor.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), f)
    fused = torch.cat([q, k, k], dim=1).to(DEV)
    qv, kv, vv = fused.split([4, 2, 2], dim=1)
    assert all(torch.equal(a, b) for a, b in zip(anchor.rotary(qv, kv, pos.to(DEV), f), want))
    anchor.rotary(qv, kv, pos.to(DEV), f, in_place=True)
    assert torch.equal(qv, want[0]) and torch.equal(kv, want[1]) and torch.equal(vv.cpu(), k)
    alone, none = anchor.rotary(q.to(DEV), None, pos.to(DEV), f)
    assert none is None and torch.equal(alone, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(interleaved):
    """The map is linear: its gradient is the inverse turn, and <R x, y> = <x, R' y>."""
    q, k, pos = make(20, 4, 2, 64, torch.float32, 9000)
    f, mag = anchor.rotary_frequencies(48, scaling="parts", factor=8.0)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k)]
    qo, ko = anchor.rotary(*leaves, pos.to(DEV), f.to(DEV), interleaved=interleaved, magnitude=mag)
    g = torch.Generator().manual_seed(5)
    dq, dk = (torch.randn(t.shape, generator=g) for t in (q, k))
    torch.autograd.backward([qo, ko], [dq.to(DEV), dk.to(DEV)])
    close(leaves[0].grad, dq, pos, f, mag, interleaved=interleaved, inverse=True)
    close(leaves[1].grad, dk, pos, f, mag, interleaved=interleaved, inverse=True)


@pytest.mark.gpu
def test_refusals():
    q, k, pos = (t.to(DEV) for t in make(4, 2, 1, 64, torch.bfloat16, 10))
    f = anchor.rotary_frequencies(64)[0].to(DEV)
    for bad in (dict(positions=pos[:3]), dict(positions=pos.float()), dict(inv_freq=f.float()), dict(inv_freq=torch.cat([f, f])),
                dict(k=k.float())):
        args = dict(q=q, k=k, positions=pos, inv_freq=f) | bad
        with pytest.raises(ValueError):
            anchor.rotary(**args)
    with pytest.raises(ValueError):
        anchor.rotary(q.float().requires_grad_(True), None, pos, f, in_place=True)
    with pytest.raises(ValueError):
        anchor.rotary_frequencies(63)
    with pytest.raises(ValueError):
        anchor.rotary_frequencies(64, scaling="other")
