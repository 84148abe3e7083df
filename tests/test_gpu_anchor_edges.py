"""The anchor layers' surface at its edges on the GPU: first calls in a capture, on another stream and in inference mode,
rows that no sequence has, layouts with odd strides, autograd's other modes, steps without tokens."""
import pytest
import torch

from layers import AnchorAttentionLayer

DEV = "cuda:0"


def layer_and_input(**kw):
    torch.manual_seed(0)
    return AnchorAttentionLayer(256, 4, 2, rotary_dim=32, **kw).to(DEV), torch.randn(2, 40, 256, device=DEV)


@pytest.mark.gpu
def test_layer_first_called_on_two_streams():
    layer, x = layer_and_input()
    with torch.no_grad():
        want = AnchorAttentionLayer.forward(layer, x)
        torch.cuda.synchronize()
        again, _ = layer_and_input()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        out = []
        for s in (a, b):  # neither waits for the other
            with torch.cuda.stream(s):
                out.append(again(x))
        torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in out)


@pytest.mark.gpu
def test_layer_first_called_in_a_capture():
    layer, x = layer_and_input()
    with torch.no_grad():
        layer.w_q(x)  # the library's handles, which a capture cannot make
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x)
        eager = layer(x)  # before the first replay
        torch.cuda.synchronize()
        other, _ = layer_and_input()
        assert torch.equal(eager, other(x))
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


@pytest.mark.gpu
def test_layer_trains_after_inference_mode():
    layer, x = layer_and_input()
    with torch.inference_mode():
        want = layer(x).clone()
    y = layer(x)
    assert torch.equal(y.detach(), want.clone())
    y.sum().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in layer.parameters())
