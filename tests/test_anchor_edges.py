"""The anchor layers' surface at its edges, with no GPU: the layer's frequencies, a plan's arguments, the operators' checks."""
import torch

from layers import AnchorAttentionLayer


def test_frequencies_are_made_with_the_layer():
    """They are there before the first call, normal tensors whichever mode that call is in (training saves them), and float64
    whatever the layer is cast to."""
    layer = AnchorAttentionLayer(128, 2, 1, rotary_dim=32)
    with torch.inference_mode():
        first = layer.inv_freq(torch.device("cpu"))
    assert not first.is_inference()
    want = 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    for cast in (layer, layer.to(torch.bfloat16), layer.double()):
        f = cast.inv_freq(torch.device("cpu"))
        assert f.dtype == torch.float64 and float((f - want).abs().max()) < 1e-15
    with torch.inference_mode():
        assert not AnchorAttentionLayer(128, 2).inv_freq(torch.device("cpu")).is_inference()


def test_frequencies_follow_the_parameters():
    with torch.device("meta"):
        layer = AnchorAttentionLayer(128, 2, 1, rotary_dim=32)
    assert layer.inv_freq(torch.device("meta")).device.type == "meta"
    layer.to_empty(device="cpu")
    f = layer._inv_freq
    assert f.device.type == "cpu" and float(f[0]) == 1.0
    assert layer.inv_freq(torch.device("cpu")) is f
    assert "inv_freq" not in "".join(layer.state_dict())
