"""Reference-named layer surface of the prefill path on MI355X (reference layers/__init__.py:5), and the softmax anchor layer."""
from .anchor_attention_layer import AnchorAttentionLayer
from .kernel_deltanet_layer import KernelDeltaNetLayer, KernelTTTLayer, MultiHeadRKHSKernel

__all__ = ["AnchorAttentionLayer", "KernelDeltaNetLayer", "KernelTTTLayer", "MultiHeadRKHSKernel"]
