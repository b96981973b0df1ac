from ._layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
