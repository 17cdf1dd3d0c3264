from torchsso.nn.layer_norm import LayerNorm, add_layer_norm, layer_norm  # NOQA
from torchsso.nn.rms_norm import RMSNorm, add_rms_norm, rms_norm  # NOQA
