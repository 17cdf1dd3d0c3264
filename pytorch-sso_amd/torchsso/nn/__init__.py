from torchsso.nn.rms_norm import RMSNorm, add_rms_norm, rms_norm  # NOQA
