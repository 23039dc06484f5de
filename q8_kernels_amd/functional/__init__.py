from . import cross_attention, fast_hadamard, flash_attention, fma, fused, layer_norm, linear, quantizer, rms_norm, rope, rotary  # noqa: F401
