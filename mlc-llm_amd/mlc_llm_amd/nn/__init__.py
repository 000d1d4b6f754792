"""Layer-level mirror: the quantized Mixtral MoE block; layers on 8-bit block-scaled weights."""
from .fp8 import Fp8Linear, Fp8MoE  # noqa: F401
from .mixtral_moe import MixtralMoE  # noqa: F401
