"""gfx950 HIP kernels for the training hot path + their fp32 references."""
from .functional import cross_entropy, norm_rope_qkv, rmsnorm, rope_qkv, swiglu  # noqa: F401
from .attn import attention, attention_packed  # noqa: F401
from .packed import PackedBatch  # noqa: F401
from .adamw import FusedAdamW  # noqa: F401
