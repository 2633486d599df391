from primus_turbo.pytorch.ops.moe.moe_decode import moe_decode  # noqa: F401
from primus_turbo.pytorch.ops.moe.moe_permute import moe_permute, moe_unpermute  # noqa: F401

__all__ = ["moe_decode", "moe_permute", "moe_unpermute"]
