from primus_turbo.pytorch.ops.attention.paged_attention import (  # noqa: F401
    kv_cache_read,
    kv_cache_write,
    paged_attention,
)

__all__ = ["kv_cache_read", "kv_cache_write", "paged_attention"]
