from primus_turbo.pytorch.ops.attention.kv_pages import kv_cache_copy, kv_cache_fork  # noqa: F401
from primus_turbo.pytorch.ops.attention.paged_attention import (  # noqa: F401
    kv_cache_read,
    kv_cache_write,
    paged_attention,
)
from primus_turbo.pytorch.ops.attention.qk_norm_rope import qk_norm_rope, qk_norm_rope_cache_write  # noqa: F401
from primus_turbo.pytorch.ops.attention.sparse_attention import (  # noqa: F401
    kv_page_ranges,
    select_pages,
    sparse_paged_attention,
)

__all__ = [
    "kv_cache_copy",
    "kv_cache_fork",
    "kv_cache_read",
    "kv_cache_write",
    "kv_page_ranges",
    "paged_attention",
    "qk_norm_rope",
    "qk_norm_rope_cache_write",
    "select_pages",
    "sparse_paged_attention",
]
