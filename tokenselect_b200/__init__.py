"""tokenselect_b200: decode-time token selection + sparse paged attention as sm_100a CUDA kernels
behind a C ABI (``include/tokenselect_b200.h``), with the host-side mirror of the reference patcher's
decode surface.  No CPU path: the CUDA library is required."""
from .engine import TokenSelectConfig, TokenSelectEngine, rotary_tables  # noqa: F401
from .prompt import norm_rotate, prompt_attend  # noqa: F401
from .quant_cache import kv4_attend, kv4_attend_workspace, kv4_pool, kv4_read, kv4_row_bytes, kv4_write  # noqa: F401
from ._lib import TokenSelectError, TS_FLAG_DENSE, TS_FLAG_RECOMPUTE, TS_FLAG_REUSE  # noqa: F401

__all__ = ["TokenSelectConfig", "TokenSelectEngine", "TokenSelectError", "rotary_tables",
           "TS_FLAG_DENSE", "TS_FLAG_RECOMPUTE", "TS_FLAG_REUSE", "norm_rotate", "prompt_attend", "kv4_attend",
           "kv4_attend_workspace", "kv4_pool", "kv4_read", "kv4_row_bytes", "kv4_write"]
