"""Model decode step around the packed projections."""
from .packed import PackedGraphDecoder, PagedCache
from .qwen35 import GraphDecoder, Qwen35Args, Qwen35Cache, Qwen35Model, build_qwen35

__all__ = ["GraphDecoder", "PackedGraphDecoder", "PagedCache", "Qwen35Args", "Qwen35Cache", "Qwen35Model", "build_qwen35"]
