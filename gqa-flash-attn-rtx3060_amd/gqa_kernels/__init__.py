"""MI355X (gfx950) GQA flash-attention forward.

Drop-in for reference gqa_kernels/__init__.py:1-4: same import path and the
same public function, ``gqa_flash_attn(q, k, v, causal=True)``.
"""
from .dispatch import gqa_flash_attn
from .rotary import RotaryTable, qk_norm_rope, qk_norm_rope_write  # noqa: F401
from .scores import DocumentSpans, document_spans  # noqa: F401

# (``from gqa_kernels import *`` gives the reference's name alone; the others
# are the package's attributes.)
__all__ = ["gqa_flash_attn"]
__version__ = "0.1.0"
