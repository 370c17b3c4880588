"""fna2_amd — FlashNaylisAttention-2 forward/backward for AMD MI355X (gfx950).

The hot path is ``flash_naylis_attn`` (module ``flash_naylis_attn``), backed by
hand-written HIP kernels in ``csrc/`` behind the C ABI of ``include/fna2.h``.
``attention_fna2`` holds the ``NaylisAttention`` caller with the reference's
constructor and forward signatures.  Around the path: ``rope.rope_varlen``
(varlen rotary embedding, optionally with the QK RMSNorm) and
``decode.flash_naylis_decode`` (one-token decode against a KV cache), and
for serving from a paged cache ``paged.flash_naylis_paged`` (chunks of new
tokens), ``paged.flash_naylis_shared`` (the same for sequences that share
their first rows), ``paged.paged_append`` and ``paged.paged_evict``, and its
books on the GPU, ``paged.DevicePageTable``.  ``rope.rotary_embed`` rotates in other
layouts, over part of the head, and scaled.
``ops`` registers the path as the custom operators ``fna2::fwd`` /
``fna2::bwd`` (fake and autograd registrations), which ``flash_naylis_attn``
calls, so that ``torch.compile`` traces it.
"""
from .decode import flash_naylis_decode  # noqa: F401
from .flash_naylis_attn import (  # noqa: F401
    BLOCK_M,
    BLOCK_N,
    BLOCK_R,
    FlashNaylisAttnFunc,
    flash_naylis_attn,
)
from .paged import (  # noqa: F401
    DevicePageTable,
    PagedKVCache,
    PageTable,
    flash_naylis_paged,
    flash_naylis_shared,
    paged_append,
    paged_evict,
    paged_extend,
    paged_groups,
    paged_trim,
)
from .rope import rope_varlen, rotary_embed, rotary_frequencies  # noqa: F401
from . import ops  # noqa: F401,E402  (registers the fna2::fwd / fna2::bwd custom ops)

__all__ = ["BLOCK_M", "BLOCK_N", "BLOCK_R", "FlashNaylisAttnFunc", "flash_naylis_attn",
           "flash_naylis_decode", "flash_naylis_paged", "flash_naylis_shared", "DevicePageTable", "PagedKVCache",
           "PageTable", "paged_append", "paged_evict", "paged_extend", "paged_groups", "paged_trim",
           "rope_varlen", "rotary_embed", "rotary_frequencies"]
