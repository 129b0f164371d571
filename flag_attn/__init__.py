"""Import-name shim: ``import flag_attn`` resolves the SageAttention path to the MI355X build.

Only ``flag_attn.sage_attention`` and the forward pass of ``flag_attn.flash_attention``
(src/flag_attn/__init__.py:48) exist here, and this build's own operators for serving (packed sequences, paged
cache); the other FlagAttention operators are not part of this package.  Metadata strings follow the reference's src/flag_attn/__init__.py:22-25.
"""
from flagattention_amd import (append_to_cache, backend_info, copy_pages, device, flash_attention, flash_attention_varlen,
                               paged_attention, vendor, vendor_name)
from . import sage_attention  # noqa: F401  (stays a namespace, as in the reference :115-117)
from . import testing  # noqa: F401

__all__ = ["sage_attention", "flash_attention", "flash_attention_varlen", "paged_attention", "append_to_cache", "copy_pages",
           "testing", "device", "vendor", "vendor_name", "backend_info"]
