"""MI355X (gfx950) fused attention for the Supra2-Img Web attention hot path.

The operator itself is HIP code behind the C ABI in include/supra_attn.h
(lib/libsupra_attn.so); this package is its Python binding:

- `_lib`      ctypes declarations of every exported symbol, the argument structs, status codes
- `device`    device buffers / stream / events over the C ABI helpers
- `workloads` seeded inputs for the DiT, T5 and VAE call shapes
- `runner`    stage a workload on the device and launch it
"""

from ._lib import (  # noqa: F401
    AttnArgs, KvAttnArgs, KvCache, KvRowsArgs, KvSeqs, LinearArgs, QkRopeArgs, SaError, attention, bucket_lut, kernel_name, kv_attention,
    kv_attention_shape, kv_attention_workspace_bytes, kv_cache_bytes, kv_read, kv_write, linear, load, qk_norm_rope, workspace_bytes)

__all__ = ["AttnArgs", "KvAttnArgs", "KvCache", "KvRowsArgs", "KvSeqs", "LinearArgs", "QkRopeArgs", "SaError", "attention", "bucket_lut",
           "kernel_name", "kv_attention", "kv_attention_shape", "kv_attention_workspace_bytes", "kv_cache_bytes", "kv_read", "kv_write",
           "linear", "load", "qk_norm_rope", "workspace_bytes"]
