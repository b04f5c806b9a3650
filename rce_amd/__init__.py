"""rce_amd -- MI355X (gfx950) GGUF block-quantized matmul path.

The product is the C-ABI library ``rce_amd/lib/librce_qmm.so`` (HIP kernels
in ``rce_amd/csrc``, interface ``include/rce_qmm.h``).  ``rce_amd.qmm`` is the
Python mirror of the reference operator API (``rce-op-qmm``) over that ABI;
``rce_amd.llama`` mirrors the TinyLlama decode runtime (``rce-tinyllama``);
``rce_amd.gguf`` the GGUF file reader (``rce-ingest-gguf``); ``rce_amd.kv`` the
paged 8-bit KV cache and its pages, attention over it and sampling.
"""
from .qmm import (  # noqa: F401
    NOALLOC_SCRATCH_BYTES, Context, DeviceBuffer, GgufDtype, Mode, QmmError, QuantWeight, block_geometry, mm_1d,
    mm_1d_serial, mm_batched, mm_batched_dev, mm_batched_dev_noalloc, moe_ffn_dev, moe_route_dev, moe_router,
    moe_swiglu_dev, MoeRouting, quantize, row_bytes, supports,
)
from .kv import (Heads, KvBatch, KvCache, KvTable, Rope, kv_append_dev, kv_attention_dev,  # noqa: F401,E402
                 kv_attention_sinks_dev, kv_compact_dev, kv_copy_dev, kv_fork_dev, kv_read_dev, kv_release_dev,
                 kv_reserve_dev, qk_norm_rope_dev, sample_dev)
from .llama import TinyLlamaBlock, TinyLlamaConfig, TinyLlamaRuntime, TinyLlamaWeights, load_weights  # noqa: F401,E402
from .gguf import GgufFile, GgufMetadata, GgufTensorInfo, GgufValue, split_experts  # noqa: F401,E402
from .placement import (GpuEnergyMeter, HipQmm, HostQuantWeight, LinearCoeffs, hip_cost_prior,  # noqa: F401,E402
                        pick_priced, qmm_dtype_id)
