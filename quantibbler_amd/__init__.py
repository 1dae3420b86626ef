"""quantibbler_amd -- MI355X (gfx950) implementation of quantibbler-kernels'
two hot paths behind the reference's own API surface:

* the binary latent-factor linear (decode GEMV, prefill GEMM) over 1-bit
  sign matrices: ``FactorLayer`` / ``FactorSet`` and the packed products of
  ``kernels`` (the ``quantibbler_kernels`` PyO3 names);
* SageAttention: ``GpuContext.attention_sage`` (the reference's [SA] s4
  scheme) and ``GpuContext.attention_sage_blk_dev`` (block-scaled INT8 Q/K,
  fp16 P.V).

Beside them, for serving: a KV cache in 8 or 4 bits and batched attention
over it behind a shared prefix (``KvCache``), heads normed and rotated
(``Rope``, ``gpu.rotate_heads_dev``), verification of drafted tokens
(``gpu.verify_drafts_dev``) and log probabilities (``gpu.logprobs_dev``).

All compute runs in libqbk.so (hand-written HIP, C ABI in include/qbk.h).
"""
from ._lib import DeviceError, InitError, KernelError, load as _load_lib  # noqa: F401
from .gpu import (AttentionShape, DecoderBlock, FactorLayer, FactorSet, GpuContext,  # noqa: F401
                  KvCache, LmHead, Rope, SageDecodeState, gpu_available)

_load_lib()

__version__ = "0.1.0"
