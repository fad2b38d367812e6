"""sm_100a kernels behind LITHE's index-resident serving path (API of lithe/kernels).

* ``packed``  9-bit index packing (7 indices per uint64 word), the packed resident bank and
              the whole-adapter decode kernel.
* ``shared``  index-resident per-sample LoRA delta with the decode fused into the
              shrink / expand tiles (one launch per linear).
* ``rotary``  rotary positions with several axes, alone or with the per-head norm of q and k.
* ``int8``    linear on 8-bit integers (scales per token and output channel) with the adapters'
              expand added before the rounding.
* ``layers``  nn.Module wrappers that route each sample of a batch to its own adapter.
"""
from ._launch import device_errors, raise_device_errors
from .int8 import QuantizedRows, int8_linear, quantize_rows, quantize_weight
from .layers import (IndexLoRALinear, Int8Linear, PackedLoRALinear, PerSampleLoRALinear, SharedInputPrep,
                     group_shared_inputs, wrap_int8, wrap_linears, wrap_packed)
from .packed import (PackedBank, PackedLayout, SlotLoader, decode_packed, flat_indices, pack_adapter,
                     pack_indices, split_decoded, unpack_indices)
from .rotary import qk_norm_rotate, rotate_axes
from .shared import packed_codebook_lora_delta_, shared_codebook_lora_delta, shared_codebook_lora_delta_

__all__ = [
    "IndexLoRALinear", "PackedLoRALinear", "PerSampleLoRALinear", "SharedInputPrep", "group_shared_inputs",
    "wrap_linears", "wrap_packed", "Int8Linear", "wrap_int8",
    "PackedBank", "PackedLayout", "SlotLoader", "decode_packed", "flat_indices", "pack_adapter", "pack_indices",
    "split_decoded", "unpack_indices",
    "shared_codebook_lora_delta", "shared_codebook_lora_delta_", "packed_codebook_lora_delta_",
    "QuantizedRows", "quantize_rows", "quantize_weight", "int8_linear",
    "rotate_axes", "qk_norm_rotate",
    "device_errors", "raise_device_errors",
]
