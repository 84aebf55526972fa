"""The decoder in the clear, on the device: the operators of the model that
the encrypted programs evaluate, in bf16 and fp16, with their gradients.

What the encrypted prefill computes on ciphertexts runs here on plain tensors:
for scoring decrypted hidden states, for generating after an encrypted prompt,
and for adapting weights before they are encoded.  (16 bits are too coarse to
check a decrypted result with; that is done in fp64, and so is calibration,
which needs every layer's intermediates.)  Rotary positions, attention and the
vocabulary loss are hand-written gfx950 kernels (``libclear_mi355x.so``) on
torch tensors; ``ClearDecoder`` runs them together, with torch's products and
norms between them.
"""

from .attention import attention, attention_backward, attention_forward
from .decoder import ClearCache, ClearDecoder, rms_norm
from .loss import (
    linear_cross_entropy,
    linear_cross_entropy_backward,
    linear_cross_entropy_forward,
)
from .rope import RopeTable, WavelengthScaling, apply_rope, rope, rope_backward

__all__ = [
    "ClearCache", "ClearDecoder", "RopeTable", "WavelengthScaling", "apply_rope", "attention",
    "attention_backward", "attention_forward", "linear_cross_entropy",
    "linear_cross_entropy_backward", "linear_cross_entropy_forward", "rms_norm", "rope",
    "rope_backward",
]
