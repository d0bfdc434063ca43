"""MI355X-native streaming KV cache + MTP block-masked attention for
MTP-GLoRA's chunked training.

The package mirrors the reference's operator boundaries for this path:

* ``StreamingKVCacheManager``   - mtp_glora/data_utils/collator.py:178-363
* ``StreamingKVCache``          - the transformers ``Cache`` the adapters call
  (``update`` / ``get_seq_length`` / legacy tuple access)
* ``mtp_attention_forward``     - the ``ALL_ATTENTION_FUNCTIONS`` entry
  (signature of [tf]integrations/flex_attention.py:262)
* ``build_mtp_block_mask``      - the BlockMask of collator.py:290-363
* ``StableSoftCrossEntropy``    - the sampler's soft cross-entropy,
  mtp_glora/core/loss.py:259-330
* ``GatedLoRALinear`` / ``apply_lora_to_model`` - the gated LoRA layers,
  mtp_glora/models/layers/gated_lora.py
* ``qk_norm_rope`` / ``qwen3_attention_forward`` - q_norm, k_norm and
  apply_rotary_pos_emb of Qwen3Attention.forward
  (mtp_glora/models/modeling_qwen3.py:254-305), fused
* ``top_logits``, ``top_logits_cross_entropy``, ``top_logits_loss_and_grad`` - a
  teacher's top logits and the distillation loss from them, beside the soft
  cross-entropy against whole rows
* ``sample_tokens``             - tokens from logits with temperature, top-k,
  top-p and min-p, from given random numbers
* ``adjust_logits``             - penalties for repeated tokens, biases and masks of
  allowed tokens, before sample_tokens
* ``PagedKVCache`` / ``paged_append`` / ``paged_attention`` - decoding: a paged 8-bit
  cache of several sequences, filled with the rotation on the way, and the attention
  of new tokens over it
* ``scaled_embedding`` / ``ScaledEmbedding`` / ``embedding_grad`` - the lookup at
  the start of a chunk and its gradient by sorted tokens

All arithmetic runs in libmtp_glora_amd.so (HIP, gfx950) through the C ABI in
include/mtp_glora_amd.h. The directory name is not a Python identifier; import
it with ``importlib.import_module("mtp-glora_amd")``.
"""
from . import _lib, ops
from .attention import mtp_attention, mtp_attention_forward, register
from .block_mask import MTPBlockMask, build_mtp_block_mask
from .cache import StreamingKVCache
from .distill import (TopLogits, TopLogitsCrossEntropy, top_logits, top_logits_cross_entropy,
                      top_logits_loss_and_grad)
from .embedding import ScaledEmbedding, embedding_grad, scaled_embedding
from .lora import GatedLoRALinear, apply_lora_to_model, gated_lora_linear
from .loss import StableSoftCrossEntropy
from .manager import StreamingKVCacheManager
from .paged import KVPages, PagedKVCache, paged_append, paged_attention
from .rope import qk_norm_rope, qwen3_attention_forward
from .sampling import adjust_logits, sample_tokens

__all__ = [
    "StreamingKVCache", "StreamingKVCacheManager", "MTPBlockMask", "build_mtp_block_mask",
    "mtp_attention", "mtp_attention_forward", "register", "ops", "StableSoftCrossEntropy",
    "qk_norm_rope", "qwen3_attention_forward", "GatedLoRALinear", "apply_lora_to_model", "gated_lora_linear",
    "TopLogits", "TopLogitsCrossEntropy", "top_logits", "top_logits_cross_entropy", "top_logits_loss_and_grad",
    "sample_tokens", "ScaledEmbedding", "scaled_embedding", "embedding_grad", "PagedKVCache", "KVPages",
    "paged_append", "paged_attention", "adjust_logits",
]


def library_path() -> str:
    return str(_lib.LIB_PATH)


def load_library():
    """Load libmtp_glora_amd.so (raises if it is not built)."""
    return _lib.load()
