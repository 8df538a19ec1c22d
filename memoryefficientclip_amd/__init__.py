"""MI355X-native (gfx950) memory-efficient CLIP / LiT contrastive loss.

Drop-in replacement for b0nce/MemoryEfficientCLIP's ``clip_loss`` and
``lit_loss`` modules: the same ``nn.Module`` and ``autograd.Function`` classes,
backed by hand-written HIP kernels in ``lib/libmec.so`` (C ABI:
``include/mec.h``).  Beside it, the vocabulary side of the text tower: scaled
token embedding, token log probabilities and distillation from a teacher's top
logits; and the towers' attention, with the rotation of its queries and keys.
"""
from .clip_loss import (
    MemoryEfficientCLIPLoss,
    MemoryEfficientCLIPLossNormed,
    StableMemoryEfficientCLIPLoss,
    StableMemoryEfficientCLIPLossNormed,
)
from .distill_loss import TopKDistillationLoss
from .lit_loss import (
    MemoryEfficientLiTLoss,
    MemoryEfficientLiTLossNormed,
    StableMemoryEfficientLiTLoss,
    StableMemoryEfficientLiTLossNormed,
)
from .token_embedding import ScaledTokenEmbedding, scaled_embedding
from .token_scores import TokenScores, token_log_probs
from .tower_attention import attention
from .tower_rotary import norm_rotary

__version__ = "0.1.0"

__all__ = [
    "MemoryEfficientCLIPLoss",
    "MemoryEfficientCLIPLossNormed",
    "StableMemoryEfficientCLIPLoss",
    "StableMemoryEfficientCLIPLossNormed",
    "MemoryEfficientLiTLoss",
    "MemoryEfficientLiTLossNormed",
    "StableMemoryEfficientLiTLoss",
    "StableMemoryEfficientLiTLossNormed",
    "ScaledTokenEmbedding",
    "TokenScores",
    "TopKDistillationLoss",
    "attention",
    "norm_rotary",
    "scaled_embedding",
    "token_log_probs",
]
