"""MI355X-native (gfx950) memory-efficient CLIP / LiT contrastive loss.

Drop-in replacement for b0nce/MemoryEfficientCLIP's ``clip_loss`` and
``lit_loss`` modules: the same ``nn.Module`` and ``autograd.Function`` classes,
backed by hand-written HIP kernels in ``lib/libmec.so`` (C ABI:
``include/mec.h``).  Beside it, the vocabulary side of the text tower: scaled
token embedding, token log probabilities and distillation from a teacher's top
logits.
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
    "scaled_embedding",
    "token_log_probs",
]
