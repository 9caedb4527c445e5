"""Ops of the GPT stage program: hand-written sm_100a kernels on CUDA, PyTorch references on CPU."""
from . import native, raw  # noqa: F401
from .functional import *  # noqa: F401,F403
from .functional import gemm, colsum  # noqa: F401
from .packed_attention import PackedLayout, flash_attention_packed  # noqa: F401
from .token_losses import TokenScores, token_logprobs, topk_distillation_loss  # noqa: F401
