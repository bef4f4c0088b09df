"""torch bindings: Genred, KernelSolve, LazyTensor (Vi, Vj, Pm), generic_* shortcuts, cluster helpers and the sequence
operators (bucket_attention, decay_attention, token_logprobs)."""
from . import cluster  # noqa: F401
from .generic_ops import generic_argkmin, generic_argmin, generic_logsumexp, generic_sum  # noqa: F401
from .generic_red import Genred  # noqa: F401
from .lazytensor import LazyTensor, Pm, Vi, Vj  # noqa: F401
from .operations import KernelSolve  # noqa: F401
from .sequence import (  # noqa: F401
    PositionBuckets, TokenLogprobs, bucket_attention, decay_attention, decay_attention_step, token_logprobs,
)
