"""MI355X (gfx950) PRIME moment attention.

Drop-in host API mirroring the reference package ``prime_moment_attention``
(PrimeMomentAttention, chunked_prime_ssd_core, ChunkedPrimeSSD,
PrimeMomentCache, PrimeConfig / PrimeForCausalLM,
ChunkedGatedDeltaPrimeAttention, PrimeSelectiveMomentAttention) over the HIP library
libprime_mi355x.so; beside it the gated linear recurrence, dropout with the residual
add, sampled tokens, and a training step's two ends: the embedding with its gradient, log
probabilities of tokens with theirs, and gradient clipping.
"""
from .attention import PrimeMomentAttention
from .cache import PrimeMomentCache
from .chunked_delta_prime import ChunkedGatedDeltaPrimeAttention
from .chunked_ssd import ChunkedPrimeSSD, chunked_prime_ssd_core
from .dropout import dropout_add, dropout_rng
from .embedding import embedding_lookup
from .gated_recurrence import GatedLinearRecurrence, gated_recurrence
from .grad_clip import clip_grad_norm_, clip_grads_with_norm_, grad_norm
from .logprobs import TokenLogprobs, token_logprobs
from .model import GreedyDecoder, PrimeConfig, PrimeForCausalLM, SamplingDecoder, prime_125m_config
from .sampling import sample_tokens
from .selective import PrimeSelectiveMomentAttention

__version__ = "0.1.0"

__all__ = ["PrimeMomentAttention", "PrimeMomentCache", "ChunkedPrimeSSD", "chunked_prime_ssd_core",
           "PrimeConfig", "PrimeForCausalLM", "GreedyDecoder", "SamplingDecoder", "prime_125m_config",
           "ChunkedGatedDeltaPrimeAttention", "PrimeSelectiveMomentAttention",
           "GatedLinearRecurrence", "gated_recurrence", "dropout_add", "dropout_rng", "sample_tokens",
           "embedding_lookup", "TokenLogprobs", "token_logprobs", "grad_norm", "clip_grad_norm_",
           "clip_grads_with_norm_"]
