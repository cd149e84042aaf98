"""MI355X (gfx950) PRIME moment attention.

Drop-in host API mirroring the reference package ``prime_moment_attention``
(PrimeMomentAttention, chunked_prime_ssd_core, ChunkedPrimeSSD,
PrimeMomentCache, PrimeConfig / PrimeForCausalLM,
ChunkedGatedDeltaPrimeAttention, PrimeSelectiveMomentAttention) over the HIP library
libprime_mi355x.so; beside it the gated linear recurrence, dropout with the residual
add, and sampled tokens.
"""
from .attention import PrimeMomentAttention
from .cache import PrimeMomentCache
from .chunked_delta_prime import ChunkedGatedDeltaPrimeAttention
from .chunked_ssd import ChunkedPrimeSSD, chunked_prime_ssd_core
from .dropout import dropout_add, dropout_rng
from .gated_recurrence import GatedLinearRecurrence, gated_recurrence
from .model import GreedyDecoder, PrimeConfig, PrimeForCausalLM, SamplingDecoder, prime_125m_config
from .sampling import sample_tokens
from .selective import PrimeSelectiveMomentAttention

__version__ = "0.1.0"

__all__ = ["PrimeMomentAttention", "PrimeMomentCache", "ChunkedPrimeSSD", "chunked_prime_ssd_core",
           "PrimeConfig", "PrimeForCausalLM", "GreedyDecoder", "SamplingDecoder", "prime_125m_config",
           "ChunkedGatedDeltaPrimeAttention", "PrimeSelectiveMomentAttention",
           "GatedLinearRecurrence", "gated_recurrence", "dropout_add", "dropout_rng", "sample_tokens"]
