"""B200-native token sampling for miniserve (sm_100a CUDA behind a C ABI).

    from miniserve_b200 import Sampler
    tok = Sampler().sample(logits, temperature=0.7, top_k=50, top_p=0.9, seed=1)
    tokens, probs, status = Sampler().sample_batch(logits_bxv, temperature=T, top_k=K, top_p=P,
                                                   uniforms=U)

The rest of a decode step's hot path lies beside it:

    from miniserve_b200 import append_kv, rope_table      # keys and values into a paged cache, rotated
    from miniserve_b200 import prefix_attention            # attention over the cache, a shared prefix read once
    from miniserve_b200 import Int8Linear                  # projections and LM head in 8-bit integers
"""
from .attention import prefix_attention  # noqa: F401
from .int8 import Int8Linear, int8_matmul, quantize_rows  # noqa: F401
from .kvcache import append_kv, rope_table  # noqa: F401
from .sampler import Sampler, uniform_for_seed  # noqa: F401

__version__ = "0.1.0"
