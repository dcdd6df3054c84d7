"""B200-native token sampling for miniserve (sm_100a CUDA behind a C ABI).

    from miniserve_b200 import Sampler
    tok = Sampler().sample(logits, temperature=0.7, top_k=50, top_p=0.9, seed=1)
    tokens, probs, status = Sampler().sample_batch(logits_bxv, temperature=T, top_k=K, top_p=P,
                                                   uniforms=U)

The rest of a decode step's hot path lies beside it:

    from miniserve_b200 import append_kv, rope_table      # keys and values into a paged cache, rotated
    from miniserve_b200 import prefix_attention            # attention over the cache, a shared prefix read once
    from miniserve_b200 import Int8Linear                  # projections and LM head in 8-bit integers

and the parts of a drafted-token step over a cache held in 4 bits:

    from miniserve_b200 import KvCache4, append_kv4, read_kv4   # quantised as it is written, and read back
    from miniserve_b200 import attention_kv4                    # one or several tokens a row over it
    from miniserve_b200 import verify_drafts                    # drafted tokens against the target's logits
"""
from .attention import prefix_attention  # noqa: F401
from .attention4 import attention_kv4  # noqa: F401
from .int8 import Int8Linear, int8_matmul, quantize_rows  # noqa: F401
from .kvcache import append_kv, rope_table  # noqa: F401
from .kvcache4 import KvCache4, append_kv4, read_kv4  # noqa: F401
from .sampler import Sampler, uniform_for_seed  # noqa: F401
from .verify import verify_drafts  # noqa: F401

__version__ = "0.1.0"
