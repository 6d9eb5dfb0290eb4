"""MI355X-native single-query (decoding) attention: MHA / GQA / MQA / MLA over packed variable-length KV."""
__version__ = "0.1.0"

from .interface import (decoding_attn_fwd, decoding_attn_paged_fwd, decoding_attn_paged_shared_prefix_fwd,  # noqa: F401
                        decoding_attn_shared_prefix_fwd, fwd, kv_cache_append, kv_cache_read, pack_int4, quantize_int4_per_group, quantize_int4_per_token, quantize_int8_per_group,
                        quantize_int8_per_token)
