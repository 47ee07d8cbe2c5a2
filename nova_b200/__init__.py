"""nova_b200 -- B200-native (sm_100a) kernels for Nova's quantized decode hot path.

Drop-in modules mirroring the reference package ``nova`` (captain-wangrun-cn/Nova):

* ``nova_b200.kvquant``  quantize_int8 / dequantize_int8 (token axis, int8t64)
* ``nova_b200.kvattn``   int8_attn_decode, pack_int8_kv, tail_attend, KVInt8Cache

Beside them, for independent requests in one batch:

* ``nova_b200.paged``    paged int8 cache, append, attention of chunks and single tokens
* ``nova_b200.lora``     low-rank adapters of many requests on a shared projection
* ``nova_b200.logits``   penalties, biases and masks on each request's logits
* ``nova_b200.serving``  a server loop that runs them together

All compute goes through ``libnova_b200.so`` (C ABI in ``include/nova_b200.h``);
there is no CPU or Triton fallback.
"""

from ._lib import available, version

__all__ = ["available", "version"]
