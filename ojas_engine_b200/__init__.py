"""ojas_engine_b200 — the quantized-matmul hot path of ojas-engine, rebuilt for B200 (sm_100a), with the rotary positions, paged
cache and attention between a layer's projections.

The product is ``libojas_b200.so`` (CUDA kernels behind the C ABI of ``include/ojas_b200.h``);
this package is its host-side mirror of the engine's backend interface.  There is no CPU
fallback: compute calls need the built library and a B200.
"""
from .runtime import (ACCUM, BF16, BIAS, F16, F32, GEMV_MAX_M, IQ4_NL, IQ4_XS, PLAIN, Q4_K, Q5_K, Q6_K, Q8_0, ROPE_HALF, ROPE_INTERLEAVED, B200Gpu, Buf, Enc,
                      ExpertCache, KvCache, Lin, OjasB200Error, Rope, Seqs, encode, raw_bytes, repack_host, repacked_bytes, rope_frequencies)

__all__ = ["ACCUM", "BF16", "BIAS", "F16", "F32", "GEMV_MAX_M", "IQ4_NL", "IQ4_XS", "PLAIN", "Q4_K", "Q5_K", "Q6_K", "Q8_0", "ROPE_HALF", "ROPE_INTERLEAVED", "B200Gpu", "Buf",
           "Enc", "ExpertCache", "KvCache", "Lin", "OjasB200Error", "Rope", "Seqs", "encode", "raw_bytes", "repack_host", "repacked_bytes", "rope_frequencies"]
