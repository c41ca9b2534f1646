"""ecq_b200 -- B200 (sm_100a) implementation of ecq's hot path: interleaved
rANS decode of 4-bit weight symbols fused with per-group dequantisation and
the GEMV that consumes them, behind the reference's Python interface.

Host-side codec:   RANSTable, InterleavedEncodedTile, interleaved_rans_encode,
                   InterleavedRANSEncoder, encode_matrix
GPU decode:        interleaved_rans_decode, InterleavedRANSDecoder,
                   CudaInterleavedRANS, DeviceMatrix.decode
Fused GEMV:        DeviceMatrix.gemv, entropy_coded_matmul, EntropyCodedLinear
Plain 4-bit:       Packed4Matrix (the CACHED store and the HBM-bound control)
4-bit KV cache:    KV4Cache, kv4_extend / kv4_release (block tables and slot
                   maps), kv4_append / kv4_gather, kv4_attention
"""
from .codec import (EncodedMatrix, InterleavedEncodedTile, InterleavedRANSEncoder, RANSTable,  # noqa: F401
                    encode_matrix, interleaved_rans_encode, pack_reference_tiles, choose_tile_cols)

PROB_BITS = 14
PROB_SCALE = 1 << PROB_BITS
RANS_BYTE_L = 1 << 23


# GPU-side modules import torch; they are loaded when one of their names is first used
_LAZY = {
    "device": ("DeviceMatrix", "Packed4Matrix", "device_info"),
    "interleaved": ("interleaved_rans_decode", "InterleavedRANSDecoder", "CudaInterleavedRANS", "verify_interleaved_roundtrip"),
    "ops": ("entropy_coded_matmul", "EntropyCodedLinear", "rans_gemv", "rans_matmul"),
    "strategies": ("SmartDecoder", "DecodeMode", "DecodedWeights"),
    "kv4": ("KV4Cache", "KV4Step", "kv4_pages", "kv4_extend", "kv4_release", "kv4_append", "kv4_gather", "kv4_attention"),
}


def __getattr__(name):
    for module, names in _LAZY.items():
        if name in names:
            from importlib import import_module
            value = globals()[name] = getattr(import_module(f".{module}", __name__), name)
            return value
    raise AttributeError(name)
