from .palimpsa import DecodeGraph, chunk_palimpsa, decode_step, fused_recurrent_palimpsa, palimpsa_ref
from .ssm import chunk_ssm, ssm_step

__all__ = ["palimpsa_ref", "chunk_palimpsa", "fused_recurrent_palimpsa", "decode_step", "DecodeGraph", "chunk_ssm", "ssm_step"]
