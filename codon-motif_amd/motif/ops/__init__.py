'''Public op surface, named as the reference's motif/ops/__init__.py:1-10.

`HAS_TRITON` keeps its name because the layers read it as "the fast backend
is present"; here it is True when libmotif_hip.so loaded and a ROCm device is
visible.
'''
from . import _lib
from .rms_norm import RMSNorm, GatedRMSNorm
from .swiglu import SwiGLU
from .chord_attention import apply_chord_attention, apply_chord_attention_varlen
from .kv4 import (KV4Slab, chord_attention_kv4, chord_decode_kv4_cursor, chord_decode_kv4_workspace, chord_kv4_prep,
                  kv4_alloc, kv4_append, kv4_read)
from .gated_deltanet import (
    recurrent_gated_delta_rule,
    chunk_gated_delta_rule,
    chunk_gated_delta_rule_triton,
    chunk_gated_delta_rule_varlen,
    chunk_gated_delta_rule_gated_norm,
    gdn_prefill_fused,
)
from .short_conv import short_conv_silu, short_conv_silu_multi, short_conv_silu_varlen
from .attn_res import apply_block_attn_res, attn_res_read, attn_res_read_norms
from .gdn_decode import gdn_decode_fused
from .linear_rows import cat_weights, linear_rows, project, rows_eligible

HAS_TRITON = _lib.available()
HAS_HIP = HAS_TRITON

__all__ = [
    'RMSNorm', 'GatedRMSNorm', 'SwiGLU',
    'apply_chord_attention', 'apply_chord_attention_varlen',
    'KV4Slab', 'kv4_alloc', 'kv4_append', 'kv4_read', 'chord_attention_kv4', 'chord_decode_kv4_cursor',
    'chord_decode_kv4_workspace', 'chord_kv4_prep',
    'recurrent_gated_delta_rule', 'chunk_gated_delta_rule',
    'chunk_gated_delta_rule_triton', 'chunk_gated_delta_rule_varlen', 'chunk_gated_delta_rule_gated_norm',
    'gdn_prefill_fused',
    'short_conv_silu', 'short_conv_silu_multi', 'short_conv_silu_varlen',
    'apply_block_attn_res', 'attn_res_read', 'attn_res_read_norms', 'gdn_decode_fused',
    'cat_weights', 'linear_rows', 'project', 'rows_eligible',
    'HAS_TRITON', 'HAS_HIP',
]
