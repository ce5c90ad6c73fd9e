"""B200-native Selective Attention operator (drop-in for the reference's ``selective_attention.kernels``)."""

from .beams import beam_select
from .kernels import (CARRY_M, DTYPES, HAS_KERNELS, HAS_TRITON, HEAD_DIMS, check_inputs, decode_step,
                      selective_attention, selective_attention_forward, selective_attention_reference,
                      selective_logits, supported)
from .layers import add_layer_norm, embedding, layer_norm, linear_cross_entropy
from .paged import append_tokens, begin_pages, begin_tables, move_rows, paged_attention, reorder_rows

__all__ = ["CARRY_M", "DTYPES", "HAS_KERNELS", "HAS_TRITON", "HEAD_DIMS", "check_inputs", "decode_step",
           "selective_attention", "selective_attention_forward", "selective_attention_reference",
           "selective_logits", "supported", "add_layer_norm", "append_tokens", "beam_select", "begin_pages", "begin_tables", "embedding", "layer_norm",
           "linear_cross_entropy", "move_rows",
           "paged_attention", "reorder_rows"]
