"""Host side of the grouped-query operators (head dimension 128): a decoder layer's steps around `forward`.

    rope            rotary positions with one to four axes (time, height, width ...)
    cache_append    new tokens' keys and values into the paged 8-bit cache, one scale for each page and head
    decode          attention of the newest tokens over that cache
    cross_forward   attention to an encoder's states of another length; cross_backward its gradients

Conventions as in `mla.py`: outputs and workspaces are allocated with torch unless given, work is launched on the current stream of the
inputs' device without synchronising, sizes, dtypes and devices are checked (`ValueError`), what the kernels do not support raises
`RuntimeError`.  Activations are bf16 and contiguous; where noted, the heads of a token are contiguous and tokens may lie further apart (parts of a
fused projection).  The work behind each signature is in `csrc/bindings/torch_bridge.cpp`.  No CPU fallback exists.
"""

from __future__ import annotations

import torch

from .library import extension, library
from .mla import device_status, flash_forward as forward  # noqa: F401 (the causal forward, beside its relatives)

DECODE_MAX_TOKENS = 64


def rope(query, key, positions, sections, theta=10000.0, restart=False, inverse=False, query_out=None, key_out=None):
    """Rotary embedding with several position axes (`dscuda_flash_rope`) -> (query_out, key_out).
    query [..., Hq, W], key [..., Hk, W] (either may be None), W = 64 or 128, tokens may lie apart; positions int32 [axes, ...] with one
    number for each axis and token.  Element i turns with element i + W/2; sections[a] of the W/2 pairs belong to axis a, in
    order.  The angle of pair i is position * theta^(-2i/W), with `restart` theta^(-j / sections[a]) for the j-th pair of its
    section.  `inverse` turns back: given the gradients of the outputs it returns those of the inputs.  Outputs are new
    contiguous tensors unless given; they may be the inputs themselves."""
    return extension().flash_rope(query, key, positions, sections, theta, restart, inverse, query_out, key_out)


def cache_append(key_cache, value_cache, key_scale, value_scale, key, value, block_table, start_positions=None, token_counts=None):
    """Writes new tokens into the paged 8-bit cache in place (`dscuda_flash_cache_append`).
    key_cache, value_cache [blocks, Hkv, page, 128] int8 or float8_e4m3fn (page a multiple of 16), key_scale, value_scale [blocks, Hkv]
    fp32; key, value [B, T, Hkv, 128], tokens may lie apart; block_table [B, pages] int32; start_positions / token_counts [B] int32 or None
    (0 / all T tokens).  Token t of sequence b lands at position start_positions[b] + t.
    A page's scale covers what the page holds: where new values need a larger one, the page's older codes are rounded again.  What
    a sequence held at and behind its first new position is given up.  A page must not be written twice in one call (two sequences that share it have
    to part before).  Positions and page numbers outside the cache are skipped and raise status 3 (`device_status`); an entry without tokens has none."""
    extension().flash_cache_append(key_cache, value_cache, key_scale, value_scale, key, value, block_table, start_positions, token_counts)


def decode_workspace(batch, tokens, query_heads, key_value_heads, device="cuda"):
    """Workspace of `decode` for calls of these sizes.  Calls that may run at the same time need one each."""
    return torch.empty(library("flash_attention").dscuda_flash_decode_workspace_bytes(batch, tokens, query_heads, key_value_heads), device=device,
                       dtype=torch.uint8)


def decode(query, key_cache, value_cache, key_scale, value_scale, block_table, cache_lengths, scale, workspace=None, output=None, lse=None):
    """Attention of the newest T tokens over the 8-bit cache (`dscuda_flash_decode`), T at most 64.
    query [B, T, Hq, 128]; cache and block_table as for `cache_append`; cache_lengths [B] int32, the new tokens included: token t sees the
    first cache_lengths[b] - T + 1 + t positions -> (output [B, T, Hq, 128], lse [B, Hq, T] fp32).  A token that sees none gets zeros and -inf.
    Page numbers outside the cache are read as page 0 and raise status 3.  The width of block_table (what it can hold, not the lengths) picks how the work is cut: trimmed to
    the longest sequence it is faster for short ones, and another width may change the last bits."""
    return extension().flash_decode(query, key_cache, value_cache, key_scale, value_scale, block_table, cache_lengths, scale, workspace, output, lse)


def cross_forward_workspace(batch, query_length, key_length, query_heads, key_value_heads, device="cuda"):
    lib = library("flash_attention")
    return torch.empty(lib.dscuda_flash_cross_forward_workspace_bytes(batch, query_length, key_length, query_heads, key_value_heads), device=device,
                       dtype=torch.uint8)


def cross_forward(query, key, value, scale, key_lengths=None, workspace=None, output=None, lse=None):
    """Attention to an encoder's states (`dscuda_flash_cross_forward`): no causal mask, Hq / Hkv at most 64.
    query [B, Tq, Hq, 128], key, value [B, Tk, Hkv, 128], key_lengths [B] int32 or None (all Tk): every query sees the first
    key_lengths[b] keys -> (output [B, Tq, Hq, 128], lse [B, Hq, Tq] fp32).  An entry without keys gets zeros and -inf; what lies behind
    a length is not used, NaN included.  Sizes pick how the work is cut: another padding Tk may change the last bits."""
    return extension().flash_cross_forward(query, key, value, scale, key_lengths, workspace, output, lse)


def cross_backward_workspace(batch, query_length, key_length, query_heads, key_value_heads, device="cuda"):
    lib = library("flash_attention")
    return torch.empty(lib.dscuda_flash_cross_backward_workspace_bytes(batch, query_length, key_length, query_heads, key_value_heads), device=device,
                       dtype=torch.uint8)


def cross_backward(dout, output, lse, query, key, value, scale, key_lengths=None, workspace=None, grads=None):
    """Gradients of `cross_forward` (`dscuda_flash_cross_backward`) from its output and lse -> (dquery, dkey, dvalue).
    Keys behind an entry's length get zeros, as do the queries and the key of an entry with a single key.  The same bits from call to call."""
    return extension().flash_cross_backward(dout, output, lse, query, key, value, scale, key_lengths, workspace, grads)
