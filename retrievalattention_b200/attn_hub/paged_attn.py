"""Attention over the paged cache, with the argument list of the other caches' entry points."""
from __future__ import annotations


def paged_decode_attn(query_states, key_states, value_states, layer_idx, paged_cache):
    """query_states ``[batch, 1, heads, 128]``; the step's keys and values are in the pages already (``paged_cache.append``)."""
    return paged_cache.attend(query_states, layer_idx)


def paged_prompt_attn(query_states, key_states, value_states, layer_idx, paged_cache):
    """query_states ``[rows, heads, 128]``, the step's rows of all requests, whose keys and values are in the pages already: causal, over
    all that their requests have cached or the layer's window of it."""
    return paged_cache.prompt(query_states, layer_idx)
