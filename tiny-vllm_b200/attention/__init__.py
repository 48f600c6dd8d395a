"""Attention over a paged key-value cache: the part of a decoder layer between the qkv and the output projection."""
from .cuda import copy_pages, decode_attention, prefill_attention, store_kv

__all__ = ["prefill_attention", "decode_attention", "store_kv", "copy_pages"]
