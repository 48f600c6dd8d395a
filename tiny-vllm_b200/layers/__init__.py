"""Layers of the decoder: quantized linears (reference: ``nanovllm/layers/linear.py``) and attention
(``nanovllm/layers/attention.py``)."""
from .attention import Attention
from .linear import (ColumnParallelLinear, LinearBase, MergedColumnParallelLinear,
                     QKVParallelLinear, ReplicatedLinear, RowParallelLinear)

__all__ = ["Attention", "LinearBase", "ReplicatedLinear", "ColumnParallelLinear",
           "MergedColumnParallelLinear", "QKVParallelLinear", "RowParallelLinear"]
