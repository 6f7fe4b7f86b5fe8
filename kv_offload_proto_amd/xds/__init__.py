"""Host side of the data plane, mirroring the reference's xds package
(xds/__init__.py:3-5): pool facade, row allocator, derivation helpers and the
SIEVE coordinator, and the decode-step graph capture; and the operators on
what the rows hold (8-bit rows, attention over the hot buffer)."""
from .graph import DecodeStepGraph
from .xds_attention import RowFormat, dequantize_rows, quantize_rows, reserve_attention, row_format, tree_attention
from .xds_offload import XdsOffloadCoordinator
from .xds_seg_pool import EmsPool, HostSegPool, RowAllocator, Segment, align, compute_ht_size, next_pow2

__all__ = ["DecodeStepGraph", "EmsPool", "HostSegPool", "RowAllocator", "RowFormat", "Segment", "XdsOffloadCoordinator",
           "align", "compute_ht_size", "dequantize_rows", "next_pow2", "quantize_rows", "reserve_attention", "row_format",
           "tree_attention"]
