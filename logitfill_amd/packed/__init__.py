"""Packed Key/Value history and its decode path on MI355X (reference ``logitfill.packed``)."""

from logitfill_amd.packed.cache import LogitFillCache, PackedKVManager
from logitfill_amd.packed.int4 import Int4KVManager, int4_attention, select_pages

__all__ = ["Int4KVManager", "LogitFillCache", "PackedKVManager", "int4_attention", "select_pages"]
