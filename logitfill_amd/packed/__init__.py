"""Packed Key/Value history and its decode path on MI355X (reference ``logitfill.packed``)."""

from logitfill_amd.packed.cache import LogitFillCache, PackedKVManager
from logitfill_amd.packed.int4 import Int4KVManager, int4_attention, select_pages
from logitfill_amd.packed.prompt import PromptPlan, prompt_attention
from logitfill_amd.packed.rotary import Rotary

__all__ = ["Int4KVManager", "LogitFillCache", "PackedKVManager", "PromptPlan", "Rotary", "int4_attention",
           "prompt_attention", "select_pages"]
