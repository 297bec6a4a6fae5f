"""MI355X (gfx950) mixture-of-experts layer behind RustingBrain's MoE interface."""
from .attention import Attention, DecodeAttention, KvCache
from .moe import (BackendUnavailable, Device, DeviceError, InvalidConfig, InvalidInput, Layout, MemoryBudget,
                  MoeCache, MoeConfig, MoeLayer, NetworkError, OutOfMemory, Unsupported, UNROUTED)
from .operators import Muon, ResidualJoin
from .transformer import ParameterCounts, TransformerBuilder, TransformerConfig

__all__ = ["BackendUnavailable", "Device", "DeviceError", "InvalidConfig", "InvalidInput", "Layout",
           "MemoryBudget", "MoeCache", "MoeConfig", "MoeLayer", "NetworkError", "OutOfMemory", "Unsupported",
           "UNROUTED", "Attention", "DecodeAttention", "KvCache", "Muon", "ResidualJoin", "ParameterCounts", "TransformerBuilder", "TransformerConfig"]
