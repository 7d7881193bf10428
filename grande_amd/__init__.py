"""grande_amd: an MI355X-native engine for omg's decision path.

One block-causal pass over a shared state prefix plus isolated question
branches, read out at the answer positions, on hand-written gfx950 HIP
kernels behind the C ABI in include/omg_hip.h (libomg_hip.so).
"""
from ._lib import (ELEM_BF16, ELEM_F16, ELEM_F32, ROPE_HALF, ROPE_HEAD_HALF, ROPE_INTERLEAVED, OmgError)
from .engine import (BranchOutput, BranchTokens, DeviceWeight, Engine, EngineBuilder, Group, GroupOutput, KvSource,
                     PagedBatch, PagedKv, PointerHead, PrefixSource, Role, Want, pack, sample, sample_workspace,
                     state_check, state_key)
from .model import (BASELINE_CONFIGS, F16, GEMMA4_CONFIGS, LABEL_IDS, Q4, Q8, QTensor, Weights, config_json,
                    export_dir, gemma4_config_json, quantize)

__all__ = [
    "BASELINE_CONFIGS", "BranchOutput", "BranchTokens", "DeviceWeight", "ELEM_BF16", "ELEM_F16", "ELEM_F32", "Engine",
    "EngineBuilder", "F16", "Group", "GroupOutput", "KvSource", "LABEL_IDS", "OmgError", "PagedBatch", "PagedKv",
    "PointerHead", "PrefixSource", "Q4", "Q8", "QTensor", "ROPE_HALF", "ROPE_HEAD_HALF", "ROPE_INTERLEAVED", "Role",
    "Want", "Weights", "config_json", "export_dir", "gemma4_config_json", "pack", "quantize", "sample",
    "sample_workspace", "state_check", "state_key",
]
