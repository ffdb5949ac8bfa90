from .conv import ConcatConv2d, ShiftedConv2d
from .fp8 import Fp8BlockLinear, block_scaled_linear
from .kvcache import Fp8KVCache
from .linear import ConcatLinear, ShiftedLinear
from .lowrank import AccumBranchHook, LowRankBranch, add_low_rank_branches
from .sdpa import ScaleDotProductAttention

__all__ = ["LowRankBranch", "AccumBranchHook", "ConcatLinear", "ShiftedLinear", "ConcatConv2d", "ShiftedConv2d",
           "Fp8BlockLinear", "Fp8KVCache", "ScaleDotProductAttention", "block_scaled_linear"]
