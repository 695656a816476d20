from .shard import ShardSGD, ShardAdam, ShardAdamW, ShardGNMTAdam
from .muon import ShardMuon, orthogonalize

__all__ = ["ShardSGD", "ShardAdam", "ShardAdamW", "ShardGNMTAdam", "ShardMuon", "orthogonalize"]
