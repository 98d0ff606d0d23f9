"""B200 (sm_100a) build of Zepp's expert-parallel MoE layer.

Importing this package does not touch the GPU; the CUDA library (zepp_b200/lib/libzepp_b200.so) is
loaded on first use and its absence is an error: there is no CPU path.
"""
from . import config as _config
from . import layer as _layer
from . import ops as _ops

SHAPES = _config.SHAPES
ModelShape = _config.ModelShape
EPMoEConfig = _config.EPMoEConfig
tokens_per_rank = _config.tokens_per_rank
EPMoE = _layer.EPMoE
Marks = _layer.Marks
activation = _layer.activation
token_buckets = _layer.token_buckets
route_topk = _ops.route_topk
sort_tokens = _ops.sort_tokens
unsort_tokens = _ops.unsort_tokens
SortPlan = _ops.SortPlan
expert_ffn = _ops.expert_ffn
grad_norm = _ops.grad_norm
clip_grad_norm_ = _ops.clip_grad_norm_
check_waits = _ops.check_waits

__all__ = ["SHAPES", "ModelShape", "EPMoEConfig", "tokens_per_rank", "EPMoE", "Marks", "activation", "token_buckets",
           "route_topk", "sort_tokens", "unsort_tokens", "SortPlan", "expert_ffn", "grad_norm", "clip_grad_norm_", "check_waits"]
__version__ = "0.1.0"
