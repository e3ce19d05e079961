"""granulelayer_amd: MI355X (gfx950) sparse projection -> activation -> pool layer.

Public API mirrors sparse_pooling/__init__.py (the reference package) for the Mode-A hot path:
``SparsePoolingLayer``, ``PoolingConfig``, ``LevelSpec``, ``PhysicalPlan``, ``SparseLayout``,
``init_parameters``, ``CoverTopK16Layer`` (sparse_pooling/cover_topk16.py) and ``FusedAdamW``
(sparse_pooling/optim.py).  The compute runs in the HIP
library granulelayer_amd/lib/libgranulelayer_amd.so through its C ABI
(include/granulelayer_amd.h).

Beside them, without a counterpart in the reference: ``DenseProjection`` / ``dense_projection`` (a dense
product with bias, activation and residual in its epilogue) and ``pack_activation`` /
``PackedActivation`` (activations kept in 8 bits, also ``activation_checkpoint="int8"`` of the layers),
``LayerNorm`` / ``layer_norm``, and ``DenseCrossEntropy`` / ``dense_cross_entropy`` (the loss of a dense head over
many classes, without its logits).
"""
from .activations8 import PackedActivation, pack_activation
from .config import LevelSpec, PhysicalPlan, PoolingConfig
from .cover_topk16 import CoverTopK16Layer
from .cross_entropy import DenseCrossEntropy, dense_cross_entropy
from .dense import DenseProjection, dense_projection
from .layer import SparsePoolingLayer
from .layout import SparseLayout, init_parameters
from .norm import LayerNorm, layer_norm
from .optim import FusedAdamW

__all__ = ["SparsePoolingLayer", "PoolingConfig", "LevelSpec", "PhysicalPlan", "SparseLayout", "init_parameters",
           "CoverTopK16Layer", "FusedAdamW", "DenseProjection", "dense_projection", "PackedActivation", "pack_activation",
           "LayerNorm", "layer_norm", "DenseCrossEntropy", "dense_cross_entropy"]
