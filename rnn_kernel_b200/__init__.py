"""B200-native FP32 GRU training path with an ``nn.GRU``-compatible surface.

Importing the package needs neither a GPU nor the CUDA library; the library
(``librnn_kernel_b200.so``, built in-tree) is loaded on first use.
"""
from .delta import GatedDelta, GatedDeltaRuleFunction, gated_delta_rule, gated_delta_step
from .gru import (
    GRU,
    GRUFunction,
    MAX_HIDDEN_SIZE,
    from_torch_gru,
    gru_forward_inference,
    is_b200_available,
    is_supported_gru,
)
from .loss import MSELossFunction, mse_loss
from .optim import AdamW
from .train import DataParallelTrainer, GraphedTrainStep, HostBatchPrefetcher, flatten_parameters_

B200GRU = GRU

__all__ = [
    "AdamW",
    "GRU",
    "B200GRU",
    "GRUFunction",
    "MAX_HIDDEN_SIZE",
    "DataParallelTrainer",
    "GraphedTrainStep",
    "GatedDelta",
    "GatedDeltaRuleFunction",
    "HostBatchPrefetcher",
    "flatten_parameters_",
    "from_torch_gru",
    "gated_delta_rule",
    "gated_delta_step",
    "gru_forward_inference",
    "is_b200_available",
    "is_supported_gru",
    "mse_loss",
    "MSELossFunction",
]
