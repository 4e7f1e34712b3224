"""MI355X-native stacked LSTM + Linear inference forward, and the operators of residual blocks around a
recurrence that is parallel over time (gfx950 HIP kernels behind a C ABI).

The LSTM's public surface mirrors mantuoluozk/persistent_lstm_hip's `persistent_lstm_hip` package
(persistent_lstm_hip/__init__.py:1-20).
"""
from .api import convert_lstm_module, convert_model_copy, convert_regressor_module, replace_lstm_inplace
from .extension import load_extension
from .gated import GatedScanBlock, GatedScanRegressor
from .model import (
    NativeModuleFallback,
    PersistentLSTM,
    PersistentLSTM4LayerRegressor,
    PersistentLSTMRegressor,
    StandardLSTMRegressor,
)
from .ops import (
    causal_conv,
    causal_conv_step,
    clip_grad_norm,
    dropout_add,
    gated_scan,
    gated_scan_step,
    layer_norm,
    selective_scan,
    selective_scan_step,
)
from .selective import SelectiveScanBlock, SelectiveScanRegressor

__all__ = [
    "PersistentLSTM",
    "PersistentLSTMRegressor",
    "PersistentLSTM4LayerRegressor",
    "NativeModuleFallback",
    "StandardLSTMRegressor",
    "convert_lstm_module",
    "convert_regressor_module",
    "replace_lstm_inplace",
    "convert_model_copy",
    "load_extension",
    "GatedScanBlock",
    "GatedScanRegressor",
    "SelectiveScanBlock",
    "SelectiveScanRegressor",
    "gated_scan",
    "gated_scan_step",
    "layer_norm",
    "dropout_add",
    "causal_conv",
    "causal_conv_step",
    "selective_scan",
    "selective_scan_step",
    "clip_grad_norm",
]
