"""MI355X-native LSTM forward + BPTT (gfx950 HIP kernels behind a C ABI).

`LstmCore` drives the device-resident core (`include/flashlstm/lstm_core.h`) from torch tensors;
the drop-in `flashlstm` Python package of the streaming surface lives in `flashlstm_poc_amd/python`.
"""
from .core import LstmCore, load_library, library_path, LibraryMissing, add_flashlstm_to_path
from .stack import LstmStack, StackedLSTM
from .lm_ops import (LayerNorm, decay_attention, decay_attention_backward, decay_attention_forward, decay_attention_step,
                     distillation_backward, distillation_forward, distillation_loss, distillation_train, layer_norm, layer_norm_backward,
                     layer_norm_forward)

__all__ = ["LstmCore", "LstmStack", "StackedLSTM", "load_library", "library_path", "LibraryMissing", "add_flashlstm_to_path",
           "LayerNorm", "decay_attention", "decay_attention_backward", "decay_attention_forward", "decay_attention_step",
           "distillation_backward", "distillation_forward", "distillation_loss", "distillation_train", "layer_norm", "layer_norm_backward",
           "layer_norm_forward"]
