"""MI355X-native Tucker convolution (TDC hot path) — Python host layer over libtdc_amd.so."""
from ._lib import (LIB_PATH, ConvDesc, TdcError, Tile, TileInfo, conv_desc, lib, model_enumerate, model_evaluate,
                   model_select, set_autotune)

__all__ = ["LIB_PATH", "ConvDesc", "TdcError", "Tile", "TileInfo", "conv_desc", "lib", "model_enumerate",
           "model_evaluate", "model_select", "set_autotune", "Conv2dPlan", "TKConvOp", "TKConv2dC", "ranks_dict", "partial_tucker2",
           "group_norm_act", "group_norm_act_mx4", "mx4_quantize", "mx4_linear", "mx4_conv1x1", "Mx4Tensor",
           "GroupNormAct", "TuckerBlockMx4",
           "linear_act", "conv1x1_act", "rms_norm", "rms_norm_mx8", "mx8_quantize", "mx8_linear", "mx8_conv1x1", "Mx8Tensor"]


def __getattr__(name):
    # torch-dependent classes are imported lazily so the model API works without torch; once loaded they are plain attributes.
    if name in ("Conv2dPlan", "TKConvOp"):
        from . import conv as module
    elif name in ("TKConv2dC", "ranks_dict", "partial_tucker2"):
        from . import TKConv as module
    elif name in ("group_norm_act", "group_norm_act_mx4", "mx4_quantize", "mx4_linear", "mx4_conv1x1", "Mx4Tensor"):
        from . import channels_last as module
    elif name in ("linear_act", "conv1x1_act", "rms_norm", "rms_norm_mx8", "mx8_quantize", "mx8_linear", "mx8_conv1x1", "Mx8Tensor"):
        from . import pointwise as module
    elif name in ("GroupNormAct", "TuckerBlockMx4"):
        from . import mx4_block as module
    else:
        raise AttributeError(name)
    globals()[name] = value = getattr(module, name)
    return value
