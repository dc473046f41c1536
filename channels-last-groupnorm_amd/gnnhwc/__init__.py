from .custom_gn import GN_NHWC_Func, GN_NHWC  # noqa: F401  (same exports as src/gnnhwc/__init__.py:1)
from .custom_gn import group_norm_nhwc  # noqa: F401  (traceable functional form; no counterpart in the reference)
from .custom_gn import GN_NCHW_Func  # noqa: F401  (channels-first input; the reference falls back to torch there)
# operators for token streams (no counterparts in the reference)
from .tokens import RMSNorm, Rotary, clip_grad_norm_, clip_gradients, rms_norm, rms_norm_quant, rotary, rotary_frequencies  # noqa: F401
from .attention import window_attention, window_attention_cached  # noqa: F401
from .dropout import Dropout, dropout  # noqa: F401
