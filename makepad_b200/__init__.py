"""makepad_b200: B200-native block-quantised linear operators (libmpq), what runs between them in a decoder layer, and a thin
Python host mirror."""
from .decoder import DecoderLayer, PagedCache  # noqa: F401
from .decoder_ops import KvStep, kv_append, kv_plan, paged_attention, prompt_attention, residual_norm, rotary_frequencies  # noqa: F401
from .quant_linear import (Context, MpqError, Nvfp4Weight, Q4Weight, QuantLinear, load_canonical, load_weight,  # noqa: F401
                           nvfp4_quantize, save_canonical, swiglu)
