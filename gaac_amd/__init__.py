"""gaac_amd: the GAAC compressed-KV decode path (lossless BF16 KV codec, block encoder, fused split-K decode attention,
slot cache) for AMD MI355X, with the Python surface of the reference's `gaac` package; beside it a slot cache in 4 bits with its attention, and the steps of a decode
loop before and behind: norms and rotation of queries and keys, sampling, log probabilities; and
its layers on weights in 8 bits: norm, projections, gated block."""
from .codec import Codec, Page
from .encoder import TileEncoder
from .kernel import attention, choose_nsplit
from .kv_cache import CompressedKVCache
from .calibration import BaseCollector
from .fp4_cache import FP4KVCache
from .rope import qk_norm_rope
from .sampling import sample, token_logprobs, LogProbs
from .fp8 import FP8Rows, FP8Weight, quantize_fp8, rms_norm_fp8, fp8_linear, fp8_gated

__all__ = ["Codec", "Page", "TileEncoder", "attention", "choose_nsplit", "CompressedKVCache", "BaseCollector", "FP4KVCache", "qk_norm_rope", "sample", "token_logprobs", "LogProbs",
           "FP8Rows", "FP8Weight", "quantize_fp8", "rms_norm_fp8", "fp8_linear", "fp8_gated"]
