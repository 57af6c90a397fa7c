"""Denoising-step execution over the quantized data plane: cross-step block
reuse (shadowinfer/execution/step_reuse.py), the confidence-aware unmasking
round (shadowinfer/execution/block_decoding.py) and a Llama-shaped diffusion
LM step on packed KV + INT8 FFN, and the rotary positions of a decode step."""

from .denoise import DiffusionLlamaShape, PackedDiffusionLlama, mask_tokens
from .rotary import RotaryEmbedding, RotaryScaling
from .schedule import ScheduleDecision, argmax_confidence, schedule_round
from .step_reuse import LayerRecord, StepReuseConfig, StepReuseState

__all__ = [
    "DiffusionLlamaShape",
    "LayerRecord",
    "PackedDiffusionLlama",
    "RotaryEmbedding",
    "RotaryScaling",
    "ScheduleDecision",
    "StepReuseConfig",
    "StepReuseState",
    "argmax_confidence",
    "mask_tokens",
    "schedule_round",
]
