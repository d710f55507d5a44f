"""Model zoo: the MLP and the GPT-2 / Llama-shaped decoder transformer."""

from .generation import GenerationCache, GenerationOutput, generate
from .mlp import MLP, MLPBlock, build_activation
from .transformer import ParallelPlan, TensorParallelAttention, TinyTransformer, TransformerBlock, build_reference_linear

__all__ = [
    "GenerationCache",
    "GenerationOutput",
    "MLP",
    "MLPBlock",
    "ParallelPlan",
    "TensorParallelAttention",
    "TinyTransformer",
    "TransformerBlock",
    "build_activation",
    "build_reference_linear",
    "generate",
]
