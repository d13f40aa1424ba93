from .adapters import EncoderAdapters, StepAdapters
from .attention import ConformerAttention, PositionalEncoding
from .cache import ModelCache, StreamingState
from .encoder import ConformerEncoder, ConformerLayer, EncoderStepGraph

__all__ = [
    "EncoderAdapters",
    "StepAdapters",
    "ConformerAttention",
    "PositionalEncoding",
    "ModelCache",
    "StreamingState",
    "ConformerEncoder",
    "ConformerLayer",
    "EncoderStepGraph",
]
