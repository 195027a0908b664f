"""Decoder architecture description: the fields of the reference's ModelConfig (modeling/config.py:8-85)
that the projection / MLP path and its callers read."""

from dataclasses import dataclass


@dataclass(frozen=True)
class ModelConfig:
    hidden_size: int = 4096
    intermediate_size: int = 13568
    vocab_size: int = 185600
    num_hidden_layers: int = 40
    num_attention_heads: int = 32
    num_key_value_heads: int = 1
    head_dim: int = 128
    partial_rotary_factor: float = 0.5
    rope_theta: float = 1e9
    rms_norm_eps: float = 1e-6
    max_position_embeddings: int = 2097152
    pad_token_id: int = 0
    eos_token_id: int = 1
    attention_bias: bool = True
    embed_scale: float = 1.0            # factor of the token embeddings (1 in the reference, which has no such field)

    def __post_init__(self):
        if self.num_key_value_heads != 1 or self.hidden_size != self.num_attention_heads * self.head_dim:
            raise ValueError("Only MQA with hidden_size = heads * head_dim is supported")
        if self.rotary_dim <= 0 or self.rotary_dim % 2 or self.rotary_dim > self.head_dim:
            raise ValueError("The partial rotary dimension must be positive and even")
        if not self.attention_bias:
            raise ValueError("Unsupported architecture settings")

    @property
    def rotary_dim(self):
        return int(self.head_dim * self.partial_rotary_factor)

    @classmethod
    def tiny(cls):
        return cls(hidden_size=32, intermediate_size=68, vocab_size=97, num_hidden_layers=2,
                   num_attention_heads=4, head_dim=8, pad_token_id=0, eos_token_id=1)

    def parameter_counts(self, rank=256):
        h, i, d, v = self.hidden_size, self.intermediate_size, self.head_dim, self.vocab_size
        decoder = 2 * h * h + 2 * d * h + 3 * i * h + h + 2 * d + 2 * h
        base = self.num_hidden_layers * decoder + 2 * v * h + h
        adapters = self.num_hidden_layers * rank * (9 * h + 3 * i + 2 * d)
        return base, adapters
