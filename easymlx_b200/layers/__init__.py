from .rotary import LongRopeEmbedding, MultiAxisRotaryEmbedding, RotaryEmbedding, get_rope

__all__ = ("LongRopeEmbedding", "MultiAxisRotaryEmbedding", "RotaryEmbedding", "get_rope")
