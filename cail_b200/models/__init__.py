"""Models used by the benchmarks."""
from .gpt2 import GPT2, GPT2Config, KVCache

__all__ = ["GPT2", "GPT2Config", "KVCache"]
