"""Attention, rotary positions and a cache of keys and values in 4 or 8 bits (not in the reference)."""
import torch

from torchpairwise_amd.ops.cache import quantized_cache  # noqa: F401
from torchpairwise_amd.ops.rotary import rotary_frequencies  # noqa: F401

attention = torch.ops.torchpairwise.attention
rotary_embedding = torch.ops.torchpairwise.rotary_embedding
cache_write_ = torch.ops.torchpairwise.cache_write_
cache_read = torch.ops.torchpairwise.cache_read
cache_attention = torch.ops.torchpairwise.cache_attention
