"""Attention and rotary positions (not in the reference)."""
import torch

from torchpairwise_amd.ops.rotary import rotary_frequencies  # noqa: F401

attention = torch.ops.torchpairwise.attention
rotary_embedding = torch.ops.torchpairwise.rotary_embedding
