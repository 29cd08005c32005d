"""Type stubs of attention, rotary positions and the cache in 4 or 8 bits: signatures as the registered
torch.ops.torchpairwise schemas give them."""
from typing import Optional, Tuple

from torch import Tensor, dtype as Dtype

def attention(query: Tensor,
              key: Tensor,
              value: Tensor,
              mask: Optional[Tensor] = None,
              *,
              causal: bool = False,
              scale: Optional[float] = None,
              lengths: Optional[Tensor] = None) -> Tensor: ...


def rotary_embedding(x: Tensor,
                     positions: Tensor,
                     frequencies: Tensor,
                     *,
                     interleaved: bool = False,
                     scale: float = 1.0) -> Tensor: ...


def rotary_frequencies(width: int,
                       base: float = 10000.0,
                       *,
                       scaling: str = 'none',
                       factor: float = 1.0,
                       original_length: Optional[int] = None,
                       fast: float = 32.0,
                       slow: float = 1.0,
                       device=None) -> Tuple[Tensor, float]: ...


def quantized_cache(batch: int,
                    heads: int,
                    rows: int,
                    width: int,
                    value_width: Optional[int] = None,
                    *,
                    bits: int = 4,
                    device=None) -> Tuple[Tensor, Tensor, Tensor, Tensor]: ...


def cache_write_(key_codes: Tensor,
                 key_scales: Tensor,
                 value_codes: Tensor,
                 value_scales: Tensor,
                 key: Tensor,
                 value: Tensor,
                 starts: Tensor,
                 *,
                 counts: Optional[Tensor] = None,
                 pages: Optional[Tensor] = None) -> None: ...


def cache_read(key_codes: Tensor,
               key_scales: Tensor,
               value_codes: Tensor,
               value_scales: Tensor,
               *,
               key_width: Optional[int] = None,
               value_width: Optional[int] = None,
               dtype: Optional[Dtype] = None,
               starts: Optional[Tensor] = None,
               rows: Optional[int] = None,
               counts: Optional[Tensor] = None,
               pages: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]: ...


def cache_attention(query: Tensor,
                    key_codes: Tensor,
                    key_scales: Tensor,
                    value_codes: Tensor,
                    value_scales: Tensor,
                    mask: Optional[Tensor] = None,
                    *,
                    causal: bool = False,
                    scale: Optional[float] = None,
                    lengths: Optional[Tensor] = None,
                    pages: Optional[Tensor] = None,
                    value_width: Optional[int] = None) -> Tensor: ...
