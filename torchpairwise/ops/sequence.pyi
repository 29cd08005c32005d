"""Type stubs of attention and rotary positions: signatures as the registered torch.ops.torchpairwise
schemas give them."""
from typing import Optional, Tuple

from torch import Tensor

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
