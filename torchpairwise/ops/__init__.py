"""Op bindings (reference: torchpairwise/ops/__init__.py); attention, rotary positions and the
cache in 4 or 8 bits beside them."""
from .cpdist import *  # noqa: F401,F403
from .metrics import *  # noqa: F401,F403
from .sequence import *  # noqa: F401,F403
