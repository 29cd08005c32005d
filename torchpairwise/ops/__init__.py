"""Op bindings (reference: torchpairwise/ops/__init__.py); attention and rotary positions beside them."""
from .cpdist import *  # noqa: F401,F403
from .metrics import *  # noqa: F401,F403
from .sequence import *  # noqa: F401,F403
