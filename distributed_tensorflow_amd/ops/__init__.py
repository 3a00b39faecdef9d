from . import native, reference  # noqa: F401
from .clip import GlobalNormClip  # noqa: F401
from .vocab_head import vocab_head_bwd, vocab_head_fwd  # noqa: F401
