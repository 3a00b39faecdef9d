from . import native, reference  # noqa: F401
from .clip import GlobalNormClip  # noqa: F401
