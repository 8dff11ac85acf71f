from .arena import ParamArena, SGD, Adam, Muon  # noqa: F401
from . import layers  # noqa: F401
