"""Weight quantisation helpers (`fni8.quant.core`, `fni8.quant.lowbit`, `fni8.quant.fp4`)."""
from . import core, fp4, lowbit  # noqa: F401
