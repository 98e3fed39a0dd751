from . import bwd, fwd, moe, quant  # noqa: F401
