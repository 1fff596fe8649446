"""mlx_turboquant_b200: TurboQuant KV-cache compression and attention over the compressed cache
as hand-written sm_100a CUDA kernels, behind the operator surface of alex-rentel/mlx-turboquant.

Public names follow the reference (mlx_turboquant/__init__.py:45-59); ``BlockKVCache`` (8-bit blocks, for the layers that 2 to 4 bits would hurt and
for sliding windows) is new here.
"""

__version__ = "0.1.0"

from .blocks import BlockKVCache  # noqa: F401  (the reference's names are the ones in __all__)
from .cache import TurboQuantKVCache
from .patch import apply_turboquant, enable_turboquant
from .quantizer import QuantizedTensor, TurboQuantMSE, TurboQuantProd

__all__ = [
    "__version__",
    "apply_turboquant",
    "enable_turboquant",
    "TurboQuantKVCache",
    "TurboQuantMSE",
    "TurboQuantProd",
]
