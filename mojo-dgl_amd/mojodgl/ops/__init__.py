"""Operators (the `dgl.ops` names)."""

from . import edge_softmax as _es_mod
from . import gather_mm as _gm_mod
from . import norm as _norm_mod
from . import route as _route_mod
from . import scan as _scan_mod
from . import sddmm as _sddmm_mod
from . import segment as _seg_mod
from . import spmm as _spmm_mod

# The star imports shadow the `edge_softmax` and `gather_mm` module names with
# the same-named functions, as upstream's package does.
from .edge_softmax import *  # noqa: F401,F403
from .gather_mm import *  # noqa: F401,F403
from .norm import *  # noqa: F401,F403
from .route import *  # noqa: F401,F403
from .scan import *  # noqa: F401,F403
from .sddmm import *  # noqa: F401,F403
from .segment import *  # noqa: F401,F403
from .spmm import *  # noqa: F401,F403

__all__ = (
    _es_mod.__all__
    + _gm_mod.__all__
    + _sddmm_mod.__all__
    + _seg_mod.__all__
    + _spmm_mod.__all__
)

# Operators over packed rows without a counterpart in the reference: `__all__`
# above keeps to its names.
row_ops = _norm_mod.__all__ + _scan_mod.__all__ + _route_mod.__all__
