"""Neural-network helpers: `functional.edge_softmax`, as the reference, and
`functional.layer_norm`."""

from . import functional  # noqa: F401
