"""`nn.functional.edge_softmax` is `ops.edge_softmax` itself, and `layer_norm`
`ops.layer_norm`."""

from ...ops import edge_softmax, layer_norm  # noqa: F401
