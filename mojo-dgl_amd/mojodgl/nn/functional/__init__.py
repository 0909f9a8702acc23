"""`nn.functional.edge_softmax` is `ops.edge_softmax` itself, `layer_norm` and
`rms_norm` are those of `ops`."""

from ...ops import edge_softmax, layer_norm, rms_norm  # noqa: F401
