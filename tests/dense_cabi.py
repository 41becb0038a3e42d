"""The argument structures of the dense linear layer's and layer norm's C entry points, as a ctypes host packs them."""

import struct

from conftest import wf

# pointers, 64-bit sizes, then 32-bit fields, in the header's order
LINEAR_ARGS = struct.Struct("=7Q9q4i")
LINEAR_GRAD_ARGS = struct.Struct("=10Q11q4i")
COPY_ROWS = struct.Struct("=2Q4q")
LAYER_NORM_ARGS = struct.Struct("=6Q5qf3i")
LAYER_NORM_GRAD_ARGS = struct.Struct("=9Q7q2i")


def launch(name, packed):
    """Entry point `name` on PyTorch's current device and stream; raises for a refusal."""
    ext = wf("_ext")
    ext.check(getattr(ext.lib(), name)(packed, ext.stream_of("cuda")), name)
