"""Products with quantised weights as they are stored (``exl3_linear``, HIP).

``quantized_linear`` multiplies rows of activations with the weight that
``serialization.decode_weight_from_storage`` would decode, without decoding it
to memory: a served model reads K bits a weight instead of 16 or 32.
"""

from __future__ import annotations

import torch

from . import _native
from .hadamard import records
from .trellis_format import CB_MUL1


def quantized_linear(x: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor,
                     K: int, cb: int = CB_MUL1) -> torch.Tensor:
    """``x @ W`` (..., out) in x's type, for x (..., in) in float16 or bfloat16
    and W the (in, out) weight of a stored projection: ``trellis`` int16 (in /
    16, out / 16, 16 K), ``suh`` (in,) and ``svh`` (out,) in float16 or float32
    (or as a column and a row of them, as ``quantize_linear_module`` returns them),
    ``cb`` its codebook; all on x's device.

    The rows are scaled and transformed in float32 and count with 22 bits, or,
    more than 64 of them in bfloat16, with 11 (three more than their own); the
    codebook's values are exact, sums are float32; the result is rounded once. A
    row with an infinity or a NaN is NaN. Tensors that do not start at a multiple
    of 16 bytes, and rows that lie otherwise, are copied first. The call enqueues
    work on the current stream of x's device and keeps nothing. It has no
    gradient: train through ``x @ decode_weight_from_storage(...)``."""
    for t in (x, suh, svh):
        if isinstance(t, torch.Tensor) and records(t):
            raise RuntimeError("quantized_linear has no gradient: detach its inputs")
    return _native.linear(x, trellis, suh, svh, K, cb)
