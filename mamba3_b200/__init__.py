"""B200-native (sm_100a) Mamba-3 mixer: drop-in for jreoka/mamba3's ``Mamba3``, with a gated
recurrence, 4-bit projections for decoding and an orthogonalising optimiser beside it."""

from .model import Mamba3
from .optim import Muon, orthogonalize
from .quant import LinearW4, dequantize_w4, linear_w4, quantize_projections, quantize_w4
from .recurrence import GatedRecurrence, gated_scan, gated_step

# a star import gives what the reference's does; the other operators are imported by name
__all__ = ["Mamba3"]
