"""eacs_b200 -- B200 (sm_100a) kernels for CST-SSM's EACS temporal hot path.

Modules under eacs_b200.ops mirror the reference's operator modules
(cst_ssm/ops/scan.py, scan_cuda.py, eacs_gated_scan.py, eacs_cell_train.py)
with the same function names and argument meaning; eacs_b200.install() points
an imported reference package at these kernels.

Operators beside the reference's: ops.layer_norm, ops.gated_delta (a recurrence
with a matrix state), ops.selective_ssm (a diagonal recurrence whose steps go by
the token), ops.causal_conv (the short convolution in front of a recurrence) and
ops.block_norm (the norms before and after a block with its gate and residual).
"""
from ._lib import LIB_PATH, device_status, version  # noqa: F401
from .install import install  # noqa: F401

__version__ = "0.1.0"
