"""A tensor that an operator cannot do without, left out: refused with the operator's own error, before anything else."""
import pytest
import torch

from eacs_b200.ops.block_norm import gated_norm, residual_norm
from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step
from eacs_b200.ops.gated_delta import gated_delta_rule, gated_delta_step
from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step

t = torch.zeros(2, 5, 8)
CALLS = [(selective_ssm, 5, {}), (selective_ssm_step, 6, {}), (causal_conv, 2, {}), (causal_conv_step, 2, {"state": t}),
         (causal_conv_step, 2, {"state": None}), (gated_delta_rule, 5, {}), (gated_delta_step, 6, {}), (gated_norm, 1, {}), (residual_norm, 2, {})]


@pytest.mark.parametrize("f,needed,kw", CALLS)
def test_a_missing_tensor_is_refused(f, needed, kw):
    kw = dict(kw, bias=None) if f is causal_conv_step else kw
    for i in range(needed):
        args = [t] * needed
        args[i] = None
        with pytest.raises(RuntimeError, match=f.__name__ + ": expects (tensors|a residual)"):
            f(*args, **kw)
    if kw.get("state", t) is None:
        with pytest.raises(RuntimeError, match="the state"):
            f(*[t] * needed, **kw)
