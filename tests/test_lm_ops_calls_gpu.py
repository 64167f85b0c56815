"""Calls of layer norm, token log probabilities and distillation that their programs make rarely."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from test_lm_ops_cpu import _norm_vars, teacher_rows

from tensorflow_examples_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reverse", [False, True])
def test_forward_mode_is_refused(gpu, reverse):
    """As on the CPU: a result without the tangent would be taken for one that does not depend on the input"""
    x = torch.randn(4, 8, device=gpu, requires_grad=reverse)
    tok = torch.zeros(4, dtype=torch.long, device=gpu)
    t, ids = teacher_rows(4, 8, 3, gpu)
    _, g, b = _norm_vars(8, gpu)
    calls = (lambda v: ops.token_log_probs(v, tok, top_k=2).logp, lambda v: ops.distillation_loss(v, t, ids),
             lambda v: ops.distillation_loss(v, t, ids, unit_seed=True), lambda v: ops.layer_norm(v),
             lambda v: ops.layer_norm(v, g, b))
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError):
                call(d)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(d)
            call(x)
