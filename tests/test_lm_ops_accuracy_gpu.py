"""Sums over long rows of logits, against 64 bits and bounds that count the kernels' roundings (U = 2^-24 each)."""
import math

import lm_oracle as oracle
import pytest
import torch

from tensorflow_examples_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
U = oracle.U


# A sum over a row, relative: a lane's piece of up to 32 terms (31 roundings, exponents below 1 and their exponentials 3),
# the pieces (in 64 bits and one rounding, or of up to 16 vectors 4), the wave (6), its own scale (2), the waves' join (5).
SUM = 31 + 3 + 4 + 6 + 2 + 5


def _close(got, want, bound, what):
    off = (got.double() - want.double()).abs().max()
    assert float(off) <= bound, (what, float(off), bound)


@pytest.mark.parametrize("dtype,V,base", [(torch.bfloat16, 131072, -1.0), (torch.float32, 131072, -1.0),
                                          (torch.bfloat16, 1 << 20, -1.0), (torch.float32, 1 << 20, -1.0),
                                          (torch.float32, 1 << 22, -1.0), (torch.float32, 1 << 20, 3e7)])
def test_long_rows_of_two_values(gpu, dtype, V, base):
    """Nearly all terms equal: every addition to a running sum would round the same way.  3e7: so far from 0 that the row
    is gone over again, against its maximum."""
    rows, step = 600, 2.0 if base > 0 else 0.5  # rows enough for each to be one part
    row = torch.full((V,), base, device=gpu)
    row[torch.arange(4, device=gpu) * 64 * (16 // torch.empty(0, dtype=dtype).element_size())] = base + step
    row = row.to(dtype)
    x = row.expand(rows, V)
    tok = torch.full((rows,), V - 1, device=gpu)
    r = ops.token_log_probs(x, tok, entropy=True)
    n = V - 4
    s = 4 + n * math.exp(-step)  # against the larger value
    logp = -step - math.log(s)
    H = math.log(s) + step * n * math.exp(-step) / s
    # the exponents' sizes beside what SUM counts: 3 at 2 nats; the logarithm and the result are rounded at their own size
    e = SUM + 3 + 2 * math.log(s) + 2
    _close(r.logp, torch.full((rows,), logp, dtype=torch.float64, device=gpu), e * U, "logp")
    # t / s takes both sums' errors
    _close(r.entropy, torch.full((rows,), H, dtype=torch.float64, device=gpu), (e + 2 * (SUM + 3) * step + 4 * H) * U, "entropy")
    leaf = x[:512].detach().requires_grad_()
    ids, t = torch.full((512, 1), V - 1, device=gpu), torch.zeros(512, 1, device=gpu)
    for unit in (False, True) if V == 131072 else ():
        loss = ops.distillation_loss(leaf, t, ids, unit_seed=unit)  # the mean of equal rows; two roundings more
        _close(loss.detach(), torch.tensor(-logp, dtype=torch.float64, device=gpu), (e - 2 * logp) * U, "distillation")
