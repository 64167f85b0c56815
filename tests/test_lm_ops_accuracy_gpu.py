"""Sums over long rows of logits, against 64 bits and bounds that count the kernels' roundings (U = 2^-24 each)."""
import math

import lm_oracle as oracle
import pytest
import torch
from test_lm_ops_cpu import _norm_vars, check_distill, check_tokens, teacher_rows

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


def _one_value(rows, V, gap, at, dtype, device):
    """Rows of two tokens, in places of one lane: at 0 one that is ``gap`` nats below the other, which is 0; the rest is masked"""
    x = torch.full((rows, V), -math.inf, device=device)
    x[:, 0] = -gap
    x[:, at] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3000, 8000, 10000, 50003, 131072])
def test_rows_that_one_value_makes_up(gpu, dtype, V):
    """The best token lies behind what the wave of lanes that holds it sees first, 4.3 to 13 nats above that.

    No sum has more than two terms here.  Whatever the wave's reference, it is at most 3.9 nats below the best token; where
    it was further, the best token is it: then the exponents are below 1 and their logarithm rounds at that size, 2 U at
    most for each of the exponential, the scale, the sums, the logarithm and the last difference, weighted sum and plain."""
    N = 16 // torch.empty(0, dtype=dtype).element_size()
    rows = 600
    gap = torch.linspace(4.3, 13.0, rows, device=gpu)
    at = {3000: 64, 8000: 64}.get(V, 256) * N * 2  # the same lane's third vector
    at = at if at < V else 64 * N
    x = _one_value(rows, V, gap, at, dtype, gpu)
    low = x[:, 0].double()
    logp = -torch.log1p(torch.exp(low))
    H = -logp - torch.exp(low + logp) * low
    tok = torch.full((rows,), at, device=gpu)
    leaf = x.detach().requires_grad_()
    r = ops.token_log_probs(leaf, tok, entropy=True, top_k=0)
    _close(r.logp.detach(), logp, 12 * U, "logp")
    _close(r.entropy.detach(), H, 12 * U, "entropy")
    again = ops.token_log_probs(x, tok, entropy=True, top_k=5)
    _close(again.logp, logp, 12 * U, "logp beside alternatives")
    _close(again.entropy, H, 12 * U, "entropy beside alternatives")
    _close(again.top_logp[:, 0], logp, 12 * U, "the best alternative")
    # d(H)/dx of the other token: -p (log p + H), f32 or rounded once more
    (dx,) = torch.autograd.grad(r.entropy.sum(), [leaf])
    p, lp = torch.exp(low + logp), low + logp
    want = -p * (lp + H)
    step = 2 * U if dtype == torch.float32 else oracle.half_step(torch.ones(()), dtype).item()
    assert bool(((dx[:, 0].double() - want).abs() <= want.abs() * (40 * U + step)).all())
    for unit in (False, True):
        loss = ops.distillation_loss(leaf, torch.zeros(rows, 1, device=gpu), tok[:, None], row_weight=torch.ones(rows, device=gpu),
                                     unit_seed=unit)
        _close(loss.detach(), -logp.sum(), rows * 12 * U + 4 * U * float(-logp.sum()), "distillation")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [700, 5003, 9000, 50003])
@pytest.mark.parametrize("rows", [12, 600])
def test_values_far_from_zero_and_from_what_comes_first(gpu, rows, V, dtype):
    """A reference that is too low again and again, that is missing, that is too far out to be one"""
    torch.manual_seed(V)
    x = 2 * torch.randn(12, V, device=gpu)
    i = torch.arange(V, device=gpu, dtype=torch.float32)
    x[0] += i * (300.0 / V)                     # rising all the way
    x[1] = torch.floor(i / 2048) * 7.0          # in steps
    x[2] -= i * (300.0 / V)
    x[3] = -3e8 + 64 * torch.floor(8 * torch.rand(V, device=gpu))   # all far out
    x[4, :V // 2] = -1.2e7                      # far out (2^24 halvings are 1.163e7 nats), then not
    x[4, V // 2:] = -1.1e7
    x[5, :V // 2] = torch.finfo(dtype).min
    x[6, V // 3] = 3e38                         # one value above everything
    x[7, :V - 3] = -math.inf
    x[8] = -1.163e7 + torch.floor(4 * torch.randn(V, device=gpu))   # around where far out begins
    x[9] = 1.163e7 + torch.floor(4 * torch.randn(V, device=gpu))
    x[10, :V // 2] = -math.inf
    x[10, V // 2:] -= 400.0
    x[11] = -math.inf
    x[11, V // 2] = -5e7
    x = x.to(dtype).repeat(rows // 12, 1)
    tok = torch.randint(0, V, (rows,), device=gpu)
    tok[:12] = x[:12].float().argmax(1)
    g = torch.randn(rows, device=gpu)
    # powers of two above 1: 3e38 / T is within f32, and exact (the oracle allows alternatives of probability 0 no rounding)
    for T in (1.0, 2.0):
        check_tokens(x, tok, 0, T, g, g)
        check_tokens(x, tok, 6, T)
    keep = torch.tensor([k for k in range(rows) if k % 12 not in (3, 6, 7, 8, 9, 11)], device=gpu)
    t, ids = teacher_rows(len(keep), V, 4, gpu)
    ids = torch.where(ids < 0, ids, V - 1 - ids % 5)
    for unit in (False, True):
        check_distill(x[keep], t, ids, None, 1.0, unit_seed=unit)
    for bad in (math.nan, math.inf):  # alone among masked places, and in front of others
        y = x[:4].clone()
        y[0] = -math.inf
        y[0, V // 2], y[1, 0], y[2, V - 1], y[3, V // 2] = bad, bad, bad, bad
        r = ops.token_log_probs(y, tok[:4] % V, entropy=True, top_k=3)
        assert torch.isnan(r.logp).all() and torch.isnan(r.entropy).all()


def test_layer_norm_of_very_wide_equal_rows(gpu):
    """The mean of 2^22 equal values: up to 32 terms in f32 at a time (31 roundings), 64 bits, the tree (10), the division (2); what
    it is off is scaled by 1 / sqrt(eps)"""
    x = torch.full((3, 1 << 22), 0.1, device=gpu)
    y = ops.layer_norm(x)
    assert float(y.abs().max()) <= (31 + 1 + 10 + 2) * U * 0.1 / math.sqrt(1e-5)


@pytest.mark.parametrize("C", [16400, 600])
def test_layer_norm_weights_gradients_of_many_equal_rows(gpu, C):
    """40000 equal rows: blocks or threads of at most 157 rows one after the other, of wide rows up to 32, and 64 bits"""
    torch.manual_seed(0)
    rows = 40000
    _, g, b = _norm_vars(C, gpu)
    x, dy = torch.randn(1, C, device=gpu), 0.1 + torch.rand(1, C, device=gpu)
    ops.layer_norm(x.expand(rows, C), g, b).backward(dy.expand(rows, C))
    xh = (x.double() - x.double().mean()) * torch.rsqrt(x.double().var(unbiased=False) + 1e-5)
    n = 31 + 20 if C > 16384 else 157 + 24  # of a thread or a group; the joins
    want = rows * dy.double()[0]
    assert bool(((b.grad - want).abs() <= n * U * want).all())
    want = want * xh[0]
    # the mean is off by 60 U of itself and its standard deviation's 60 U, xh by as much and 4 U of itself
    assert bool(((g.grad - want).abs() <= n * U * want.abs() + rows * dy[0] * U * (60 + 64 * xh[0].abs())).all())
