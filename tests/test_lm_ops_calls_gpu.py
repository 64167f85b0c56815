"""Calls of layer norm, token log probabilities and distillation that their programs make rarely."""
import copy
import ctypes
import gc
import pickle

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


def _norm_case(gpu, C=40, **kw):
    torch.manual_seed(0)
    store, g, b = _norm_vars(C, gpu, **kw)
    x, dy = torch.randn(70, C, device=gpu), torch.randn(70, C, device=gpu)
    ops.layer_norm(x, g, b).backward(dy)
    want = g.grad.clone(), b.grad.clone()
    store.grad.zero_()
    return store, g, b, x, dy, want


def test_layer_norm_hook_set_behind_the_forward_pass(gpu):
    """The hook is looked at when the gradients are there, as with every other operator"""
    store, g, b, x, dy, want = _norm_case(gpu)
    fired = []

    def hook(v):
        fired.append((v, v.grad.clone()))
    y = ops.layer_norm(x, g, b)
    store.grad_ready_hook = hook
    y.backward(dy)
    assert [v for v, _ in fired] == [g, b] and all(torch.equal(t, w) for (_, t), w in zip(fired, want))
    y = ops.layer_norm(x, g, b)  # taken away again
    store.grad_ready_hook = None
    y.backward(dy)
    assert len(fired) == 2
    y = ops.layer_norm(x, g)  # one weight
    store.grad_ready_hook = hook
    y.backward(dy)
    assert len(fired) == 3 and fired[2][0] is g

    def failing(v):
        raise KeyError("from the hook")
    store.grad_ready_hook = None
    y = ops.layer_norm(x, g, b)
    store.grad_ready_hook = failing
    with pytest.raises(KeyError, match="from the hook"):
        y.backward(dy)


def test_layer_norm_gradients_go_where_the_store_has_them_then(gpu):
    store, g, b, x, dy, want = _norm_case(gpu)
    y = ops.layer_norm(x, g, b)
    old, store.grad = store.grad, torch.zeros_like(store.grad)
    y.backward(dy)
    assert torch.equal(g.grad, want[0]) and torch.equal(b.grad, want[1]) and not old.any()


def test_layer_norm_of_copied_and_of_gone_stores(gpu):
    store, g, b, x, dy, want = _norm_case(gpu)
    y = ops.layer_norm(x, g, b)
    other = copy.deepcopy(store)
    ops.layer_norm(x, *other.vars).backward(dy)
    assert not store.grad.any() and torch.equal(other.vars[0].grad, want[0])
    again = pickle.loads(pickle.dumps(store))
    ops.layer_norm(x, *again.vars).backward(dy)
    assert not store.grad.any() and torch.equal(again.vars[1].grad, want[1])
    leaf = x.clone().requires_grad_()
    y = ops.layer_norm(leaf, g, b)
    store.grad_ready_hook = lambda v: None
    del store, g, b
    gc.collect()
    y.backward(dy)  # the node keeps what it writes to
    assert torch.isfinite(leaf.grad).all()


def test_an_earlier_error_of_anothers_stays_its_owners(gpu):
    """A refused runtime call (a device that is not there) leaves an error on this thread: the operators neither take it for
    theirs nor take it away"""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    x = torch.randn(6, 300, device=gpu)
    tok = torch.zeros(6, dtype=torch.long, device=gpu)
    t, ids = teacher_rows(6, 300, 3, gpu)
    torch.cuda.synchronize()
    hip.hipGetLastError()
    assert hip.hipSetDevice(1000) != 0
    left = hip.hipPeekAtLastError()
    try:
        if left == 0:
            pytest.skip("this runtime keeps no error of a refused call")
        with torch.no_grad():
            ops.token_log_probs(x, tok, top_k=2, entropy=True)
            ops.distillation_loss(x, t, ids)
            ops.layer_norm(x)
        assert hip.hipPeekAtLastError() == left
    finally:
        hip.hipGetLastError()
