"""Dense decoder operators at their borders: what autograd may ask beside a plain backward pass, layouts of operands that are
copied, tiles that four waves share, lambdas beyond f16's range, gradients of the module.

Bounds and references are those of test_decoder_ops_gpu."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from test_decoder_ops_gpu import DEV, TYPES, UF, Ref, attn_check, attn_drop, attn_inputs, causal, rand, within

pytestmark = pytest.mark.gpu


def operators(x, lam, seed=None):
    """the three operators on x (2, n, 2, 2, d)"""
    F = UF()
    return {'dropout': lambda: F.dropout(x, 0.3, True, seed=seed), 'layer_norm': lambda: F.layer_norm(x),
            'diff_attention': lambda: F.diff_attention(x, x, x.detach().flatten(3), lam, p=0.3, training=True, seed=seed)}


OPERATORS = ['dropout', 'layer_norm', 'diff_attention']


# --------------------------------------------------------------------------------------- what the nodes have no derivative for
@pytest.mark.parametrize('op', OPERATORS)
def test_a_forward_derivative_of_the_result_is_refused(op):
    """a tangent that enters must not vanish: neither a dual input nor a dual gradient of the result"""
    x = torch.randn(2, 5, 2, 2, 16, device=DEV)
    lam = torch.ones(2, device=DEV)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            operators(forward_ad.make_dual(x, torch.ones_like(x)), lam)[op]()
    x.requires_grad_()
    y = operators(x, lam)[op]()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    y = operators(x, lam)[op]()                                           # and the plain pass still runs
    assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()


@pytest.mark.parametrize('op', OPERATORS)
def test_tracing_and_batched_gradients_are_refused(op):
    x = torch.randn(2, 5, 2, 2, 16, device=DEV)
    lam = torch.ones(2, device=DEV)
    with pytest.raises(RuntimeError, match='trace'):
        torch.jit.trace(lambda t: operators(t, lam)[op](), (x,))
    with pytest.raises(RuntimeError, match='trace'):
        make_fx(lambda t: operators(t, lam)[op]())(x)
    x.requires_grad_()
    y = operators(x, lam)[op]()
    with pytest.raises(RuntimeError, match='ordinary tensors'):
        torch.autograd.grad(y, x, torch.ones(3, *y.shape, device=DEV), is_grads_batched=True)


# ----------------------------------------------------------------------------------------------------- layouts that are copied
@pytest.mark.parametrize('Dh,Dv', [(20, 20), (7, 13), (6, 42), (16, 20), (20, 32)])
@pytest.mark.parametrize('dt', TYPES)
def test_attention_channels_first_views_of_any_width(Dh, Dv, dt):
    """operands and grad_out whose tokens are the fastest axis, at widths that are no whole 16-byte pieces"""
    B, H, Hk, Nq, Nk = 2, 4, 2, 9, 33
    q, k, v, lam, go = (t.to(DEV) for t in attn_inputs(B, H, Hk, Nq, Nk, Dh, Dv, dt))

    def run(f):
        leaves = [f(t).requires_grad_() for t in (q, k, v)] + [lam.clone().requires_grad_()]
        y = UF().diff_attention(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, f(go))]

    def tokens_last(t):
        return t.movedim(1, -1).contiguous().movedim(-1, 1)
    assert tokens_last(v).stride(1) == 1
    for got, want in zip(run(tokens_last), run(torch.clone)):
        assert torch.equal(got, want)
