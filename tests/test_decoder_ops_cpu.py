"""Dropout, layer norm and differential attention where no GPU is needed: the C entries refuse bad arguments before any launch,
the Python entries refuse CPU tensors, the module builds from the registry."""
import ctypes
import os

import pytest
import torch

from unibev_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(1 << 20)          # a 16-byte aligned address that no refused call may touch


def refused(status, word):
    assert status == -1, status
    assert word in _lib.lib().ubv_last_error().decode()


def test_dropout_entry_refuses():
    f = _lib.lib().ubv_dropout
    refused(f(None, None, P, 8, 0.1, 0, None, 0, 0, None), 'bad arguments')
    refused(f(P, None, P, -1, 0.1, 0, None, 0, 0, None), 'bad arguments')
    refused(f(P, None, P, 8, 0.1, 0, None, 3, 0, None), 'dtype')
    refused(f(P, None, P, 8, 0.1, 0, None, 1, 2, None), '16-bit')
    refused(f(P, None, P, 8, 1.5, 0, None, 0, 0, None), 'p = 1.5')
    refused(f(P, None, P, 8, float('nan'), 0, None, 0, 0, None), 'p = ')
    assert f(None, None, None, 0, 0.1, 0, None, 0, 0, None) == 0


def test_layer_norm_entries_refuse():
    f, b = _lib.lib().ubv_layer_norm_forward, _lib.lib().ubv_layer_norm_backward
    refused(f(P, None, None, P, None, None, 4, 0, 1e-5, 0, None), 'out of range')
    refused(f(P, None, None, P, None, None, 1 << 31, 4, 1e-5, 0, None), 'out of range')
    refused(f(P, None, None, P, None, None, 4, 4, 1e-5, 7, None), 'dtype')
    refused(f(None, None, None, P, None, None, 4, 4, 1e-5, 0, None), 'null')
    refused(f(P, None, None, P, P, None, 4, 4, 1e-5, 0, None), 'null')
    assert f(None, None, None, None, None, None, 0, 4, 1e-5, 0, None) == 0
    refused(b(P, P, None, P, P, P, None, None, 0, 4, 0, None, 0, None), 'no rows')
    refused(b(P, P, None, P, P, None, None, None, 4, 4, 0, None, 0, None), 'null')
    refused(b(P, P, None, P, P, P, P, None, 4, 4, 0, None, 0, None), 'workspace')
    need = _lib.lib().ubv_layer_norm_backward_workspace(4, 4)
    assert need > 0
    refused(b(P, P, None, P, P, P, P, P, 4, 4, 0, P, need - 1, None), 'workspace')


def attn_call(q=P, k=P, v=P, lam=P, mask=None, kind=0, out=P, stat=None, maps=None, strides=None, B=1, H=4, Hk=2, Nq=8, Nk=8, Dh=32,
              Dv=64, p=0.0, dtype=0, scale=0.1):
    s = strides if strides is not None else [0] * 18
    return _lib.lib().ubv_diff_attention_forward(q, k, v, lam, None, mask, kind, out, stat, maps, (ctypes.c_int64 * 18)(*s), B, H, Hk, Nq,
                                                 Nk, Dh, Dv, scale, 0, p, 0, None, dtype, None, 0, None)


@pytest.mark.parametrize('kw,word', [(dict(q=None), 'null'), (dict(lam=None), 'null'), (dict(dtype=3), 'dtype'), (dict(Nq=0), 'empty'),
                                     (dict(Hk=3), 'share'), (dict(Dh=129), 'widths'), (dict(Dv=257), 'widths'), (dict(p=-0.1), 'p = '),
                                     (dict(kind=1), 'mask kind'), (dict(mask=P, kind=3), 'mask kind'), (dict(out=None), 'out'),
                                     (dict(stat=P), 'maps'), (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'),
                                     (dict(strides=[0, 1 << 22] + [0] * 16), 'token stride'), (dict(strides=[0] * 7 + [1 << 26] + [0] * 10), 'map stride'), (dict(q=ctypes.c_void_p((1 << 20) + 2)), 'aligned'),
                                     (dict(strides=[0] * 5 + [6] + [0] * 12), '16 bytes'), (dict(Nq=1 << 30, H=8, Hk=2), 'out of range')])
def test_attention_forward_entry_refuses(kw, word):
    refused(attn_call(**kw), word)


def test_attention_backward_entry_refuses():
    f = _lib.lib().ubv_diff_attention_backward
    need = _lib.lib().ubv_diff_attention_backward_workspace(1, 4, 2, 8, 8, 32, 64, 0, 0)
    s = (ctypes.c_int64 * 18)()

    def call(go=P, stat=P, gq=P, gk=P, gv=P, ws=P, n=need):
        return f(go, P, P, P, P, None, None, 0, stat, P, gq, gk, gv, P, s, 1, 4, 2, 8, 8, 32, 64, 0.1, 0, 0.0, 0, None, 0, ws, n, None)

    assert need > 0 and _lib.lib().ubv_diff_attention_backward_workspace(0, 4, 2, 8, 8, 32, 64, 0, 0) == 0
    refused(call(go=None), 'grad_out')
    refused(call(stat=None), 'stat')
    refused(call(gv=None), 'come together')
    refused(call(gq=ctypes.c_void_p((1 << 20) + 4)), 'aligned')
    refused(call(n=need - 1), 'workspace')
    refused(call(ws=None), 'workspace')


@pytest.mark.parametrize('Nq,Nk,causal', [(1 << 30, 8, 0), (1 << 29, 8, 0), (8, (1 << 31) - 1, 0), (8, (1 << 31) - 256, 0), (1 << 28, (1 << 31) - 300, 1)])
def test_attention_workspace_of_a_call_out_of_range(Nq, Nk, causal):
    """sizes that 32-bit counts do not hold: the workspace entries answer (another process: they used to divide by zero), the call refuses"""
    import subprocess
    import sys
    code = (f'from unibev_amd import _lib; l = _lib.lib(); a = (1, 8, 2, {Nq}, {Nk}, 32, 64, {causal}, 0); '
            'print(l.ubv_diff_attention_forward_workspace(*a), l.ubv_diff_attention_backward_workspace(*a) >= 28 * 8 * a[3])')
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.split() == ['0', 'True'], (r.returncode, r.stdout, r.stderr[-500:])
    s = (ctypes.c_int64 * 18)()
    refused(_lib.lib().ubv_diff_attention_forward(P, P, P, P, None, None, 0, P, None, None, s, 1, 8, 2, Nq, Nk, 32, 64, 0.1, causal, 0.0, 0, None,
                                                  0, None, 0, None), 'out of range')


def test_cpu_tensors_are_refused():
    from unibev_amd import functional as UF
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match='GPU only'):
        UF.dropout(x, 0.1, True)
    with pytest.raises(RuntimeError, match='GPU only'):
        UF.layer_norm(x)
    with pytest.raises(RuntimeError, match='GPU only'):
        UF.diff_attention(torch.zeros(1, 3, 2, 2, 8), torch.zeros(1, 3, 2, 2, 8), torch.zeros(1, 3, 2, 16), torch.ones(2))


def test_module_builds_from_the_registry():
    from unibev_amd import build_attention
    m = build_attention(dict(type='DifferentialAttention', embed_dims=64, num_heads=4, num_kv_heads=2, dropout=0.1))
    assert m.attn_drop == m.residual_drop == 0.1 and m.head_dims == 16
    assert {k: tuple(v.shape) for k, v in m.state_dict().items() if 'lambda' in k or 'k_proj.w' in k} == {
        'lambda_a': (2, 8), 'lambda_b': (2, 8), 'k_proj.weight': (32, 64)}
    with torch.no_grad():
        m.lambda_a.zero_()
    assert m.lam().item() == pytest.approx(0.8)
    for bad in (dict(num_heads=3), dict(num_heads=64), dict(num_heads=4, num_kv_heads=3)):
        with pytest.raises(ValueError):
            build_attention(dict(type='DifferentialAttention', embed_dims=64, **bad))


def test_layer_norm_workspace_counts_the_rows_that_are_written():
    """rows of at most 8192 elements: one row of 2 C sums a block, 1024 blocks at most; wider ones are summed in 64 slabs"""
    need = _lib.lib().ubv_layer_norm_backward_workspace
    assert need(1000, 256) == 1000 * 2 * 256 * 4 and need(5000, 8192) == 1024 * 2 * 8192 * 4
    assert need(5000, 8193) == 64 * 2 * 8193 * 4 and need(3, 20000) == 3 * 2 * 20000 * 4
    assert need(0, 20000) == 0


def decoder_calls():
    """name -> call with one operand replaced"""
    from unibev_amd import functional as UF
    x, w = torch.randn(2, 3, 2, 16), torch.ones(16)
    q, v, lam, mask = torch.randn(1, 3, 2, 2, 8), torch.randn(1, 3, 2, 16), torch.ones(2), torch.zeros(3, 3)
    return {'dropout x': (x, lambda t: UF.dropout(t, 0.1, True)), 'dropout identity': (x, lambda t: UF.dropout(x, 0.1, True, identity=t)),
            'norm x': (x, lambda t: UF.layer_norm(t, w, w)), 'norm gamma': (w, lambda t: UF.layer_norm(x, t, w)),
            'norm beta': (w, lambda t: UF.layer_norm(x, w, t)), 'attention q': (q, lambda t: UF.diff_attention(t, q, v, lam)),
            'attention k': (q, lambda t: UF.diff_attention(q, t, v, lam)), 'attention v': (v, lambda t: UF.diff_attention(q, q, t, lam)),
            'attention lam': (lam, lambda t: UF.diff_attention(q, q, v, t)),
            'attention mask': (mask, lambda t: UF.diff_attention(q, q, v, lam, attn_mask=t))}


@pytest.mark.parametrize('name', list(decoder_calls()))
def test_forward_mode_derivatives_are_refused(name):
    import torch.autograd.forward_ad as forward_ad
    t, call = decoder_calls()[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
    with pytest.raises(RuntimeError, match='forward-mode|ordinary tensors'):
        torch.autograd.functional.jacobian(call, t, strategy='forward-mode', vectorize=True)


@pytest.mark.parametrize('name', list(decoder_calls()))
def test_tracing_is_refused(name):
    t, call = decoder_calls()[name]
    with pytest.raises(RuntimeError, match='trace'):
        torch.jit.trace(call, (t,))
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    for mode in ('real', 'fake'):
        with pytest.raises(RuntimeError, match='trace'):
            make_fx(call, tracing_mode=mode)(t)
    with FakeTensorMode() as fake, pytest.raises(RuntimeError, match='trace'):
        call(fake.from_tensor(t))


@pytest.mark.parametrize('name', list(decoder_calls()))
def test_transformed_tensors_are_refused(name):
    t, call = decoder_calls()[name]
    with pytest.raises(RuntimeError, match='ordinary tensors'):
        torch.vmap(call)(torch.stack([t, t]))
    with pytest.raises(RuntimeError, match='ordinary tensors'):
        torch.func.grad(lambda t: call(t).sum())(t)
    with pytest.raises(RuntimeError, match='ordinary tensors'):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))
    with pytest.raises(RuntimeError, match='ordinary tensors'):
        call(t.to_sparse())
