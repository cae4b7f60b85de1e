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


# ------------------------------------------------------------------------------------------------------ lambdas of any size
@pytest.mark.parametrize('Dh,Dv,size', [(16, 32, 0.01), (32, 64, 0.01), (16, 256, 2.0)])
def test_attention_f16_lam_beyond_the_types_range(Dh, Dv, size):
    """|lam| past 255: (A_1 - lam A_2) 2^8 and dS_2 would leave f16's range, the gradients do not.  Both enter the products at a
    power of two s <= 1 of their usual size, (1 + largest |lam| of the group) 2^8 s < 2^15: beside the usual bounds they may be off
    by half of f16's smallest step, 2^-25 over s (2^8 s), times what they are multiplied with."""
    B, H, Hk, Nq, Nk, dt = 1, 4, 2, 6, 5, torch.float16
    q, k, v, _, go = attn_inputs(B, H, Hk, Nq, Nk, Dh, Dv, dt)
    go = (go.float() * size).to(dt)
    lam = torch.tensor([0.5, -300.0, 20000.0, 3.0])
    scale = 2.0 ** -6
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam)]
    y = UF().diff_attention(*leaves, scale=scale)
    y.backward(go.to(DEV))
    r = Ref(q, k, v, lam, go, dt, scale=scale)
    assert max(t.abs().max() for t in (r.out, r.q, r.k, r.v)) < 65504
    s = torch.tensor([2.0 ** -2, 2.0 ** -8]).double()                          # 14 - floor(log2(1 + |lam|)) - 8 of 300 and 20000
    rows = Nq * H // Hk
    ek = r.ek + scale * 2.0 ** -25 / s.view(1, 1, Hk, 1, 1) * rows * q.double().abs().max()
    ev = r.ev + 2.0 ** -33 / s.view(1, 1, Hk, 1) * rows * go.double().abs().max()
    within(y, r.out, r.e_out, 'out')
    for t, ref, e, what in ((leaves[0], r.q, r.eq, 'grad_q'), (leaves[1], r.k, ek, 'grad_k'), (leaves[2], r.v, ev, 'grad_v'),
                            (leaves[3], r.lam, r.e_lam, 'grad_lam')):
        within(t.grad, ref, e, what)


def test_attention_f16_lam_of_the_last_of_many_shared_heads():
    """the largest |lam| of a group counts, whichever of its heads has it, where a few keys' rows are split over blocks too"""
    B, H, Hk, Nq, Nk, Dh, Dv, dt = 1, 8, 1, 400, 5, 32, 64, torch.float16
    q, k, v, _, go = attn_inputs(B, H, Hk, Nq, Nk, Dh, Dv, dt)
    go = (go.float() * 0.01).to(dt)
    lam = torch.tensor([0.5] * 7 + [-5000.0])                                  # s = 2^(14 - 12 - 8)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam)]
    y = UF().diff_attention(*leaves)
    y.backward(go.to(DEV))
    r = Ref(q, k, v, lam, go, dt)
    rows, s = Nq * H, 2.0 ** -6
    within(y, r.out, r.e_out, 'out')
    within(leaves[1].grad, r.k, r.ek + Dh ** -0.5 * 2.0 ** -25 / s * rows * q.double().abs().max(), 'grad_k')
    within(leaves[2].grad, r.v, r.ev + 2.0 ** -33 / s * rows * go.double().abs().max(), 'grad_v')


# ------------------------------------------------------------------------------------------------------ the device seed base
@pytest.mark.parametrize('op', ['dropout', 'diff_attention'])
def test_a_changed_seed_base_is_noticed(op):
    """the backward pass draws the forward pass's mask again: not from another base"""
    F = UF()
    base = torch.zeros(1, dtype=torch.int64, device=DEV)
    x = torch.randn(2, 9, 2, 2, 16, device=DEV, requires_grad=True)
    lam = torch.ones(2, device=DEV)
    F.set_seed_base(base)
    try:
        y = operators(x, lam)[op]()
        base.add_(1)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()
        y = operators(x, lam, seed=3)[op]()                                    # a given seed does not look at it
        base.add_(1)
        y.sum().backward()
        y = operators(x, lam)[op]()
        torch.autograd.grad(y.sum(), x)
    finally:
        F.set_seed_base(None)


# ------------------------------------------------------------------------------------------------- what the 16-bit types keep
@pytest.mark.parametrize('Dh,Dv', [(16, 32), (32, 64), (64, 64), (64, 128), (128, 128), (128, 256)])
@pytest.mark.parametrize('kind', ['plain', 'causal dropped shared heads'])
@pytest.mark.parametrize('dt', [torch.float16, torch.bfloat16])
def test_attention_16_bit_results_are_off_by_little_more_than_their_own_rounding(Dh, Dv, kind, dt):
    """By norm, in units of what rounding the exact result to the type does.  out and grad_v add one rounding of each probability:
    the errors of N terms against one of the sum, sqrt(1 + 1) at most where the terms are independent.  dS enters with the rest of
    its rounding, so grad_q and grad_k add what del = grad_out . o takes over from out, P del k in size: over rows whose squared
    probabilities sum to S, sqrt(S) of a rounding; S is under 0.2 here (300 keys, scores of deviation 1.5 and under), so
    sqrt(1 + 0.2) = 1.1.  Both with a tenth on top."""
    B, H, Hk, Nq, Nk = 1, 4, 4, 300, 300
    hidden, p, kw = None, 0.0, {}
    if kind != 'plain':
        Hk, Nq, hidden, p, kw = 2, 60, causal(60, 300), 0.1, dict(causal=True)
    q, k, v, lam, go = attn_inputs(B, H, Hk, Nq, Nk, Dh, Dv, dt)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, lam)]
    y = UF().diff_attention(*leaves, p=p, training=True, seed=77, **kw)
    y.backward(go.to(DEV))
    r = Ref(q, k, v, lam, go, dt, hidden, None, attn_drop(77, B, H, Nq, Nk, p))
    for what, t, ref, most in (('out', y, r.out, 1.56), ('grad_q', leaves[0].grad, r.q, 1.21), ('grad_k', leaves[1].grad, r.k, 1.21),
                               ('grad_v', leaves[2].grad, r.v, 1.56)):
        one = (ref.to(dt).double() - ref).norm()
        off = (t.detach().double().cpu() - ref).norm()
        assert off <= most * one, f'{what}: {(off / one).item():.2f} roundings'


# ------------------------------------------------------------------------------------------------- tiles that four waves share
def check_heads(B, H, Hk, Nq, Nk, Dh, Dv, dt, hidden=None, bias=None, p=0.0, **kw):
    """a call of many heads, of which the first, a middle and the last key head (and their query heads) are compared"""
    gen = torch.Generator(DEV).manual_seed(Dh + Dv)

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dt)
    q, k, v, go = randn(B, Nq, H, 2, Dh, std=1.5), randn(B, Nk, Hk, 2, Dh), randn(B, Nk, Hk, Dv), randn(B, Nq, H, Dv)
    lam = torch.randn(H, generator=gen, device=DEV) * 0.2 + 0.5
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = UF().diff_attention(*leaves, p=p, training=True, seed=77, **kw)
    y.backward(go)
    kv, G = [0, Hk // 2 - 1, Hk - 1], H // Hk
    hq = [h * G + g for h in kv for g in range(G)]
    D = attn_drop(77, B, H, Nq, Nk, p)
    r = Ref(*(t.detach().cpu() for t in (q[:, :, hq], k[:, :, kv], v[:, :, kv], lam[hq], go[:, :, hq])), dt, hidden,
            None if bias is None else bias[:, hq].cpu(), None if D is None else D[:, hq])
    within(y[:, :, hq], r.out, r.e_out, 'out')
    for t, ref, e, what in ((q.grad[:, :, hq], r.q, r.eq, 'grad_q'), (k.grad[:, :, kv], r.k, r.ek, 'grad_k'),
                            (v.grad[:, :, kv], r.v, r.ev, 'grad_v'), (lam.grad[hq], r.lam, r.e_lam, 'grad_lam')):
        within(t, ref, e, what)
    assert all(torch.isfinite(t.grad).all() for t in leaves) and torch.isfinite(y).all()


@pytest.mark.parametrize('Dh,Dv', [(16, 32), (32, 64), (64, 64), (64, 128), (128, 128), (128, 256)])
@pytest.mark.parametrize('kind', ['plain', 'dropped', 'causal', 'padded causal', 'masked', 'float dropped causal'])
@pytest.mark.parametrize('dt', TYPES)
def test_attention_shared_tiles_of_every_kind_of_call(Dh, Dv, kind, dt):
    """So many heads that tiles of 128 own items fill the chip (causal: over 1638 tiles of 32 items; else several rounds of the
    chip's 256 blocks), in every pass but grad_k / grad_v at 128 / 128, which has none.  Several such tiles a head, the last of
    them part empty, and with two query heads to a key head rows that run on from one to the other inside a tile."""
    if kind in ('plain', 'dropped'):
        return check_heads(2, 56, 56, 250, 250, Dh, Dv, dt, p=0.1 if kind == 'dropped' else 0.0)
    if kind == 'masked':
        Nq = Nk = 250
        m = torch.rand(Nq, Nk, generator=torch.Generator().manual_seed(1)) < 0.3
        m[::9] = True
        return check_heads(2, 56, 56, Nq, Nk, Dh, Dv, dt, hidden=m, attn_mask=m.to(DEV))
    B, H, Hk, Nq, Nk = 2, 192, 96, 230, 300
    hidden, kw = causal(Nq, Nk), dict(causal=True)
    if kind == 'padded causal':
        pad = torch.arange(Nk)[None] >= torch.tensor([[Nk], [171]])
        hidden, kw['key_padding_mask'] = hidden | pad[:, None, None], pad.to(DEV)
    elif kind == 'float dropped causal':
        gen = torch.Generator(DEV).manual_seed(2)
        bias = -torch.rand(1, H, Nq, Nk, generator=gen, device=DEV) * 20
        kw.update(attn_mask=bias, bias=bias, p=0.1)
    check_heads(B, H, Hk, Nq, Nk, Dh, Dv, dt, hidden=hidden, **kw)


@pytest.mark.parametrize('Nq,Nk', [(45, 77), (77, 45), (300, 300)])
@pytest.mark.parametrize('dt', TYPES)
def test_attention_padded_causal_without_dropout(Nq, Nk, dt):
    """the causal kernels beside hidden keys, a sample with none left"""
    pad = torch.arange(Nk)[None] >= torch.tensor([[Nk], [20], [0]])
    pad[1, 3:7] = True
    attn_check(*attn_inputs(3, 4, 2, Nq, Nk, 32, 64, dt), dt, hidden=pad[:, None, None] | causal(Nq, Nk), causal=True,
               key_padding_mask=pad.to(DEV))


# ------------------------------------------------------------------------------------------------------ gradients of the module
class NoisyLinear(torch.autograd.Function):
    """a Linear in 64 bits whose products (y, grad_x, grad_w) and sum (grad_b) are off by up to eps of the sum of their terms' sizes"""

    @staticmethod
    def forward(ctx, x, w, b, eps, gen):
        ctx.save_for_backward(x, w)
        ctx.eps, ctx.gen = eps, gen
        return NoisyLinear.off(x @ w.t(), x.abs() @ w.abs().t(), eps, gen) + b

    @staticmethod
    def off(y, size, eps, gen):
        return y + eps * size * (torch.randint(0, 2, y.shape, generator=gen) * 2 - 1) if eps else y

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        gf, xf = g.flatten(0, -2), x.flatten(0, -2)
        return (NoisyLinear.off(g @ w, g.abs() @ w.abs(), ctx.eps, ctx.gen),
                NoisyLinear.off(gf.t() @ xf, gf.abs().t() @ xf.abs(), ctx.eps, ctx.gen),
                NoisyLinear.off(gf.sum(0), gf.abs().sum(0), ctx.eps, ctx.gen), None, None)


def module_pass(m, ins, go, hidden, eps, seed=0):
    """output and gradients (parameters by name, then inputs) of the module's definition in 64 bits on the CPU"""
    gen = torch.Generator().manual_seed(seed)
    P = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    query, key, value, identity, qpos, kpos = (None if t is None else t.double().requires_grad_() for t in ins)
    leaves = [t for t in (query, key, value, identity, qpos, kpos) if t is not None]
    flip = (lambda t: t) if m.batch_first else (lambda t: t.transpose(0, 1))

    def lin(x, name):
        return NoisyLinear.apply(x, P[name + '.weight'], P[name + '.bias'], eps, gen)
    k_in = query if key is None else key
    v_in = k_in if value is None else value
    kp = qpos if kpos is None and qpos is not None and qpos.shape == k_in.shape else kpos
    q = flip(lin(query if qpos is None else query + qpos, 'q_proj'))
    k = flip(lin(k_in if kp is None else k_in + kp, 'k_proj'))
    v = flip(lin(v_in, 'v_proj'))
    H, dv = m.num_heads, m.head_dims
    q, k, v = q.unflatten(-1, (H, 2, dv // 2)), k.unflatten(-1, (-1, 2, dv // 2)), v.unflatten(-1, (-1, dv))
    G = H // k.shape[2]
    k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    e = (P['lambda_a'] * P['lambda_b']).sum(-1).exp()
    lam = e[0] - e[1] + m.lambda_init
    A = []
    for i in (0, 1):
        s = torch.einsum('bqhd,bkhd->bhqk', q[:, :, :, i], k[:, :, :, i]) / math.sqrt(dv // 2)
        A.append((s if hidden is None else s.masked_fill(hidden, -math.inf)).softmax(-1))
    o = torch.einsum('bhqk,bkhd->bqhd', A[0] - lam * A[1], v)
    o = torch.nn.functional.layer_norm(o, (dv,), P['head_norm.weight'], P['head_norm.bias'], m.head_norm.eps) * (1 - m.lambda_init)
    y = lin(flip(o.flatten(2)), 'out_proj') + (query if identity is None else identity)
    named = {**P, **dict(zip(('query', 'key', 'value', 'identity', 'query_pos', 'key_pos'), (query, key, value, identity, qpos, kpos)))}
    named = {n: t for n, t in named.items() if t is not None}
    return y.detach(), dict(zip(named, torch.autograd.grad(y, list(named.values()), go.double())))


@pytest.mark.parametrize('case', ['self', 'self batch_first shared', 'cross', 'cross padded batch_first'])
def test_module_gradients(case):
    """Training mode without dropout, f32.  Each of the module's Linears is a split-bf16 product (2^-16 of its terms' sizes, forward
    and both gradients), its bias gradient an f32 sum over at most 166 tokens (166 x 2^-24 < 2^-16 of its terms' sizes: what remains of
    k_proj.bias, whose gradient is zero because a softmax does not see it), everything else f32 operators within a few 2^-24.  So the bound of a gradient is what such errors do to
    it in the definition: the largest of three draws of errors of FULL size and random sign, by norm, times 4."""
    from unibev_amd import build_attention
    torch.manual_seed(11)
    batch_first, kv = 'batch_first' in case, 2 if 'shared' in case else None
    m = build_attention(dict(type='DifferentialAttention', embed_dims=128, num_heads=4, num_kv_heads=kv, batch_first=batch_first)).to(DEV).train()
    with torch.no_grad():
        m.head_norm.weight.uniform_(0.5, 1.5)
        m.head_norm.bias.uniform_(-0.5, 0.5)
        for lin in (m.q_proj, m.k_proj, m.v_proj, m.out_proj):
            lin.bias.uniform_(-0.5, 0.5)
    B, Nq, Nk = 2, 60, 83 if 'cross' in case else 60

    def tokens(n):
        return torch.randn(B, n, 128) if batch_first else torch.randn(n, B, 128)
    cross = 'cross' in case
    ins = [tokens(Nq), tokens(Nk) if cross else None, tokens(Nk) if cross else None, tokens(Nq) if cross else None, tokens(Nq),
           tokens(Nk) if cross else None]
    go = tokens(Nq)
    hidden, kw = None, {}
    if 'padded' in case:
        pad = torch.arange(Nk)[None] >= torch.tensor([[Nk], [50]])
        hidden, kw = pad[:, None, None], dict(key_padding_mask=pad.to(DEV))
    elif not cross:
        mask = torch.rand(Nq, Nq) < 0.3
        hidden, kw = mask, dict(attn_mask=mask.to(DEV))
    y0, ref = module_pass(m, ins, go, hidden, 0.0)
    noisy = [module_pass(m, ins, go, hidden, 2.0 ** -16, seed) for seed in (1, 2, 3)]
    dev = [None if t is None else t.to(DEV).requires_grad_() for t in ins]
    y = m(dev[0], key=dev[1], value=dev[2], identity=dev[3], query_pos=dev[4], key_pos=dev[5], **kw)
    y.backward(go.to(DEV))
    got = {**{n: p.grad for n, p in m.named_parameters()},
           **{n: t.grad for n, t in zip(('query', 'key', 'value', 'identity', 'query_pos', 'key_pos'), dev) if t is not None}}
    assert set(got) == set(ref)
    off = (y.detach().double().cpu() - y0).norm()
    assert off <= 4 * max((n[0] - y0).norm() for n in noisy), f'out: {off:.3e}'
    for name in ref:
        off = (got[name].double().cpu() - ref[name]).norm().item()
        bound = 4 * max((n[1][name] - ref[name]).norm().item() for n in noisy) + 2.0 ** -20 * ref[name].norm().item()
        assert off <= bound, f'{name}: off by {off:.3e}, bound {bound:.3e} (norm {ref[name].norm().item():.3e})'
