"""Cases of the transformer operators of the object-query decoder: differential attention, layer norm, dropout.

``listed()`` names real calls, ``draw(rng)`` draws more of the same ranges, ``run(state)`` makes one pass through an operator —
with the framework's kernels where ``own`` is true, else in plain torch operations — and ``exact(case, seed)`` gives the same
outputs from the definitions in 64 bits.

Definitions (f32 arithmetic or wider, one rounding to the input's type at the end):

  attention   A_m = softmax_j(scale q_m . k_m + mask), m = 1, 2;  out = (D o (A_1 - lam_h A_2)) v;  a row that sees no key is 0
  norm        y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis
  dropout     y = identity + D o x
  D           keep(element) / (1 - t / 2^16), t = p 2^16 rounded: the element is kept where its 16-bit field is >= t.  The
              field e of group g is bits 16 e .. 16 e + 15 of mix64(seed, g); dropout: element i is field i % 4 of group i // 4;
              attention: key j of row r = (b H + h) Nq + i is field j % 4 of group r ceil(Nk / 4) + j // 4.
"""
import math

import numpy as np
import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
M64 = (1 << 64) - 1


def listed():
    return [
        # the decoder's self-attention slot: 900 object queries, 256 channels as 4 heads of two 32-wide maps, attention dropout 0.1
        attn('attn_decoder_bf16_train', 'bf16', B=2, H=4, Hk=4, Nq=900, Nk=900, Dh=32, Dv=64, p=0.1, train=True),
        # the same slot in the framework's default f32, eight narrow heads, a batch whose second sample is padded
        attn('attn_decoder_f32_train', 'f32', B=2, H=8, Hk=8, Nq=900, Nk=900, Dh=16, Dv=32, p=0.1, train=True, mask='padding'),
        # BEV tokens among themselves: a 100 x 100 grid, the long end
        attn('attn_bev_grid_bf16_train', 'bf16', B=1, H=4, Hk=4, Nq=10000, Nk=10000, Dh=32, Dv=64, train=True),
        # wide heads, shared key / value heads, an odd causal sequence
        attn('attn_causal_shared_f16_train', 'f16', B=2, H=8, Hk=2, Nq=2047, Nk=2047, Dh=64, Dv=128, train=True, mask='causal'),
        # one new query against the tokens of a 200 x 200 BEV map, ragged batch
        attn('attn_one_query_bev_bf16', 'bf16', B=8, H=4, Hk=4, Nq=1, Nk=40000, Dh=32, Dv=64, mask='padding'),
        # the smallest call: one query, a few hundred keys, latency
        attn('attn_one_query_small_f16', 'f16', B=1, H=8, Hk=8, Nq=1, Nk=257, Dh=32, Dv=64),
        # the norms of the BEV encoder: 2 x 200 x 200 tokens of 256 channels
        norm('norm_bev_f32_train', 'f32', R=80000, C=256, train=True),
        # a norm of the decoder: latency
        norm('norm_decoder_bf16', 'bf16', R=900, C=256),
        # odd rows and an odd width
        norm('norm_odd_f16_train', 'f16', R=5001, C=1021, train=True),
        # hidden activations of the BEV encoder's FFN width, with a residual
        drop('drop_bev_bf16_train', 'bf16', n=(80000, 512), p=0.1, identity=True, train=True),
        # the decoder's residual: latency
        drop('drop_decoder_f32', 'f32', n=(900, 2, 256), p=0.1, identity=True),
        # an odd number of elements, no residual
        drop('drop_odd_f16_train', 'f16', n=(1000003,), p=0.3, identity=False, train=True),
    ]


def attn(name, dtype, B, H, Hk, Nq, Nk, Dh, Dv, p=0.0, train=False, mask='none'):
    return dict(name=name, op='attention', dtype=dtype, B=B, H=H, Hk=Hk, Nq=Nq, Nk=Nk, Dh=Dh, Dv=Dv, p=p, train=train, mask=mask)


def norm(name, dtype, R, C, train=False, affine=True):
    return dict(name=name, op='norm', dtype=dtype, R=R, C=C, train=train, affine=affine)


def drop(name, dtype, n, p, identity, train=False):
    return dict(name=name, op='dropout', dtype=dtype, shape='x'.join(map(str, n)), p=p, identity=identity, train=train)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    op = rng.choice(['attention', 'attention', 'norm', 'dropout'])
    if op == 'norm':
        C = _log(rng, 1, 8192)
        c = norm('', dtype, R=_log(rng, 1, min(200000, 80000 * 256 // C)), C=C, train=rng.random() < 0.6, affine=rng.random() < 0.8)
    elif op == 'dropout':
        c = drop('', dtype, (_log(rng, 1, 20000000),), rng.choice([0.1, 0.25, 0.5, 0.9]), rng.random() < 0.5, rng.random() < 0.5)
    else:
        g, Hk = rng.choice([1, 1, 2, 4]), rng.choice([1, 2, 3, 4])
        Dh = rng.choice([16, 20, 32, 40, 64, 96, 128])
        Dv = Dh * rng.choice([1, 2, 2])
        if rng.random() < 0.3:                      # a few queries against many keys
            Nq, Nk, train = rng.choice([1, 1, 2, 5]), _log(rng, 1, 60000), False
        else:
            train = rng.random() < 0.6
            Nq = _log(rng, 1 + train, 4096)
            Nk = Nq if rng.random() < 0.6 else _log(rng, 1 + train, 4096)
        B = rng.choice([1, 2, 3])
        mask = rng.choice(['none', 'causal', 'padding', 'bool', 'float'])
        top = 10000 * 10000 * 4 * 128 // (4 if dtype == 'f32' else 1)
        while B * Hk * g * Nq * Nk * (2 * Dh + Dv) > top and (B > 1 or Hk > 1 or g > 1):
            B, Hk, g = (B - 1, Hk, g) if B > 1 else (B, Hk - 1, g) if Hk > 1 else (B, Hk, 1)
        c = attn('', dtype, B, Hk * g, Hk, Nq, Nk, Dh, Dv, rng.choice([0.0, 0.0, 0.1]) if train else 0.0, train, mask)
    del c['name']
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Keys of each sample of a padded batch: all of them, then fewer."""
    return [case['Nk'] - (b * case['Nk']) // (2 * case['B']) for b in range(case['B'])]


def _shape(case):
    return tuple(int(s) for s in case['shape'].split('x'))


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dt = TYPES[case['dtype']]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device='cuda', dtype=torch.float32) * std + mean).to(dtype)

    s = dict(case=case, drop_seed=seed * 7919 + 12345)
    if case['op'] == 'attention':
        B, H, Hk, Nq, Nk, Dh, Dv = (case[k] for k in ('B', 'H', 'Hk', 'Nq', 'Nk', 'Dh', 'Dv'))
        s['q'] = randn(B, Nq, H, 2, Dh, std=1.5)
        s['k'] = randn(B, Nk, Hk, 2, Dh)
        s['v'] = randn(B, Nk, Hk, Dv)
        s['lam'] = randn(H, std=0.1, mean=0.5, dtype=torch.float32)
        leaves = ['q', 'k', 'v', 'lam']
        if case['train']:
            s['g'] = randn(B, Nq, H, Dv)
        if case['mask'] == 'padding':
            n = torch.tensor(_lengths(case), device='cuda')
            s['padding'] = torch.arange(Nk, device='cuda')[None] >= n[:, None]
        elif case['mask'] == 'bool':                # 30 % of the pairs hidden, every 97th row sees nothing
            hidden = torch.rand(Nq, Nk, generator=gen, device='cuda') < 0.3
            hidden[::97] = True
            s['mask'] = hidden
        elif case['mask'] == 'float':               # a bias that falls with the distance, another slope for each head
            far = (torch.arange(Nq, device='cuda')[:, None] - torch.arange(Nk, device='cuda')[None]).abs().float()
            s['mask'] = (-far * 2.0 ** -torch.arange(1, H + 1, device='cuda')[:, None, None])[None]
    elif case['op'] == 'norm':
        R, C = case['R'], case['C']
        s['x'] = randn(R, C, std=2.0, mean=0.5)
        s['gamma'] = randn(C, std=0.1, mean=1.0, dtype=torch.float32) if case['affine'] else None
        s['beta'] = randn(C, std=0.1, dtype=torch.float32) if case['affine'] else None
        leaves = ['x', 'gamma', 'beta'] if case['affine'] else ['x']
        if case['train']:
            s['g'] = randn(R, C)
    else:
        shape = _shape(case)
        s['x'] = randn(*shape)
        s['identity'] = randn(*shape) if case['identity'] else None
        leaves = ['x', 'identity'] if case['identity'] else ['x']
        if case['train']:
            s['g'] = randn(*shape)
    s['leaves'] = leaves
    if case['train']:
        for n in leaves:
            s[n].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state['case']
    if not own:
        with torch.no_grad():
            return {'attention': _plain_attention, 'norm': _plain_norm, 'dropout': _plain_dropout}[case['op']](state)
    from unibev_amd import functional as UF
    with torch.set_grad_enabled(case['train']):
        if case['op'] == 'attention':
            y = UF.diff_attention(state['q'], state['k'], state['v'], state['lam'], attn_mask=state.get('mask'),
                                  key_padding_mask=state.get('padding'), causal=case['mask'] == 'causal', p=case['p'],
                                  training=case['train'], seed=state['drop_seed'])
        elif case['op'] == 'norm':
            y = UF.layer_norm(state['x'], state['gamma'], state['beta'], eps=1e-5)
        else:
            y = UF.dropout(state['x'], case['p'], training=True, identity=state['identity'], seed=state['drop_seed'])
        if not case['train']:
            return y
        return (y.detach(), *torch.autograd.grad(y, [state[n] for n in state['leaves']], state['g']))


def _signed(v):
    v &= M64
    return v - (1 << 64) if v >> 63 else v


def _mix64(seed, group):
    """The counter-based generator on int64 tensors (two's complement products wrap as unsigned ones do)."""
    def shift(z, n):
        return (z >> n) & ((1 << (64 - n)) - 1)
    z = group + _signed(seed * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019)
    z = (z ^ shift(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ shift(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ shift(z, 31)


def _fields(seed, first, rows, cols):
    """16-bit fields of ``rows`` x ``cols`` elements, each row starting a new group; groups numbered from ``first``."""
    n4 = (cols + 3) // 4
    mix = _mix64(seed, torch.arange(first, first + rows * n4, device='cuda').view(rows, n4))
    e = torch.arange(0, 64, 16, device='cuda')
    return ((mix[..., None] >> e) & 0xFFFF).view(rows, 4 * n4)[:, :cols]


def _keep_scale(p):
    t = int(p * 65536 + 0.5)
    return t, 65536.0 / (65536.0 - t)


def _plain_dropout(s):
    case, x = s['case'], s['x']
    t, scale = _keep_scale(case['p'])
    D = (_fields(s['drop_seed'], 0, 1, x.numel()).view(x.shape) >= t).float() * scale
    y = x.float() * D
    if case['identity']:
        y = s['identity'].float() + y
    y = y.to(x.dtype)
    if not case['train']:
        return y
    gx = (s['g'].float() * D).to(x.dtype)
    return (y, gx, s['g']) if case['identity'] else (y, gx)


def _plain_norm(s):
    x, case = s['x'].float(), s['case']
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    h = d * rstd
    y = (h * s['gamma'] + s['beta'] if case['affine'] else h).to(s['x'].dtype)
    if not case['train']:
        return y
    g = s['g'].float()
    gh = g * s['gamma'] if case['affine'] else g
    gx = (rstd * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True))).to(s['x'].dtype)
    return (y, gx, (g * h).sum(0), g.sum(0)) if case['affine'] else (y, gx)


def _plain_attention(s):
    """All heads at once where their score matrices are small, else head by head."""
    case = s['case']
    B, H, Hk, Nq, Nk = (case[k] for k in ('B', 'H', 'Hk', 'Nq', 'Nk'))
    g = H // Hk
    dt = s['q'].dtype
    q = s['q'].permute(0, 2, 3, 1, 4).float()                                     # B H 2 Nq Dh
    k = s['k'].permute(0, 2, 3, 1, 4).float().repeat_interleave(g, dim=1)
    v = s['v'].permute(0, 2, 1, 3).float().repeat_interleave(g, dim=1)
    go = s['g'].permute(0, 2, 1, 3).float() if case['train'] else None
    if B * H * Nq * Nk <= 1 << 27:
        parts = _plain_heads(s, q, k, v, go, 0, 0)
    else:
        parts = [[_plain_heads(s, q[b:b + 1, h:h + 1], k[b:b + 1, h:h + 1], v[b:b + 1, h:h + 1],
                               None if go is None else go[b:b + 1, h:h + 1], b, h) for h in range(H)] for b in range(B)]
        parts = [torch.cat([torch.cat([p[i] for p in row], 1) for row in parts], 0) for i in range(len(parts[0][0]))]
    out = parts[0].permute(0, 2, 1, 3).to(dt)
    if not case['train']:
        return out
    _, gq, gk, gv, gl = parts
    gk, gv = (t.view(B, Hk, g, *t.shape[2:]).sum(2) for t in (gk, gv))            # shared heads: sum over their queries' heads
    return out, gq.permute(0, 3, 1, 2, 4).to(dt), gk.permute(0, 3, 1, 2, 4).to(dt), gv.permute(0, 2, 1, 3).to(dt), gl.sum(0)


def _plain_heads(s, q, k, v, go, b0, h0):
    case = s['case']
    B, H = q.shape[:2]
    Nq, Nk, scale = case['Nq'], case['Nk'], case['Dh'] ** -0.5
    hidden, bias = None, None
    if case['mask'] == 'causal':
        hidden = torch.arange(Nk, device='cuda')[None] - torch.arange(Nq, device='cuda')[:, None] > Nk - Nq
    elif case['mask'] == 'padding':
        hidden = s['padding'][b0:b0 + B, None, None]
    elif case['mask'] == 'bool':
        hidden = s['mask']
    elif case['mask'] == 'float':
        bias = s['mask'][:, h0:h0 + H]
    maps = []
    for m in (0, 1):
        t = torch.matmul(q[:, :, m] * scale, k[:, :, m].transpose(-1, -2).contiguous())
        if bias is not None:
            t = t + bias
        if hidden is not None:
            t = t.masked_fill(hidden, -math.inf)
        top = t.amax(-1, keepdim=True).clamp_min(-3e38)                           # (a row of -inf keeps exp at 0)
        e = torch.exp(t - top)
        maps.append(e / e.sum(-1, keepdim=True).clamp_min(1e-30))
    A1, A2 = maps
    lam = s['lam'].detach()[h0:h0 + H, None, None]
    A = A1 - lam * A2
    D = None
    if case['p'] > 0:
        t, up = _keep_scale(case['p'])
        n4 = (Nk + 3) // 4
        first = (b0 * case['H'] + h0) * Nq * n4
        D = (_fields(s['drop_seed'], first, B * H * Nq, Nk) >= t).view(B, H, Nq, Nk).float() * up
        A = A * D
    out = torch.matmul(A, v)
    if go is None:
        return (out,)
    gv = torch.matmul(A.transpose(-1, -2).contiguous(), go)
    gA = torch.matmul(go, v.transpose(-1, -2).contiguous())
    if D is not None:
        gA = gA * D
    d1 = (A1 * gA).sum(-1, keepdim=True)
    d2 = (A2 * gA).sum(-1, keepdim=True)
    gs1 = A1 * (gA - d1) * scale
    gs2 = A2 * (d2 - gA) * lam * scale
    gq = torch.stack([torch.matmul(gs1, k[:, :, 0]), torch.matmul(gs2, k[:, :, 1])], 2)
    gk = torch.stack([torch.matmul(gs1.transpose(-1, -2).contiguous(), q[:, :, 0]),
                      torch.matmul(gs2.transpose(-1, -2).contiguous(), q[:, :, 1])], 2)
    return out, gq, gk, gv, -d2.sum((-1, -2))


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _kept(seed, first, n):
    """Fields of ``n`` groups from ``first``, in unsigned numpy arithmetic."""
    with np.errstate(over='ignore'):
        z = np.arange(first, first + n, dtype=np.uint64) + np.uint64((seed * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019) & M64)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    return z.astype('<u8').view('<u2').astype(np.int64)


def exact(case, seed):
    s = prepare(case, seed)
    leaf = {n: s[n].detach().double().requires_grad_(case['train']) for n in s['leaves']}
    g = s['g'].double() if case['train'] else None
    t16 = int(case.get('p', 0) * 65536 + 0.5)
    if case['op'] == 'norm':
        x = leaf['x']
        y = (x - x.mean(-1, keepdim=True)) * (x.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
        if case['affine']:
            y = y * leaf['gamma'] + leaf['beta']
    elif case['op'] == 'dropout':
        x = leaf['x']
        n = x.numel()
        kept = torch.from_numpy(_kept(s['drop_seed'], 0, (n + 3) // 4)[:n] >= t16).cuda().view(x.shape)
        y = torch.where(kept, x * (65536.0 / (65536.0 - t16)), torch.zeros_like(x))
        if case['identity']:
            y = leaf['identity'] + y
    else:
        return _exact_attention(case, s, leaf, g, t16)
    if not case['train']:
        return y
    return (y.detach(), *torch.autograd.grad(y, [leaf[n] for n in s['leaves']], g))


def _exact_attention(case, s, leaf, g, t16):
    """Head by head, the definition as it stands; gradients by differentiation of it."""
    B, H, Hk, Nq, Nk, Dh = (case[k] for k in ('B', 'H', 'Hk', 'Nq', 'Nk', 'Dh'))
    out = torch.zeros(B, Nq, H, case['Dv'], dtype=torch.float64, device='cuda')
    for b in range(B):
        for h in range(H):
            q, k, v = leaf['q'][b, :, h], leaf['k'][b, :, h * Hk // H], leaf['v'][b, :, h * Hk // H]
            see = torch.ones(Nq, Nk, dtype=torch.bool, device='cuda')
            if case['mask'] == 'causal':
                see = see.tril(Nk - Nq)
            elif case['mask'] == 'padding':
                see[:, _lengths(case)[b]:] = False
            elif case['mask'] == 'bool':
                see = ~s['mask']
            live = see.any(-1, keepdim=True)
            A = []
            for m in (0, 1):
                t = q[:, m] @ k[:, m].t() / math.sqrt(Dh)
                if case['mask'] == 'float':
                    t = t + s['mask'][0, h].double()
                A.append(torch.softmax(torch.where(see | ~live, t, torch.full_like(t, -math.inf)), -1) * live)
            A = A[0] - leaf['lam'][h] * A[1]
            if t16:
                n4 = (Nk + 3) // 4
                kept = _kept(s['drop_seed'], (b * H + h) * Nq * n4, Nq * n4).reshape(Nq, 4 * n4)[:, :Nk] >= t16
                A = torch.where(torch.from_numpy(kept).cuda(), A * (65536.0 / (65536.0 - t16)), torch.zeros_like(A))
            o = A @ v
            out[b, :, h] = o.detach()
            if case['train']:
                o.backward(g[b, :, h])
    if not case['train']:
        return out
    return (out, *(leaf[n].grad for n in s['leaves']))


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'norm':
        n = case['R'] * case['C']
        w = 8 * case['C'] * case['affine']
        return {'bytes': e * n * (4 if case['train'] else 2) + w * (2 if case['train'] else 1), 'flops': n * (22 if case['train'] else 8)}
    if case['op'] == 'dropout':
        n = math.prod(_shape(case))
        # forward x (, identity) -> y; backward g -> gx (the residual's gradient is g itself)
        return {'bytes': e * n * (2 + case['identity'] + 2 * case['train']), 'flops': n * (2 + case['train'])}
    B, H, Hk, Nq, Nk, Dh, Dv = (case[k] for k in ('B', 'H', 'Hk', 'Nq', 'Nk', 'Dh', 'Dv'))
    keys = B * Nk
    if case['mask'] == 'causal':
        pairs = B * sum(max(0, min(Nk, i + 1 + Nk - Nq)) for i in range(Nq))
    elif case['mask'] == 'padding':
        keys = sum(_lengths(case))
        pairs = keys * Nq
    elif case['mask'] == 'bool':
        pairs = int(B * Nq * Nk * 0.7)
    else:
        pairs = B * Nq * Nk
    per_q, per_k = H * (2 * Dh + Dv), Hk * (2 * Dh + Dv)            # q and out; k and v
    nbytes = e * (B * Nq * per_q + keys * per_k) + 4 * H
    if case['mask'] == 'padding':
        nbytes += B * Nk
    elif case['mask'] == 'bool':
        nbytes += Nq * Nk
    elif case['mask'] == 'float':
        nbytes += 4 * H * Nq * Nk
    flops = pairs * H * (4 * Dh + 2 * Dv)                           # q k for each map, the difference times v
    if case['train']:
        nbytes += e * (B * Nq * per_q + B * Nk * per_k) + 4 * H     # + grad_out, grad_q; grad_k, grad_v
        flops += pairs * H * (8 * Dh + 4 * Dv)
    return {'bytes': nbytes, 'flops': flops}
