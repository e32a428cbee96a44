"""Cases of the token operators: attention over feature-map tokens (forward, few queries over a long
cache, training), the root-mean-square norm with the residual's addition (training, and with an 8-bit
output), and the 8-bit integer product with a scale for each token and channel.

``own = False`` computes each operator from elementary torch operations in 32 bits, rounded once at
the end; ``own = True`` makes the framework's calls.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-6


def listed():
    return [
        # the smallest call: the tokens of two 128x160 frames (16x20 grid), fp32, a padding mask over the keys
        dict(name='attn_small_fp32', op='attn', B=2, Lq=320, Lk=320, Hkv=4, G=1, D=32, dtype='fp32',
             causal=False, mask='keys', ragged=False),
        # inference over Sintel feature maps: 440x1024 frames at 1/8, 55x128 = 7040 tokens, 2 heads of 64
        dict(name='attn_sintel_bf16', op='attn', B=8, Lq=7040, Lk=7040, Hkv=2, G=1, D=64, dtype='bf16',
             causal=False, mask='none', ragged=False),
        # one new token of one stream over its cache: latency counts
        dict(name='attn_token_fp16', op='attn', B=1, Lq=1, Lk=4097, Hkv=8, G=1, D=64, dtype='fp16',
             causal=False, mask='none', ragged=False),
        # one new token of each of 32 streams over caches filled to different lengths, shared key heads
        dict(name='attn_cache_bf16', op='attn', B=32, Lq=1, Lk=16384, Hkv=8, G=4, D=128, dtype='bf16',
             causal=False, mask='none', ragged=True),
        # training over FlyingChairs feature maps: 368x496 frames at 1/8, 46x62 = 2852 tokens, batch 12,
        # the 128 context channels as one head
        dict(name='attn_train_chairs_bf16', op='attn_train', B=12, Lq=2852, Lk=2852, Hkv=1, G=1, D=128,
             dtype='bf16', causal=False, mask='none', ragged=False),
        # training on padded sequences of odd length, causal, shared key heads
        dict(name='attn_train_causal_fp16', op='attn_train', B=3, Lq=777, Lk=777, Hkv=2, G=4, D=64,
             dtype='fp16', causal=True, mask='none', ragged=True),
        # training norm over the tokens of a FlyingChairs batch (12 x 46 x 62), 256 channels
        dict(name='rms_train_chairs_bf16', op='rms_train', rows=34224, C=256, dtype='bf16', residual=True),
        # a short odd training call
        dict(name='rms_train_small_fp32', op='rms_train', rows=333, C=100, dtype='fp32', residual=True),
        # serving a long prompt: the norm that feeds an 8-bit product
        dict(name='rms_int8_prompt_bf16', op='rms_int8', rows=16384, C=4096, dtype='bf16', residual=True),
        # serving single tokens of 5 streams
        dict(name='rms_int8_token_fp16', op='rms_int8', rows=5, C=4096, dtype='fp16', residual=True),
        # 8-bit product of a prompt
        dict(name='int8_prompt_bf16', op='int8', M=8192, N=8192, K=4096, dtype='bf16', bias=False),
        # 8-bit product of single tokens of 5 streams: bound by reading the weights
        dict(name='int8_token_bf16', op='int8', M=5, N=4096, K=4096, dtype='bf16', bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case over the ranges of the listed ones."""
    op = rng.choice(['attn', 'attn', 'attn_cache', 'attn_train', 'attn_train', 'rms_train', 'rms_int8', 'int8'])
    dtype = rng.choice(['bf16', 'fp16', 'fp32'])
    limits = {c['op']: 0 for c in listed()}
    for c in listed():
        w = work(c)
        limits[c['op']] = max(limits[c['op']], w['flops'] + 100 * w['bytes'])
    while True:
        if op == 'attn_cache':
            c = dict(op='attn', B=_log(rng, 1, 32), Lq=rng.choice([1, 1, 2, 5]), Lk=_log(rng, 16, 32768),
                     Hkv=rng.choice([1, 2, 4, 8]), G=rng.choice([1, 2, 4, 7]), D=rng.choice([32, 64, 80, 128]),
                     dtype=dtype, causal=rng.random() < 0.5, mask=rng.choice(['none', 'none', 'keys']),
                     ragged=rng.random() < 0.5)
            c['Lq'] = min(c['Lq'], c['Lk'])
        elif op in ('attn', 'attn_train'):
            lk = _log(rng, 1, 8192)
            same = rng.random() < 0.6
            c = dict(op=op, B=_log(rng, 1, 12), Lq=lk if same else _log(rng, 1, 8192), Lk=lk,
                     Hkv=rng.choice([1, 2, 3, 4, 8]), G=rng.choice([1, 1, 2, 4]), D=rng.choice([32, 40, 64, 96, 128]),
                     dtype=dtype, causal=same and rng.random() < 0.4, mask=rng.choice(['none', 'none', 'keys', 'full']),
                     ragged=rng.random() < 0.4)
        elif op == 'rms_train':
            c = dict(op=op, rows=_log(rng, 1, 65536), C=_log(rng, 8, 8192), dtype=dtype, residual=rng.random() < 0.7)
        elif op == 'rms_int8':
            c = dict(op=op, rows=_log(rng, 1, 65536), C=_log(rng, 16, 8192), dtype=dtype, residual=rng.random() < 0.7)
        else:
            c = dict(op=op, M=_log(rng, 1, 16384), N=_log(rng, 16, 8192), K=_log(rng, 16, 8192), dtype=dtype,
                     bias=rng.random() < 0.5)
        w = work(c)
        limit = limits[c['op']]
        if dtype == 'fp32' and 'attn' in op:
            limit /= 16   # matrix products in 32 bits run at 1/16 of the 16-bit rate
        # the plain form holds the scores of all heads in 32 bits
        scores = c['B'] * c['Hkv'] * c['G'] * c['Lq'] * c['Lk'] if 'attn' in op else 0
        if w['flops'] + 100 * w['bytes'] <= limit and scores <= 8 * 2 * 7040 * 7040:
            return c


def _lengths(case):
    """How many keys each item of the batch holds: spread from about half of Lk to all of it."""
    B, Lk = case['B'], case['Lk']
    return [max(1, Lk - (Lk // 2) * ((5 * b) % B) // max(1, B)) for b in range(B)]


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch (a random mask counts as full)."""
    def causal(keys):
        # query i sits at position first + i and sees the keys up to its own position
        first = keys - case['Lq'] if case['Lq'] < case['Lk'] else 0
        return sum(min(keys, max(0, first + i + 1)) for i in range(case['Lq']))
    held = _lengths(case) if case['ragged'] else [case['Lk']] * case['B']
    return sum(causal(n) if case['causal'] else case['Lq'] * n for n in held)


def work(case):
    size = {'bf16': 2, 'fp16': 2, 'fp32': 4}[case['dtype']]
    if case['op'] in ('attn', 'attn_train'):
        H = case['Hkv'] * case['G']
        keys = sum(_lengths(case)) if case['ragged'] else case['B'] * case['Lk']
        q = case['B'] * case['Lq'] * H * case['D'] * size
        kv = 2 * keys * case['Hkv'] * case['D'] * size
        mask = {'none': 0, 'keys': case['B'] * case['Lk'], 'full': case['B'] * case['Lq'] * case['Lk']}[case['mask']]
        f = 4 * case['D'] * H * _pairs(case)
        if case['op'] == 'attn':
            return {'bytes': 2 * q + kv + mask, 'flops': f}
        return {'bytes': 4 * q + 2 * kv + mask, 'flops': f * 3.5}
    if case['op'] == 'rms_train':
        n = case['rows'] * case['C']
        return {'bytes': (7 if case['residual'] else 4) * n * size, 'flops': 12 * n}
    if case['op'] == 'rms_int8':
        n = case['rows'] * case['C']
        return {'bytes': (3 if case['residual'] else 1) * n * size + n + 4 * case['rows'], 'flops': 6 * n}
    M, N, K = case['M'], case['N'], case['K']
    return {'bytes': M * K + N * K + M * N * size, 'flops': 2 * M * N * K}


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case['dtype']]

    def rn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).to(dt)

    s = {'case': case}
    if case['op'] in ('attn', 'attn_train'):
        B, Lq, Lk, Hkv, G, D = (case[n] for n in ('B', 'Lq', 'Lk', 'Hkv', 'G', 'D'))
        if Lq == Lk:
            # the three parts of one projection's output, as it leaves the product
            qkv = rn(B, Lq, (G + 2) * Hkv, D, scale=1.3)
            q, k, v = qkv.split([G * Hkv, Hkv, Hkv], dim=2)
        else:
            q, k, v = rn(B, Lq, G * Hkv, D, scale=1.3), rn(B, Lk, Hkv, D, scale=1.3), rn(B, Lk, Hkv, D)
        s['lengths'] = s['mask'] = s['q_offset'] = None
        if case['ragged']:
            lengths = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)
            # what lies behind a sequence's end was never written: it must not be read
            behind = torch.arange(Lk, device=dev) >= lengths[:, None]
            k[behind] = float('nan')
            v[behind] = float('nan')
            s['lengths'] = lengths
            if Lq < Lk:
                s['q_offset'] = lengths - Lq
        if case['mask'] == 'keys':
            s['mask'] = torch.rand(B, 1, 1, Lk, generator=g, device=dev) < 0.9
            # padding holds anything
            k[~s['mask'][:, 0, 0]] = float('inf')
            v[~s['mask'][:, 0, 0]] = float('nan')
        elif case['mask'] == 'full':
            m = torch.rand(B, 1, Lq, Lk, generator=g, device=dev) < 0.8
            m[:, :, Lq // 2] = False   # a row without any key
            s['mask'] = m
        s['q'], s['k'], s['v'] = q, k, v
        if case['op'] == 'attn_train':
            s['q'], s['k'], s['v'] = (t.detach().requires_grad_(True) for t in (q, k, v))
            s['dout'] = rn(B, Lq, G * Hkv, D, scale=0.1)
    elif case['op'] in ('rms_train', 'rms_int8'):
        rows, C = case['rows'], case['C']
        s['x'] = rn(rows, C)
        s['residual'] = rn(rows, C, scale=2.0) if case['residual'] else None
        s['weight'] = 1 + 0.2 * torch.randn(C, generator=g, device=dev)
        if case['op'] == 'rms_train':
            s['x'].requires_grad_(True)
            s['weight'].requires_grad_(True)
            if case['residual']:
                s['residual'].requires_grad_(True)
                s['dh'] = rn(rows, C, scale=0.1)
            s['dy'] = rn(rows, C, scale=0.1)
    else:
        M, N, K = case['M'], case['N'], case['K']
        s['x'] = torch.randn(M, K, generator=g, device=dev).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
        s['w'] = torch.randn(N, K, generator=g, device=dev).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
        s['xs'] = torch.rand(M, generator=g, device=dev) * 0.04 + 0.01
        s['ws'] = torch.rand(N, generator=g, device=dev) * 0.001 + 0.0002
        s['bias'] = torch.randn(N, generator=g, device=dev) if case['bias'] else None
    return s


# ---------------------------------------------------------------------------- plain forms
def _visible(s):
    """(B, H or 1, Lq, Lk) truth values: which keys each query sees; None if all."""
    c, dev = s['case'], s['q'].device
    B, Lq, Lk = c['B'], c['Lq'], c['Lk']
    see = None
    j = torch.arange(Lk, device=dev)
    if s['lengths'] is not None:
        see = (j < s['lengths'][:, None])[:, None, None]
    if c['causal']:
        first = s['q_offset'] if s['q_offset'] is not None else torch.full((B,), Lk - Lq, device=dev)
        pos = first[:, None] + torch.arange(Lq, device=dev)
        low = (j <= pos[..., None])[:, None]
        see = low if see is None else see & low
    if s['mask'] is not None:
        see = s['mask'] if see is None else see & s['mask']
    return see


def _hidden(s):
    """(B, Lk) truth values: keys that no query sees, whatever they hold; None if there are none."""
    hidden = None
    if s['lengths'] is not None:
        hidden = torch.arange(s['case']['Lk'], device=s['q'].device) >= s['lengths'][:, None]
    if s['case']['mask'] == 'keys':
        pad = ~s['mask'][:, 0, 0]
        hidden = pad if hidden is None else hidden | pad
    return hidden


def _plain_attention(s, grads):
    c = s['case']
    B, Lq, Lk, Hkv, G, D = (c[n] for n in ('B', 'Lq', 'Lk', 'Hkv', 'G', 'D'))
    dt = s['q'].dtype
    scale = 1 / math.sqrt(D)

    def heads(t):   # (B, L, n, D) -> (B, n, L, D) in 32 bits
        return t.detach().float().transpose(1, 2).contiguous()
    q, k, v = heads(s['q']), heads(s['k']), heads(s['v'])
    hidden = _hidden(s)
    if hidden is not None:
        k, v = k.masked_fill(hidden[:, None, :, None], 0), v.masked_fill(hidden[:, None, :, None], 0)
    q = q.view(B, Hkv, G * Lq, D)   # the heads that share keys lie together
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    see = _visible(s)
    if see is not None:
        see = see.expand(B, see.shape[1], Lq, Lk).unsqueeze(2)
        p = p.view(B, Hkv, G, Lq, Lk).masked_fill_(~see, -math.inf).view(B, Hkv, G * Lq, Lk)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p, v)

    def back(t, n, L):   # (B, n, L, D) -> (B, L, n, D), rounded
        return t.reshape(B, n, L, D).transpose(1, 2).to(dt)
    if not grads:
        return back(o, G * Hkv, Lq)
    do = heads(s['dout']).view(B, Hkv, G * Lq, D)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return {'out': back(o, G * Hkv, Lq), 'dq': back(dq, G * Hkv, Lq), 'dk': back(dk, Hkv, Lk), 'dv': back(dv, Hkv, Lk)}


def _plain_norm(s):
    """h (rounded to its type, as it is kept), 1 / rms, and the normalised weighted rows, in 32 bits."""
    x = s['x'].detach()
    h = x.float() if s['residual'] is None else (x.float() + s['residual'].detach().float()).to(x.dtype).float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    return h, rstd, h * rstd * s['weight'].detach()


def _plain_rms_train(s):
    dt = s['x'].dtype
    h, rstd, y = _plain_norm(s)
    dy = s['dy'].float()
    g = dy * s['weight'].detach()
    dx = rstd * (g - h * rstd.square() * (g * h).mean(-1, keepdim=True))
    if s['residual'] is not None:
        dx = dx + s['dh'].float()
    dw = (dy * h * rstd).sum(0)
    r = {'y': y.to(dt), 'dx': dx.to(dt), 'dw': dw}
    if s['residual'] is not None:
        r['h'] = h.to(dt)
        r['dresidual'] = dx.to(dt)
    return r


def _plain_rms_int8(s):
    h, _, y = _plain_norm(s)
    top = y.abs().amax(-1, keepdim=True)
    q = torch.round(y * torch.where(top == 0, torch.zeros_like(top), 127 / top))
    scale = top / 127
    r = {'y': (q * scale).to(s['x'].dtype if s['x'].dtype != torch.float32 else torch.float16), 'scale': scale.view(-1)}
    if s['residual'] is not None:
        r['h'] = h.to(s['x'].dtype)
    return r


def _plain_int8(s):
    acc = torch.matmul(s['x'].float(), s['w'].float().t())
    y = acc * s['xs'][:, None] * s['ws']
    if s['bias'] is not None:
        y = y + s['bias']
    return y.to(DTYPES[s['case']['dtype']])


def run(state):
    s = state
    op = s['case']['op']
    if own:
        if op in ('attn', 'attn_train'):
            from pytorch_raft_amd.ops.attention import attention
            out = attention(s['q'], s['k'], s['v'], causal=s['case']['causal'], mask=s['mask'],
                            lengths=s['lengths'], q_offset=s['q_offset'])
            if op == 'attn':
                return out
            dq, dk, dv = torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['dout'])
            return {'out': out, 'dq': dq, 'dk': dk, 'dv': dv}
        if op == 'rms_train':
            from pytorch_raft_amd.ops.rms_norm import rms_norm
            if s['residual'] is None:
                y = rms_norm(s['x'], s['weight'], eps=EPS)
                dx, dw = torch.autograd.grad(y, (s['x'], s['weight']), s['dy'])
                return {'y': y, 'dx': dx, 'dw': dw}
            y, h = rms_norm(s['x'], s['weight'], residual=s['residual'], eps=EPS)
            dx, dr, dw = torch.autograd.grad((y, h), (s['x'], s['residual'], s['weight']), (s['dy'], s['dh']))
            return {'y': y, 'h': h, 'dx': dx, 'dresidual': dr, 'dw': dw}
        if op == 'rms_int8':
            from pytorch_raft_amd.ops.rms_norm import rms_norm_int8
            q, scale, h = rms_norm_int8(s['x'], s['weight'], residual=s['residual'], eps=EPS)
            # the values that the 8 bits stand for (fp16 holds 8 bits times a scale whole enough to compare)
            y = torch.empty(q.shape, device=q.device, dtype=torch.float16 if s['x'].dtype == torch.float32 else s['x'].dtype)
            torch.mul(q, scale[:, None], out=y)
            return {'y': y, 'scale': scale} if h is None else {'y': y, 'scale': scale, 'h': h}
        from pytorch_raft_amd.ops.int8 import int8_linear
        return int8_linear(s['x'], s['xs'], s['w'], s['ws'], bias=s['bias'], out_dtype=DTYPES[s['case']['dtype']])
    if op in ('attn', 'attn_train'):
        return _plain_attention(s, op == 'attn_train')
    return {'rms_train': _plain_rms_train, 'rms_int8': _plain_rms_int8, 'int8': _plain_int8}[op](s)


# ---------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op in ('attn', 'attn_train'):
        B, Lq, Lk, Hkv, G, D = (case[n] for n in ('B', 'Lq', 'Lk', 'Hkv', 'G', 'D'))
        dev = s['q'].device
        out = torch.zeros(B, Lq, Hkv * G, D, dtype=torch.float64, device=dev)
        grads = [torch.zeros(t.shape, dtype=torch.float64, device=dev) for t in (s['q'], s['k'], s['v'])]
        at = torch.arange(Lk, device=dev)
        for b in range(B):
            n = Lk if s['lengths'] is None else int(s['lengths'][b])
            first = Lk - Lq if s['q_offset'] is None else int(s['q_offset'][b])
            see = torch.ones(Lq, n, dtype=torch.bool, device=dev)
            if case['causal']:
                see &= at[:n] <= torch.arange(first, first + Lq, device=dev)[:, None]
            if s['mask'] is not None:
                see &= s['mask'][b, 0].expand(Lq, Lk)[:, :n]
            some, used = see.any(-1), see.any(0)
            for h in range(Hkv * G):
                need = op == 'attn_train'
                q, k, v = (t.detach()[b, :m, i].double().requires_grad_(need)
                           for t, m, i in ((s['q'], Lq, h), (s['k'], n, h // G), (s['v'], n, h // G)))
                a = (q[some] @ k[used].t()) / math.sqrt(D)
                a = a.masked_fill(~see[some][:, used], -math.inf)
                o = torch.softmax(a, -1) @ v[used]
                out[b, some, h] = o.detach()
                if need and bool(some.any()):
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s['dout'][b, some, h].double())
                    grads[0][b, :, h] += dq
                    grads[1][b, :n, h // G] += dk
                    grads[2][b, :n, h // G] += dv
        return out if op == 'attn' else {'out': out, 'dq': grads[0], 'dk': grads[1], 'dv': grads[2]}
    if op in ('rms_train', 'rms_int8'):
        need = op == 'rms_train'
        h = s['x'].detach()
        if s['residual'] is not None:
            h = (h.double() + s['residual'].detach().double()).to(h.dtype)
        h = h.double().requires_grad_(need)
        w = s['weight'].detach().double().requires_grad_(need)
        y = h / torch.sqrt(torch.mean(h * h, dim=-1, keepdim=True) + EPS) * w
        if need:
            dh, dw = torch.autograd.grad(y, (h, w), s['dy'].double())
            if s['residual'] is None:
                return {'y': y.detach(), 'dx': dh, 'dw': dw}
            dh = dh + s['dh'].double()
            return {'y': y.detach(), 'h': h.detach(), 'dx': dh, 'dresidual': dh, 'dw': dw}
        scale = y.abs().max(-1).values / 127
        q = torch.round(y / scale.clamp(min=1e-300)[:, None])
        r = {'y': q * scale[:, None], 'scale': scale}
        return r if s['residual'] is None else {**r, 'h': h}
    y = (s['x'].double() @ s['w'].double().t()) * s['xs'].double()[:, None] * s['ws'].double()
    return y if s['bias'] is None else y + s['bias'].double()
