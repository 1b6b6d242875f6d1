"""What is measured of the training and serving operators on query tokens: LayerNorm with its residual add (forward and
backward) and attention of a set of queries to the states of another sequence (forward, backward, and single queries).

`run` computes a case in its plain form from elementary torch operations in 32 bits, or, where `own` is true, through the
framework's entry points (`deepinteraction_amd.ops`)."""
import math

import torch

own = False

_T = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}


def listed():
    return [
        # LayerNorm(x + branch) over the 200 object queries of one sample, the post-norm step of the decoder in a float32 training step
        dict(name='norm queries', op='norm', mode='train', rows=200, C=128, x='f32', res='f32', w='f32', y='f32', total=False),
        # the same step over the 1200 rays x 60 radii of six cameras under autocast: float32 stream, half-precision branch
        dict(name='norm rays mixed', op='norm', mode='train', rows=72000, C=128, x='f32', res='f16', w='f32', y='f32', total=False),
        # a pre-norm residual stream of a wide model: the sum is carried on and receives a gradient of its own
        dict(name='norm wide', op='norm', mode='train', rows=8192, C=4096, x='bf16', res='bf16', w='bf16', y='bf16', total=True),
        # the first stage of the Swin image backbone over six 112 x 200 maps, inference
        dict(name='norm swin', op='norm', mode='serve', rows=134400, C=96, x='f16', res='f16', w='f16', y='f16', total=True),
        # the decoder layer's object queries on the 180 x 180 BEV map, one sample, float32 training step
        dict(name='attend map', op='attend', mode='train', dtype='f32', B=1, L=200, S=32400, H=8, G=1, D=16, mask='none'),
        # the same for two samples in half precision
        dict(name='attend map half', op='attend', mode='train', dtype='f16', B=2, L=200, S=32400, H=8, G=1, D=16, mask='none'),
        # 60 ray queries to the 112 pixels of their image column, 1200 columns
        dict(name='attend rays', op='attend', mode='train', dtype='f16', B=1200, L=60, S=112, H=8, G=1, D=16, mask='none'),
        # the queries of a RoI block, each to the queries of its own camera; queries that no camera sees have an empty row
        dict(name='attend views', op='attend', mode='train', dtype='f32', B=2, L=200, S=200, H=8, G=1, D=16, mask='groups'),
        # one query to a short memory: latency
        dict(name='attend one short', op='attend', mode='serve', dtype='f16', B=1, L=1, S=37, H=8, G=1, D=16, mask='none'),
        # one query per sample to long memories of different lengths, four heads to a key head
        dict(name='attend one long', op='attend', mode='serve', dtype='bf16', B=16, L=1, S=32768, H=32, G=4, D=128, mask='lengths'),
        # a padded batch with shared key heads
        dict(name='attend shared', op='attend', mode='train', dtype='bf16', B=4, L=511, S=4100, H=16, G=4, D=64, mask='lengths'),
        # wide heads, long on both sides
        dict(name='attend wide', op='attend', mode='train', dtype='bf16', B=1, L=2048, S=8192, H=16, G=1, D=128, mask='none'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        C = rng.choice([_log(rng, 1, 8192), 8 * _log(rng, 1, 1024)])
        rows = _log(rng, 1, max(2, min(200000, 33554432 // C)))
        x = rng.choice(['f32', 'f16', 'bf16'])
        res = rng.choice([None, x, 'f16' if x == 'f32' else x])
        return dict(op='norm', mode=rng.choice(['train', 'train', 'serve']), rows=rows, C=C, x=x, res=res,
                    w=rng.choice([x, 'f32']), y=x, total=res is not None and rng.random() < 0.5)
    D, G = rng.choice([16, 16, 32, 64, 128, 24, 72]), rng.choice([1, 1, 2, 4])
    H = G * rng.choice([1, 2, 4, 8])
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    if rng.random() < 0.3:                                   # a few queries to a long memory
        L, S = rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 65536)
        B = _log(rng, 1, max(1, min(64, 16 * 32768 * 8 * 128 // (S * H // G * D))))
        return dict(op='attend', mode='serve', dtype=dtype, B=B, L=L, S=S, H=H, G=G, D=D, mask=rng.choice(['none', 'lengths', 'keys']))
    L, S = _log(rng, 1, 2048), _log(rng, 1, 32768)
    most = 2048 * 8192 * 16 // (4 if dtype == 'f32' else 1)
    B = _log(rng, 1, max(1, min(1000, most // (L * S * H))))
    while B * L * S * H > most:
        L = max(1, L // 2)
    mask = rng.choice(['none', 'lengths', 'keys'] + (['groups'] if B * L * S < 1 << 26 else []))
    return dict(op='attend', mode='train', dtype=dtype, B=B, L=L, S=S, H=H, G=G, D=D, mask=mask)


def _lengths(case):
    """The valid keys of each sample: all of the first's, none of the last's in a batch of four or more."""
    B, S = case['B'], case['S']
    if case['mask'] != 'lengths':
        return [S] * B
    return [S * (B - 1 - b) // (B - 1) for b in range(B)] if B >= 4 else [S * (B - b) // B for b in range(B)]


def _randn(g, *shape):
    return torch.randn(*shape, device='cuda', generator=g)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    st = dict(case)
    if case['op'] == 'norm':
        n, C = case['rows'], case['C']
        st['x'] = (_randn(g, n, C) + 0.5 * _randn(g, n, 1)).to(_T[case['x']])
        st['res'] = None if case['res'] is None else _randn(g, n, C).to(_T[case['res']])
        st['weight'] = (1 + 0.2 * _randn(g, C)).to(_T[case['w']])
        st['bias'] = (0.1 * _randn(g, C)).to(_T[case['w']])
        if case['mode'] == 'train':
            st['gy'] = _randn(g, n, C).to(_T[case['y']])
            st['gs'] = _randn(g, n, C).to(_T[case['y']]) if case['total'] else None
        return st
    B, L, S, H, D = (case[k] for k in 'BLSHD')
    E, Ek, t = H * D, H // case['G'] * D, _T[case['dtype']]
    st['q'] = (1.5 * _randn(g, B, L, E)).to(t)
    kv = torch.empty(B, S, 2 * Ek, device='cuda', dtype=t)       # keys and values side by side, as one projection writes them
    kv.normal_(generator=g)
    st['k'], st['v'] = kv[..., :Ek], kv[..., Ek:]
    st['lengths'] = torch.tensor(_lengths(case), dtype=torch.int32, device='cuda') if case['mask'] == 'lengths' else None
    st['key_mask'] = (torch.rand(B, S, device='cuda', generator=g) < 0.7) if case['mask'] == 'keys' else None
    st['allowed'] = None
    if case['mask'] == 'groups':                                 # seven groups; the members of group 0 have an empty row
        gq, gk = (torch.randint(0, 7, (B, n), device='cuda', generator=g) for n in (L, S))
        st['allowed'] = ((gq[:, :, None] == gk[:, None, :]) & (gq[:, :, None] > 0)).contiguous()
    if case['mode'] == 'train':
        st['go'] = _randn(g, B, L, E).to(t)
    return st


def _norm_plain(st):
    x, w = st['x'].float(), st['weight'].float()
    s, total = x, None
    if st['res'] is not None:
        s = x + st['res'].float()
        if st['total']:
            total = s.to(st['x'].dtype)
            s = total.float()
    mean = s.mean(-1, keepdim=True)
    c = s - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    hat = c * rstd
    out = {'y': (hat * w + st['bias'].float()).to(_T[st['y']])}
    if total is not None:
        out['sum'] = total
    if st['mode'] == 'train':
        gy = st['gy'].float()
        gh = gy * w
        gx = rstd * (gh - gh.mean(-1, keepdim=True) - hat * (gh * hat).mean(-1, keepdim=True))
        if st['gs'] is not None:
            gx = gx + st['gs'].float()
        out['gx'] = gx.to(st['x'].dtype)
        if st['res'] is not None:
            out['gres'] = gx.to(st['res'].dtype)
        out['gw'] = (gy * hat).sum(0).to(st['weight'].dtype)
        out['gb'] = gy.sum(0).to(st['bias'].dtype)
    return out


def _norm_own(st):
    from deepinteraction_amd import ops
    kw = dict(res=st['res'], eps=1e-5, with_sum=st['total'], out_dtype=_T[st['y']])
    if st['mode'] == 'serve':
        got = ops.layernorm(st['x'], st['weight'], st['bias'], **kw)
        return {'y': got[0], 'sum': got[1]} if st['total'] else {'y': got}
    y, total, mean, rstd = ops.layernorm_train_fwd(st['x'], st['weight'], st['bias'], **kw)
    out = {'y': y}
    if total is not None:
        out['sum'] = total
        gx, _, gw, gb = ops.layernorm_train_bwd(st['gy'], total, st['weight'], mean, rstd, grad_sum=st['gs'], grad_dtype=st['x'].dtype)
        gres = gx if st['res'].dtype == gx.dtype else gx.to(st['res'].dtype)
    else:
        gx, gres, gw, gb = ops.layernorm_train_bwd(st['gy'], st['x'], st['weight'], mean, rstd, res=st['res'])
    out['gx'] = gx
    if st['res'] is not None:
        out['gres'] = gres
    out['gw'], out['gb'] = gw, gb
    return out


def _keep(st, L, S):
    """(B, L or 1, S) truth values: the keys that take part, None for all."""
    keep = None
    if st['lengths'] is not None:
        keep = (torch.arange(S, device='cuda')[None] < st['lengths'][:, None])[:, None]
    if st['key_mask'] is not None:
        keep = st['key_mask'][:, None]
    if st['allowed'] is not None:
        keep = st['allowed']
    return keep


def _attend_plain(st):
    B, L, S, H, G, D = (st[k] for k in 'BLSHGD')
    K = H // G
    q = st['q'].float().view(B, L, K, G, D).permute(0, 2, 3, 1, 4).reshape(B, K, G * L, D)
    k = st['k'].float().reshape(B, S, K, D).transpose(1, 2).contiguous()
    v = st['v'].float().reshape(B, S, K, D).transpose(1, 2).contiguous()
    scale = D ** -0.5
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, K, G, L, S)
    s = s * scale
    keep = _keep(st, L, S)
    if keep is not None:
        s = s.masked_fill(~keep[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    den = e.sum(-1, keepdim=True)
    p = (e / torch.where(den == 0, torch.ones_like(den), den)).view(B, K, G * L, S)
    o = torch.matmul(p, v)
    rows = lambda t: t.view(B, K, G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H * D)
    cols = lambda t: t.transpose(1, 2).reshape(B, S, K * D)
    out = {'o': rows(o).to(st['q'].dtype)}
    if st['mode'] == 'train':
        go = st['go'].float().view(B, L, K, G, D).permute(0, 2, 3, 1, 4).reshape(B, K, G * L, D)
        gp = torch.matmul(go, v.transpose(-1, -2).contiguous())
        gs = p * (gp - (p * gp).sum(-1, keepdim=True)) * scale
        out['gq'] = rows(torch.matmul(gs, k)).to(st['q'].dtype)
        out['gk'] = cols(torch.matmul(gs.transpose(-1, -2).contiguous(), q)).to(st['q'].dtype)
        out['gv'] = cols(torch.matmul(p.transpose(-1, -2).contiguous(), go)).to(st['q'].dtype)
    return out


def _attend_own(st):
    from deepinteraction_amd import ops
    kw = dict(key_lengths=st['lengths'], key_mask=st['key_mask'], allowed=st['allowed'])
    if st['mode'] == 'serve':
        return {'o': ops.cross_attention(st['q'], st['k'], st['v'], st['H'], **kw)}
    o, lse = ops.cross_attention_train_fwd(st['q'], st['k'], st['v'], st['H'], **kw)
    gq, gk, gv = ops.cross_attention_train_bwd(st['q'], st['k'], st['v'], o, st['go'], lse, st['H'], **kw)
    return {'o': o, 'gq': gq, 'gk': gk, 'gv': gv}


def run(state):
    if state['op'] == 'norm':
        return _norm_own(state) if own else _norm_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def work(case):
    if case['op'] == 'norm':
        n = case['rows'] * case['C']
        x, r, y = _BYTES[case['x']], 0 if case['res'] is None else _BYTES[case['res']], _BYTES[case['y']]
        w = 2 * case['C'] * _BYTES[case['w']]
        b, f = n * (x + r + y + (x if case['total'] else 0)) + w, 8 * n
        if case['mode'] == 'train':
            b, f = b + n * (y + x + r + (y if case['total'] else 0)) + w, f + 14 * n
        return {'bytes': b, 'flops': f}
    B, L, S, H, D = (case[k] for k in 'BLSHD')
    e, kept = _BYTES[case['dtype']], sum(_lengths(case))
    Ek = H // case['G'] * D
    b, f = e * (2 * B * L * H * D + 2 * kept * Ek), 4 * D * H * L * kept
    if case['mask'] in ('keys', 'groups'):
        b += B * S * (L if case['mask'] == 'groups' else 1)
    if case['mode'] == 'train':
        b, f = b + e * (2 * B * L * H * D + 2 * B * S * Ek), f + 10 * D * H * L * kept
    return {'bytes': b, 'flops': f}


def exact(case, seed):
    st = prepare(case, seed)
    wide = lambda t: None if t is None else t.double()
    if case['op'] == 'norm':
        a, r, w = wide(st['x']), wide(st['res']), wide(st['weight'])
        s = a if r is None else a + r
        if case['total']:                                        # the sum is carried in its own type, and that is what is normalised
            s = (st['x'].float() + st['res'].float()).to(st['x'].dtype).double()
        var, mu = torch.var_mean(s, -1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        z = (s - mu) / sd
        out = {'y': z * w + wide(st['bias'])}
        if case['total']:
            out['sum'] = a + r
        if case['mode'] == 'train':
            gy = wide(st['gy'])
            t = gy * w
            C = case['C']
            gx = (C * t - t.sum(-1, keepdim=True) - z * (t * z).sum(-1, keepdim=True)) / (C * sd)
            if st['gs'] is not None:
                gx = gx + wide(st['gs'])
            out['gx'] = gx
            if r is not None:
                out['gres'] = gx
            out['gw'], out['gb'] = (gy * z).sum(0), gy.sum(0)
        return out
    B, L, S, H, G, D = (case[k] for k in 'BLSHGD')
    keep = _keep(st, L, S)
    train = case['mode'] == 'train'
    o = torch.zeros(B, L, H, D, dtype=torch.float64, device='cuda')
    gq = torch.zeros_like(o) if train else None
    gk, gv = (torch.zeros(B, S, H // G, D, dtype=torch.float64, device='cuda') if train else None for _ in range(2))
    part = max(1, 1 << 28 >> max(0, (L * S).bit_length()))       # samples at a time
    for h in range(H):
        for b0 in range(0, B, part):
            b = slice(b0, min(B, b0 + part))
            head = lambda t, j: wide(t[b, :, j * D:(j + 1) * D]).contiguous()
            q, k, v = head(st['q'], h), head(st['k'], h // G), head(st['v'], h // G)
            s = torch.bmm(q, k.mT.contiguous()) / math.sqrt(D)
            if keep is not None:
                s = torch.where(keep[b], s, torch.full_like(s, -math.inf))
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
            o[b, :, h] = torch.bmm(p, v)
            if train:
                go = head(st['go'], h)
                d = (go * o[b, :, h]).sum(-1, keepdim=True)
                ds = p * (torch.bmm(go, v.mT.contiguous()) - d) / math.sqrt(D)
                gq[b, :, h] = torch.bmm(ds, k)
                gk[b, :, h // G] += torch.bmm(ds.mT.contiguous(), q)
                gv[b, :, h // G] += torch.bmm(p.mT.contiguous(), go)
    out = {'o': o.reshape(B, L, H * D)}
    if train:
        out |= {'gq': gq.reshape(B, L, -1), 'gk': gk.reshape(B, S, -1), 'gv': gv.reshape(B, S, -1)}
    return out
