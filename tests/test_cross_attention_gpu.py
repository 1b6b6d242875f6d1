"""csrc/attention*.h / .hip: attention to the states of another sequence, forward, backward and single queries, against float64.

Tolerances (elementwise, from the float64 quantities).  u = 2^-24, e = half a step of the type (0 for float32), natural-log units:
  score        es = (D + 8) u scale sum_d |q||k| + 4 u (|s| + max|s|)       D products summed in float32, the exponent's fma and exp2
  probability  rel. ep = 2 max_j es + 64 u, plus e for its rounding to 16 bits (float16 below 2^-14 of its scale: 2^-25 absolute);
               exp2 gives 0 below the smallest normal float32: 2^-126 absolute
  o            sum_j p |v| (ep + e) + e |o|         delta = go . o  takes o as stored: sum_d |go| tol(o)
  dp           (D + 8) u sum_d |go||v|
  ds           |ds| (ep + e) + p (tol(dp) + tol(delta) + 4 u (|dp| + |delta|))   (+ 2^-25 for float16)
  gq, gk, gv   the sums of those, + 64 u of the sums' magnitudes for the float32 accumulation, + e of the result
The accumulation is blocked (32 keys or rows per product, products added one after another): n / 32 + 32 roundings at the most, of
sums that grow; 64 u covers up to 1024 keys or rows, and (n / 16) u is taken above that."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from deepinteraction_amd import ops

U, FLUSH = 2.0 ** -24, 2.0 ** -126
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def eps_half(t):
    return 0.0 if t == F32 else torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == F16 else 0.0


def make(B, L, S, H, Hk, D, t, seed=0, sharp=1.5):
    g = torch.Generator(device='cuda').manual_seed(seed + 1000 * L + S + 7 * D)
    r = lambda *s: torch.randn(*s, device='cuda', generator=g)
    q = (sharp * r(B, L, H * D)).to(t)
    kv = r(B, S, 2 * Hk * D).to(t)
    return q, kv[..., :Hk * D], kv[..., Hk * D:], r(B, L, H * D).to(t)


def split(x, H):
    B, N, E = x.shape
    return x.double().view(B, N, H, E // H).transpose(1, 2).contiguous()


def oracle(q, k, v, go, H, keep, scale, kept=None):
    """(values, tolerances) of o, lse, gq, gk, gv; kept: (B, H, L, S) dropout factors."""
    t, e = q.dtype, eps_half(q.dtype)
    B, L, E = q.shape
    D, Hk = E // H, k.shape[-1] * H // E
    G, S = H // Hk, k.shape[1]
    Q, K, V, GO = split(q, H), split(k.contiguous(), Hk).repeat_interleave(G, 1), split(v.contiguous(), Hk).repeat_interleave(G, 1), split(go, H)
    mm = lambda a, b: torch.matmul(a, b.contiguous())
    s = scale * mm(Q, K.mT)
    sa = scale * mm(Q.abs(), K.abs().mT)
    if keep is not None:
        s = s.masked_fill(~keep.unsqueeze(1).expand(B, H, L, S), -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True) if S else torch.full((B, H, L, 1), -math.inf, device=q.device, dtype=torch.float64)
    p = torch.exp(s - torch.where(lse.isinf(), torch.zeros_like(lse), lse))
    fin = torch.where(s.isinf(), torch.zeros_like(s), s).abs()
    es = (D + 8) * U * sa + 4 * U * (fin + (fin.amax(-1, keepdim=True) if S else 0))
    ep = (2 * es.amax(-1, keepdim=True) if S else 0) + 64 * U
    n = lambda x: max(64, x / 16) * U
    d = torch.ones_like(p) if kept is None else kept
    pd = p * d
    o = mm(pd, V)
    # the running maximum's slack: exponentials are rounded at up to 2^8 and at least 1 times their final size, never below
    low = tiny(t) * 256 * mm(d.expand_as(p) * (p > 0), V.abs()) / torch.where(lse.isinf(), 1, torch.exp(lse - (s.amax(-1, keepdim=True) if S else 0)).clamp_min(1))
    o_tol = mm(pd, V.abs()) * (ep + e + n(S)) + (e + U) * o.abs() + low + FLUSH * mm(d.expand_as(p), V.abs())
    lse2 = lse * math.log2(math.e)
    delta = (GO * o).sum(-1, keepdim=True)
    delta_tol = (GO.abs() * o_tol).sum(-1, keepdim=True) + (D + 8) * U * (GO.abs() * o.abs()).sum(-1, keepdim=True)
    dp, dpa = mm(GO, V.mT) * d, mm(GO.abs(), V.abs().mT) * d
    ds = p * (dp - delta)
    ds_tol = ds.abs() * (ep + e) + p * ((D + 8) * U * dpa + delta_tol + 4 * U * (dp.abs() + delta.abs())) + FLUSH * (dp.abs() + delta.abs() + 1) + tiny(t)
    gq, gq_tol = scale * mm(ds, K), scale * (mm(ds_tol, K.abs()) + n(S) * mm(ds.abs(), K.abs()))
    rows = G * L
    gk, gk_tol = scale * mm(ds.mT, Q), scale * (mm(ds_tol.mT, Q.abs()) + n(rows) * mm(ds.abs().mT, Q.abs()))
    # float16 probabilities are scaled by 2^14 before their rounding: 2^-39 absolute
    gv, gv_tol = mm(pd.mT, GO), mm((pd * (ep + e) + tiny(t) * 2.0 ** -14 * (p > 0) + FLUSH * d).mT, GO.abs()) + n(rows) * mm(pd.mT, GO.abs())
    rowsof = lambda x: x.transpose(1, 2).reshape(B, L, E)
    fold = lambda x: x.view(B, Hk, G, S, D).sum(2).transpose(1, 2).reshape(B, S, Hk * D)
    out = dict(o=(rowsof(o), rowsof(o_tol)), lse=(lse2[..., 0], (ep[..., 0] if S else 64 * U) * 2 + 4 * U * lse2[..., 0].abs()),
               gq=(rowsof(gq), rowsof(gq_tol)), gk=(fold(gk), fold(gk_tol)), gv=(fold(gv), fold(gv_tol)))
    return out, (e + 2 * U)


def close(name, got, want, tol, e):
    assert got.shape == want.shape, name
    fin = want.isfinite()
    assert torch.equal(got.isfinite(), fin) and torch.equal(got[~fin].double(), want[~fin]), name
    # below its smallest normal number, 2^-14, float16's step is 2^-24 for every value: half of it is 2^-25, not e |value|
    off = (got.double() - want).abs()[fin] - (tol if tol.dim() == 0 else tol[fin]) - e * want.abs()[fin] - tiny(got.dtype)
    assert not (off > 0).any(), (name, int((off > 0).sum()), float(off.max()), float(want[fin].abs().max()))


def check(q, k, v, go, H, keep=None, scale=None, kept=None, **kw):
    scale = (q.shape[-1] // H) ** -0.5 if scale is None else scale
    o, lse = ops.cross_attention_train_fwd(q, k, v, H, scale, **kw)
    gq, gk, gv = ops.cross_attention_train_bwd(q, k, v, o, go, lse, H, scale, **kw)
    want, e = oracle(q, k, v, go, H, keep, scale, kept)
    for name, got in (('o', o), ('lse', lse), ('gq', gq), ('gk', gk), ('gv', gv)):
        close(name, got, *[w if torch.is_tensor(w) else torch.tensor(w) for w in want[name]], e)
    if 'dropout_p' not in kw:
        assert torch.equal(ops.cross_attention(q, k, v, H, scale, **kw), o)
    return o, lse, gq, gk, gv


SHAPES = [(1, 1, 1, 1, 1, 16), (2, 1, 37, 8, 8, 16), (1, 1, 3000, 4, 4, 16), (2, 5, 63, 4, 2, 16), (1, 16, 64, 2, 2, 16), (3, 17, 65, 2, 1, 16),
          (1, 60, 112, 8, 8, 16), (2, 200, 200, 2, 2, 16), (1, 200, 3240, 8, 8, 16), (2, 70, 129, 4, 1, 24), (1, 33, 1, 2, 2, 32),
          (1, 300, 500, 3, 3, 32), (2, 1, 1025, 8, 2, 64), (1, 130, 257, 4, 2, 64), (1, 65, 700, 2, 2, 72), (2, 3, 31, 8, 1, 128),
          (1, 1, 2049, 4, 1, 128), (1, 150, 330, 2, 1, 128), (2, 64, 64, 1, 1, 128), (1, 1000, 40, 2, 2, 8), (1, 2048, 1, 1, 1, 64)]


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_shapes(shape, t):
    B, L, S, H, Hk, D = shape
    check(*make(B, L, S, H, Hk, D, t), H)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('D,H,Hk,L,S', [(16, 4, 4, 40, 150), (16, 4, 2, 1, 900), (64, 2, 1, 90, 200), (128, 2, 2, 20, 333)])
def test_masks(t, D, H, Hk, L, S):
    """Lengths 0, 1, in a tile's middle, all and beyond; a key mask; a (query, key) mask; all three - with empty rows in each."""
    B = 5
    q, k, v, go = make(B, L, S, H, Hk, D, t)
    g = torch.Generator(device='cuda').manual_seed(L)
    lengths = torch.tensor([0, 1, S // 2 + 3, S, S + 9], dtype=torch.int32, device='cuda')
    by_len = (torch.arange(S, device='cuda')[None] < lengths[:, None])[:, None].expand(B, L, S)
    key_mask = torch.rand(B, S, device='cuda', generator=g) < 0.5
    key_mask[1] = False
    allowed = torch.rand(B, L, S, device='cuda', generator=g) < 0.3
    allowed[:, L // 2] = False
    by_key = key_mask[:, None].expand(B, L, S)
    o = check(q, k, v, go, H, by_len, key_lengths=lengths)[0]
    assert not o[0].any()
    check(q, k, v, go, H, by_key, key_mask=key_mask)
    check(q, k, v, go, H, allowed, allowed=allowed)
    check(q, k, v, go, H, by_len & by_key & allowed, key_lengths=lengths.long(), key_mask=key_mask, allowed=allowed)
    check(q, k, v, go, H, allowed[:, :1].expand(B, L, S), allowed=allowed[:, :1].expand(B, L, S))
    check(q, k, v, go, H, allowed[:1].expand(B, L, S), allowed=allowed[:1].expand(B, L, S))


@pytest.mark.parametrize('t', [F32, F16], ids=str)
@pytest.mark.parametrize('B,L,S,H,Hk,D', [(5, 200, 1500, 8, 8, 64), (16, 1, 1400, 8, 4, 64), (64, 40, 130, 4, 2, 64), (65, 40, 130, 4, 2, 64), (9, 90, 700, 8, 8, 16),
                                          (3, 600, 900, 4, 4, 128), (1, 300, 5000, 8, 8, 32), (6, 70, 400, 16, 16, 128), (64, 1, 600, 8, 8, 16)])
def test_batches_of_different_lengths(B, L, S, H, Hk, D, t):
    """More workgroups than compute units: those with keys are put first; no key at all, one, a range's worth, all of them."""
    q, k, v, go = make(B, L, S, H, Hk, D, t)
    for kind in range(3):
        n = [[S, 0, 1, S - 1, 64, 65, S // 2, 128, 17][(3 * b + kind) % 9] if kind < 2 else 0 for b in range(B)]
        n = torch.tensor(n, dtype=torch.int32, device='cuda')
        keep = (torch.arange(S, device='cuda')[None, None] < n[:, None, None]).expand(B, L, S)
        check(q, k, v, go, H, keep, key_lengths=n)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('L,S,D', [(1, 300, 16), (70, 300, 16), (1, 300, 128), (40, 130, 64)])
def test_excluded_keys_may_hold_anything(t, L, S, D):
    B, H = 3, 2
    q, k, v, go = make(B, L, S, H, H, D, t)
    k, v = k.clone(), v.clone()
    lengths = torch.tensor([S, S // 3, 0], dtype=torch.int32, device='cuda')
    mask = torch.rand(B, S, device='cuda') < 0.7
    dead = ~(mask & (torch.arange(S, device='cuda')[None] < lengths[:, None]))
    clean = check(q, k, v, go, H, (~dead)[:, None].expand(B, L, S), key_lengths=lengths, key_mask=mask)
    k[dead], v[dead] = float('nan'), float('inf')
    v[:, ::2][dead[:, ::2]] = torch.finfo(t).min
    o, lse = ops.cross_attention_train_fwd(q, k, v, H, key_lengths=lengths, key_mask=mask)
    got = (o, lse) + ops.cross_attention_train_bwd(q, k, v, o, go, lse, H, key_lengths=lengths, key_mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert not got[3][dead].any() and not got[4][dead].any()


@pytest.mark.parametrize('D', [16, 24, 64, 128])
@pytest.mark.parametrize('S', [1, 2, 3, 4, 5, 13, 15, 16, 17, 31, 64, 65, 131, 258, 519])
def test_mask_rows_that_start_and_end_anywhere(S, D):
    """(query, key) masks of every width, at odd addresses, of bytes other than 0 and 1, with rows apart or shared."""
    B, L, H, Hk = 2, 21, 4, 2
    for t in (F32, F16):
        q, k, v, go = make(B, L, S, H, Hk, D, t)
        for lead, rs in ((0, S), (1, S), (3, S + 7)):
            store = (torch.rand(lead + B * L * rs, device='cuda') < 0.5).to(torch.uint8) * 6
            allowed = store[lead:].as_strided((B, L, S), (L * rs, rs, 1), lead)
            check(q, k, v, go, H, allowed != 0, allowed=allowed)
        lengths = torch.tensor([S, S // 2], dtype=torch.int32, device='cuda')
        keep = (allowed != 0) & (torch.arange(S, device='cuda') < lengths[:, None, None])
        check(q, k, v, go, H, keep, allowed=allowed, key_lengths=lengths)
        shared = allowed[:1, :1].expand(B, L, S)
        check(q, k, v, go, H, shared != 0, allowed=shared)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('D', range(8, 129, 8))
def test_every_head_dim(D, t):
    """Single queries, few rows and row blocks, ragged lengths and masks, split ranges, dropout."""
    for B, L, S, H, Hk in ((3, 1, 333, 4, 2), (2, 19, 201, 2, 1), (1, 150, 700, 2, 2)):
        q, k, v, go = make(B, L, S, H, Hk, D, t)
        check(q, k, v, go, H)
        lengths = torch.tensor([S, 0, S - 70][:B], dtype=torch.int32, device='cuda')
        mask, allowed = torch.rand(B, S, device='cuda') < 0.8, torch.rand(B, L, S, device='cuda') < 0.5
        keep = (torch.arange(S, device='cuda') < lengths[:, None]) & mask
        check(q, k, v, go, H, keep[:, None].expand(B, L, S), key_lengths=lengths, key_mask=mask)
        check(q, k, v, go, H, keep[:, None] & allowed, key_lengths=lengths, key_mask=mask, allowed=allowed)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('L,S,D', [(1, 300, 16), (70, 300, 16), (200, 40, 32), (40, 130, 64), (150, 200, 128), (5, 700, 128)])
def test_queries_without_keys_may_hold_anything(t, L, S, D):
    """A padded query: nothing allowed, NaN in its projection and its incoming gradient.  It gives zeros and reaches no other gradient."""
    B, H = 2, 2
    q, k, v, go = make(B, L, S, H, 1, D, t)
    allowed = torch.rand(B, L, S, device='cuda') < 0.6
    pad = torch.rand(B, L, device='cuda') < 0.4
    pad[0, 0], pad[1, 0] = True, False
    allowed &= ~pad[..., None]
    allowed[..., 0] |= ~pad
    q, go = q.clone(), go.clone()
    go[pad] = 0
    clean = check(q, k, v, go, H, allowed, allowed=allowed)
    q[pad], go[pad] = float('nan'), float('nan')
    go[0, 0] = float('inf')
    o, lse = ops.cross_attention_train_fwd(q, k, v, H, allowed=allowed)
    got = (o, lse) + ops.cross_attention_train_bwd(q, k, v, o, go, lse, H, allowed=allowed)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert not got[0][pad].any() and not got[2][pad].any()


@pytest.mark.parametrize('D', [16, 64])
def test_gradients_that_would_overlap_are_refused(D):
    q, k, v, go = make(2, 5, 9, 2, 2, D, F16)
    o, lse = ops.cross_attention_train_fwd(q, k, v, 2)
    for bad in (k.new_empty(2, 1, 2 * D).expand(2, 9, 2 * D), k.new_empty(1, 9, 2 * D).expand(2, 9, 2 * D),
                k.new_empty(64 * D).as_strided((2, 9, 2 * D), (24 * D, D, 1))):
        for pair in ((bad, v), (v, bad)):
            with pytest.raises((ValueError, ops._lib.HipLibraryError)):
                ops.cross_attention_train_bwd(q, k, v, o, go, lse, 2, grads_kv=pair)


@pytest.mark.parametrize('t', TYPES, ids=str)
@pytest.mark.parametrize('D', [16, 24, 64, 80, 128])
def test_a_single_key_has_no_score_gradient(D, t):
    """Exact zeros in gq and gk where every query has one key: S = 1, masks that leave one, another one for every query."""
    H, Hk = 4, 2
    for B, L, S in ((3, 70, 1), (2, 1, 1), (2, 33, 2), (1, 150, 16)):
        q, k, v, go = make(B, L, S, H, Hk, D, t)
        pick = torch.randint(0, S, (B, L), device='cuda')
        allowed = torch.zeros(B, L, S, dtype=torch.bool, device='cuda').scatter_(2, pick[..., None], True)
        allowed[:, -1] &= L == 1                                       # and a query without any
        mask = torch.zeros(B, S, dtype=torch.bool, device='cuda').scatter_(1, pick[:, :1], True)
        one = torch.ones(B, dtype=torch.int32, device='cuda')
        for kw, keep in ((dict(key_lengths=one), torch.arange(S, device='cuda')[None, None] < 1), (dict(key_mask=mask), mask[:, None]),
                         (dict(allowed=allowed), allowed)) + (((dict(), None),) if S == 1 else ()):
            _, _, gq, gk, _ = check(q, k, v, go, H, None if keep is None else keep.expand(B, L, S), **kw)
            assert not gq.any() and not gk.any()


def test_nothing_to_attend_to():
    for t in TYPES:
        for B, L, S in ((2, 5, 0), (2, 0, 7), (0, 3, 4), (2, 100, 0)):
            q, k, v, go = make(B, L, S, 4, 2, 16, t)
            o, lse = ops.cross_attention_train_fwd(q, k, v, 4)
            gq, gk, gv = ops.cross_attention_train_bwd(q, k, v, o, go, lse, 4)
            assert o.shape == q.shape and gk.shape == k.shape
            assert not any(x.any() for x in (o, gq, gk, gv)) and (lse == -math.inf).all()


@pytest.mark.parametrize('t', TYPES, ids=str)
def test_large_scores(t):
    """Scores of some hundreds, as the decoder's positional terms make them; the maximum moves late and by much."""
    q, k, v, go = make(2, 50, 400, 2, 2, 16, t, sharp=40.0)
    k = k.clone()
    k[:, 390:] *= 4
    check(q, k, v, go, 2)
    check(q, -k.abs(), v, go, 2, scale=3.0)
    check(torch.zeros_like(q), k, v, go, 2)


@pytest.mark.parametrize('t', TYPES, ids=str)
def test_layouts(t):
    """Packed q | k | v of one projection, rows that do not start on 16 bytes, a transposed sequence, one memory for all samples."""
    B, N, H, D = 2, 45, 4, 16
    E = H * D
    g = torch.Generator(device='cuda').manual_seed(3)
    qkv = torch.randn(B, N, 3 * E + 8, device='cuda', generator=g).to(t)
    go = torch.randn(B, N, E, device='cuda', generator=g).to(t)
    for lead in (0, 8, 3):
        q, k, v = (qkv[..., lead + j * E:lead + (j + 1) * E] for j in range(3))
        ref = ops.cross_attention_train_fwd(q.contiguous(), k.contiguous(), v.contiguous(), H)
        got = ops.cross_attention_train_fwd(q, k, v, H)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
        a = ops.cross_attention_train_bwd(q, k, v, got[0], go, got[1], H)
        b = ops.cross_attention_train_bwd(q.contiguous(), k.contiguous(), v.contiguous(), got[0], go, got[1], H)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    q, k, v = (qkv[..., j * E:(j + 1) * E] for j in range(3))
    qt, kt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    got = ops.cross_attention_train_fwd(qt, kt, v, H)
    assert torch.equal(got[0], ops.cross_attention(q, k, v, H))
    ke, ve = k[:1].expand(B, N, E), v[:1].expand(B, N, E)
    assert torch.equal(ops.cross_attention(q, ke, ve, H), ops.cross_attention(q, ke.contiguous(), ve.contiguous(), H))
    # packed gradients: two halves of one buffer, and nothing beside them
    o, lse = ops.cross_attention_train_fwd(q, k, v, H)
    want = ops.cross_attention_train_bwd(q, k, v, o, go, lse, H)
    buf = torch.full((B, N, 2 * E + 16), 7.0, device='cuda', dtype=t)
    got = ops.cross_attention_train_bwd(q, k, v, o, go, lse, H, grads_kv=(buf[..., :E], buf[..., E:2 * E]))
    assert torch.equal(buf[..., :E], want[1]) and torch.equal(buf[..., E:2 * E], want[2]) and (buf[..., 2 * E:] == 7).all()
    assert torch.equal(got[0], want[0])


def test_offsets_past_32_bits():
    """The last columns of a 40 000 x 65 536 matrix: 5.2 GB from the first key to the last."""
    wide = torch.empty(1, 40000, 65536, device='cuda', dtype=F16)
    k, v = wide[..., -64:-32], wide[..., -32:]
    k.normal_()
    v.normal_()
    q, go = torch.randn(1, 3, 32, device='cuda').half(), torch.randn(1, 3, 32, device='cuda').half()
    want = ops.cross_attention_train_fwd(q, k.contiguous(), v.contiguous(), 2)
    got = ops.cross_attention_train_fwd(q, k, v, 2)
    assert torch.equal(got[0], want[0])
    a = ops.cross_attention_train_bwd(q, k, v, got[0], go, got[1], 2)
    b = ops.cross_attention_train_bwd(q, k.contiguous(), v.contiguous(), got[0], go, got[1], 2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def kept_factors(B, H, L, S, p, seed, t):
    """The dropout factors (B, H, L, S) that the kernels use, read out: equal scores and one-hot values, 16 keys at a time."""
    D = 16
    q = torch.zeros(B, L, H * D, device='cuda', dtype=t)
    k = torch.zeros(B, S, H * D, device='cuda', dtype=t)
    out = []
    for s0 in range(0, S, D):
        v = torch.zeros(B, S, H, D, device='cuda', dtype=t)
        n = min(D, S - s0)
        v[:, s0:s0 + n] = torch.eye(D, device='cuda', dtype=t)[:n, None]
        o, _ = ops.cross_attention_train_fwd(q, k, v.view(B, S, H * D), H, dropout_p=p, seed=seed)
        out.append(o.view(B, L, H, D)[..., :n] * S)
    kept = torch.cat(out, -1).transpose(1, 2).double()
    scale = 1 / (1 - round(p * 65536) / 65536)
    on = kept > 0.5 * scale
    assert (kept[on] - scale).abs().max() <= 0.01 * scale and not kept[~on].any()
    return on.double() * scale


@pytest.mark.parametrize('p', [0.1, 0.5, 0.95])
def test_dropout(p):
    B, H, L, S = 2, 4, 90, 150
    kept = kept_factors(B, H, L, S, p, 77, F32)
    n, rate = kept.numel(), float((kept == 0).double().mean())
    assert abs(rate - p) <= 5 * math.sqrt(p * (1 - p) / n), rate
    for dim in (0, 1, 2, 3):                                         # neighbours in any direction are independent
        a, b = (kept == 0).double().narrow(dim, 0, kept.shape[dim] - 1), (kept == 0).double().narrow(dim, 1, kept.shape[dim] - 1)
        assert abs(float(((a - p) * (b - p)).mean())) <= 5 * p * (1 - p) / math.sqrt(a.numel()), dim
    assert torch.equal(kept, kept_factors(B, H, L, S, p, 77, F16)) and not torch.equal(kept, kept_factors(B, H, L, S, p, 78, F32))
    for t in TYPES:
        for D in (16, 64):
            check(*make(B, L, S, H, H, D, t), H, kept=kept, dropout_p=p, seed=77)
    assert torch.equal(kept[:, :, :1], kept_factors(B, H, L, S, p, 77, F32)[:, :, :1])


def test_dropout_of_shared_heads_and_the_device_word():
    B, H, Hk, L, S, D = 1, 4, 2, 5, 70, 32
    q, k, v, go = make(B, L, S, H, Hk, D, F32)
    kept = kept_factors(B, H, L, S, 0.25, 5, F32)
    check(q, k, v, go, H, kept=kept, dropout_p=0.25, seed=5)
    word = torch.full((1,), 3, dtype=torch.int64, device='cuda')
    base = ops.cross_attention_train_fwd(q, k, v, H, dropout_p=0.25, seed=8)[0]
    ops.set_i2p_seed_tensor(word)
    try:
        assert torch.equal(ops.cross_attention_train_fwd(q, k, v, H, dropout_p=0.25, seed=5)[0], base)
    finally:
        ops.set_i2p_seed_tensor(None)


@pytest.mark.parametrize('mask', [False, True])
def test_against_differences(mask):
    """Gradients against central differences of the float64 formula: their own error is h^2 and 1e-16 / h, below 1e-8 of the terms;
    the kernel's is bounded by its tolerances, which 1e-5 of the sum of magnitudes covers at these sizes (D + S + 64 < 300 u ~ 2e-5)."""
    B, L, S, H, Hk, D = 2, 6, 20, 4, 2, 16
    q, k, v, go = make(B, L, S, H, Hk, D, F32)
    keep = (torch.rand(B, L, S, device='cuda') < 0.6) if mask else None
    if mask:
        keep[0, 2] = False
    o, lse = ops.cross_attention_train_fwd(q, k, v, H, allowed=keep)
    grads = ops.cross_attention_train_bwd(q, k, v, o, go, lse, H, allowed=keep)

    def loss(q_, k_, v_):
        Q, K, V = split(q_, H), split(k_, Hk).repeat_interleave(H // Hk, 1), split(v_, Hk).repeat_interleave(H // Hk, 1)
        s = torch.matmul(Q, K.mT.contiguous()) * D ** -0.5
        if keep is not None:
            s = s.masked_fill(~keep[:, None], -math.inf)
        return (torch.softmax(s, -1).nan_to_num() @ V * split(go, H)).sum()

    wide, h = [x.double() for x in (q, k, v)], 1e-5
    for i in range(3):
        d = torch.randn_like(wide[i])
        lo, hi = ([x + sgn * h * d if j == i else x for j, x in enumerate(wide)] for sgn in (-1, 1))
        diff, got = float(loss(*hi) - loss(*lo)) / (2 * h), float((grads[i].double() * d).sum())
        assert abs(got - diff) <= 2e-5 * float((grads[i].double() * d).abs().sum()) + 1e-6, i


def test_same_bits_other_stream_and_captured():
    t = F16
    q, k, v, go = make(2, 200, 3000, 8, 8, 16, t)

    def step():
        o, lse = ops.cross_attention_train_fwd(q, k, v, 8)
        return (o, lse) + ops.cross_attention_train_bwd(q, k, v, o, go, lse, 8)
    want = [x.clone() for x in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for n in range(3):
        q.copy_(torch.randn_like(q))
        want = [x.clone() for x in step()]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_refusals():
    q, k, v, go = make(2, 5, 9, 4, 2, 16, F32)
    o, lse = ops.cross_attention_train_fwd(q, k, v, 4)
    n = torch.tensor([9, 9], device='cuda', dtype=torch.int32)
    for bad in (lambda: ops.cross_attention(q, k, v, 3), lambda: ops.cross_attention(q, k, v[:, :8], 4), lambda: ops.cross_attention(q[:1], k, v, 4),
                lambda: ops.cross_attention(q, k[..., :24], v[..., :24], 4), lambda: ops.cross_attention(q, k, v, 64),
                lambda: ops.cross_attention(q, k, v, 4, scale=0.0), lambda: ops.cross_attention(q, k, v, 4, scale=-1.0),
                lambda: ops.cross_attention(q, k, v, 4, scale=float('inf')), lambda: ops.cross_attention(q, k, v, 4, key_lengths=n[:1]),
                lambda: ops.cross_attention(q, k, v, 4, key_lengths=n.float()), lambda: ops.cross_attention(q, k, v, 4, key_mask=n[:, None] > 0),
                lambda: ops.cross_attention(q, k, v, 4, allowed=torch.ones(2, 4, 9, device='cuda', dtype=torch.bool)),
                lambda: ops.cross_attention_train_fwd(q, k, v, 4, dropout_p=1.0), lambda: ops.cross_attention_train_fwd(q, k, v, 4, dropout_p=-0.1),
                lambda: ops.cross_attention_train_bwd(q, k, v, o[:1], go, lse, 4), lambda: ops.cross_attention_train_bwd(q, k, v, o, go[:, :4], lse, 4),
                lambda: ops.cross_attention_train_bwd(q, k, v, o, go, lse[:1], 4),
                lambda: ops.cross_attention_train_bwd(q, k, v, o, go, lse, 4, grads_kv=(k.new_empty(2, 9, 30), v))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.cross_attention(q, k.half(), v, 4), lambda: ops.cross_attention(q.double(), k.double(), v.double(), 4),
                lambda: ops.cross_attention(q, k, v, 4, key_mask=torch.ones(2, 9, device='cuda'))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(ops._lib.HipLibraryError):
        ops.cross_attention(q.cpu(), k, v, 4)


def test_queries_past_32_bits():
    """More than 2^31 queries in all: every sample is the same, and so is every sample's result, bit for bit."""
    B, L, D, S = 2 ** 21 + 3, 1024, 8, 2
    q, k, v, go = (x[:1].expand(B, -1, -1) for x in make(1, L, S, 1, 1, D, F16))
    o, lse = ops.cross_attention_train_fwd(q, k, v, 1)
    gq, gk, gv = ops.cross_attention_train_bwd(q, k, v, o, go, lse, 1)
    want, e = oracle(q[:1], k[:1], v[:1], go[:1], 1, None, D ** -0.5)
    for name, got in (('o', o), ('lse', lse), ('gq', gq), ('gk', gk), ('gv', gv)):
        close(name, got[:1], *want[name], e)
        for b in range(0, B, 1 << 17):
            part = got[b:b + (1 << 17)]
            assert torch.equal(part, got[:1].expand_as(part)), (name, b)


@pytest.mark.parametrize('far', [20.0, 25.3, 27.0])
@pytest.mark.parametrize('B,L,S,G,D', [(1, 1, 65537, 1, 16), (1, 40, 65537, 1, 16), (6144, 1, 65537, 1, 16), (1, 300, 65537, 512, 16), (1, 300, 65537, 256, 64),
                                       (1, 300, 65537, 256, 128)])
def test_many_keys_far_below_the_largest(B, L, S, G, D, far):
    """(Few queries: ranges of the keys with maxima of their own.  Many: one pass, the largest key first.)  One key and tens of thousands of 2^-far of its weight, float16: they count in the sum of the softmax, and have to in o.  A far
    probability is rounded once, to 11 bits or - below 2^-21 of the largest - to a step of 2^-31 of it: off by 2^-11 of itself or 2^-32."""
    q = torch.zeros(B, L, G * D, device='cuda', dtype=F16)
    q[..., ::D] = 1
    k = torch.zeros(1, S, D, device='cuda', dtype=F16)
    k[:, :, 0] = -far * math.log(2)
    k[:, 0] = 0
    v = (1 + torch.rand(1, S, D, device='cuda')).to(F16)
    o = ops.cross_attention(q, k.expand(B, S, D), v.expand(B, S, D), G, scale=1.0).double().view(-1, D)
    s = k[0, :, 0].double()
    p = torch.softmax(s, 0)
    want = (p[:, None] * v[0].double()).sum(0)
    # (the exponent's own error is that of a score of up to 27 ln 2; the sums' as everywhere above: (S / 16) u.  65 536 keys of 2^-25.3 are worth
    # 1.6e-3 of o, three times the result's half step: left out, they would show)
    e, rel = 2.0 ** -11, p / p.max()
    off = torch.where(rel >= 2.0 ** -21, p * e, 2.0 ** -32 * p.max()) + p * (S / 16 + 300) * U
    tol = (off[:, None] * v[0].double()).sum(0) + e * want
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol).max())
