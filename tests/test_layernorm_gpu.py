"""csrc/layernorm.hip, layernorm_bwd.hip: LayerNorm with its residual add, forward and backward, against float64.

Tolerances.  With u = 2^-24 (half a float32 step) a sum of n terms that is taken as m sequential additions and a tree errs by at
most (m + log n) u sum|terms|: 16 sequential additions in a lane and at most 10 levels give K = 32 with the additions around them.
`y`: its own rounding (half a step of its type) + K u (max|s| rstd + |h|) |w|: mean and centring see errors of the size of s, the
rest is relative.  `gx`: half a step + K u (|terms| of its formula).  `gw`, `gb`: half a step + (rows a lane adds + K) u sum|terms|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from deepinteraction_amd import ops
from deepinteraction_amd.autograd import AddLayerNorm

U, K = 2.0 ** -24, 32
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t):
    return torch.finfo(t).eps / 2


def make(rows, C, xt, rt, wt, seed=0, offset=0.5):
    g = torch.Generator(device='cuda').manual_seed(seed + rows + 7 * C)
    r = lambda *s: torch.randn(*s, device='cuda', generator=g)
    x = (r(rows, C) + offset * r(rows, 1)).to(xt)
    res = None if rt is None else r(rows, C).to(rt)
    return x, res, (1 + 0.2 * r(C)).to(wt), (0.1 * r(C)).to(wt), r(rows, C), r(rows, C)


def formula(s, w, b, gy, gs, eps):
    """Everything in float64 from the sum s, with the magnitudes that the tolerances need."""
    s, w, b, gy = s.double(), w.double(), b.double(), gy.double()
    mu = s.mean(-1, keepdim=True)
    rstd = ((s - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (s - mu) * rstd
    g = gy * w
    gx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    if gs is not None:
        gx = gx + gs.double()
    rel = s.abs().amax(-1, keepdim=True) * rstd + h.abs()          # |h|'s absolute error in units of K u
    gmag = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + (rel + h.abs()) * (g * h).abs().mean(-1, keepdim=True)
                   + h.abs() * (g.abs() * rel).mean(-1, keepdim=True)) + (0 if gs is None else gs.double().abs())
    return dict(y=h * w + b, y_tol=rel * w.abs() + b.abs(), gx=gx, gx_tol=gmag, gw=(gy * h).sum(0), gw_tol=(gy * h).abs().sum(0),
                gw_rel=(gy.abs() * rel).sum(0), gb=gy.sum(0), gb_tol=gy.abs().sum(0), mean=mu[..., 0], rstd=rstd[..., 0])


def close(got, want, tol):
    assert got.shape == want.shape
    bad = (got.double() - want).abs() > half_step(got.dtype) * want.abs() + tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() - tol).max()))


def check(rows, C, xt, rt, wt, yt, with_sum, eps=1e-5, seed=0):
    x, res, w, b, gy, gs = make(rows, C, xt, rt, wt, seed)
    gy, gs = gy.to(yt), gs.to(xt) if with_sum else None
    y, total, mean, rstd = ops.layernorm_train_fwd(x, w, b, res, eps, with_sum, yt)
    s = x.double() if res is None else x.double() + res.double()
    if with_sum:
        assert torch.equal(total, (x.float() + res.float()).to(xt))
        s = total.double()
        gx, gres, gw, gb = ops.layernorm_train_bwd(gy, total, w, mean, rstd, grad_sum=gs)
        assert gres is None
    else:
        assert total is None
        gx, gres, gw, gb = ops.layernorm_train_bwd(gy, x, w, mean, rstd, res=res)
    f = formula(s, w, b, gy, gs, eps)
    smax = s.abs().amax(-1)
    assert ((mean.double() - f['mean']).abs() <= K * U * smax).all()
    assert ((rstd.double() - f['rstd']).abs() <= K * U * f['rstd'] * (1 + smax * f['rstd'])).all()
    close(y, f['y'], K * U * f['y_tol'])
    close(gx, f['gx'], 2 * K * U * f['gx_tol'])
    if gres is not None:
        close(gres, f['gx'], 2 * K * U * f['gx_tol'])
    n = rows / 256 + K
    close(gw, f['gw'], n * U * f['gw_tol'] + K * U * f['gw_rel'])
    close(gb, f['gb'], n * U * f['gb_tol'])
    # the inference form: the same bits, and the sum with it
    got = ops.layernorm(x, w, b, res, eps, with_sum, yt)
    assert torch.equal(got[0] if with_sum else got, y) and (not with_sum or torch.equal(got[1], total))
    again = ops.layernorm_train_bwd(gy, total if with_sum else x, w, mean, rstd, res=None if with_sum else res, grad_sum=gs)
    assert torch.equal(again[0], gx) and torch.equal(again[2], gw) and torch.equal(again[3], gb)


@pytest.mark.parametrize('C', [1, 2, 7, 8, 96, 127, 128, 129, 136, 512, 513, 768, 1000, 1024, 1032, 2048, 2049, 4096, 5000, 8192, 10001, 16384])
@pytest.mark.parametrize('rows', [1, 37])
def test_widths(C, rows):
    check(rows, C, F32, F32, F32, F32, False)
    check(rows, C, BF16, BF16, BF16, BF16, True)


@pytest.mark.parametrize('types', [(F32, None, F32, F32), (F32, F16, F32, F32), (F32, BF16, F32, F32), (F16, F32, F32, F32),
                                   (F16, F16, F16, F16), (F16, F16, F32, F32), (F16, None, F16, F16), (BF16, None, F32, BF16),
                                   (BF16, BF16, BF16, F32)], ids=str)
@pytest.mark.parametrize('rows,C', [(200, 128), (1000, 131), (333, 640), (70, 1536), (9, 6000)])
def test_types(rows, C, types):
    xt, rt, wt, yt = types
    check(rows, C, xt, rt, wt, yt, False)
    if rt is not None:
        check(rows, C, xt, rt, wt, yt, True)


@pytest.mark.parametrize('rows,C', [(72000, 128), (200001, 16), (20011, 257), (8192, 4096)])
def test_many_rows(rows, C):
    check(rows, C, F32, F16, F32, F32, False)


def test_no_rows():
    x = torch.empty(0, 128, device='cuda')
    w, b = torch.ones(128, device='cuda'), torch.zeros(128, device='cuda')
    y, _, mean, rstd = ops.layernorm_train_fwd(x, w, b)
    gx, _, gw, gb = ops.layernorm_train_bwd(x, x, w, mean, rstd)
    assert y.shape == gx.shape == (0, 128) and not gw.any() and not gb.any()


@pytest.mark.parametrize('lead,C', [(8, 128), (3, 128), (5, 131), (64, 1024)])
def test_strided_rows_and_offsets(lead, C):
    """Columns of a wider matrix, read in place: row stride and start are not the kernel's own (lead 3 and 5: no 16-byte rows)."""
    g = torch.Generator(device='cuda').manual_seed(5)
    wide = torch.randn(50, 2 * C + 2 * lead, device='cuda', generator=g)
    x, res = wide[:, lead:lead + C], wide[:, lead + C:lead + 2 * C]
    w, b = torch.randn(C, device='cuda', generator=g), torch.randn(C, device='cuda', generator=g)
    y, _, mean, rstd = ops.layernorm_train_fwd(x, w, b, res)
    # a row that starts on 16 bytes is read in chunks of 8 columns, any other one column by column: two orders of the same sums,
    # each within K u of the formula's - so both are held to the formula, and their bits may differ
    gy = wide[:, :C]
    f = formula(x.double() + res.double(), w, b, gy, None, 1e-5)
    close(y, f['y'], K * U * f['y_tol'])
    got = ops.layernorm_train_bwd(gy, x, w, mean, rstd, res=res)
    close(got[0], f['gx'], 2 * K * U * f['gx_tol'])
    ref = ops.layernorm_train_bwd(gy.contiguous(), x.contiguous(), w, mean, rstd, res=res.contiguous())
    for p, q, tol in zip((got[0], got[2], got[3]), (ref[0], ref[2], ref[3]), (2 * f['gx_tol'], f['gw_tol'] + f['gw_rel'], f['gb_tol'])):
        assert ((p.double() - q.double()).abs() <= 2 * K * U * tol + U * q.double().abs()).all()
    t = torch.randn(7, C, 5, device='cuda', generator=g).transpose(1, 2)          # (7, 5, C): columns not contiguous
    assert torch.equal(ops.layernorm(t, w, b), ops.layernorm(t.contiguous(), w, b))
    e = torch.randn(1, 1, C, device='cuda', generator=g).expand(6, 4, C)          # one row for all
    assert torch.equal(ops.layernorm(e, w, b), ops.layernorm(e.contiguous(), w, b))


def test_a_row_of_nan_or_inf_stays_alone():
    x, res, w, b, gy, _ = make(40, 128, F32, F32, F32)
    y0, _, m0, r0 = ops.layernorm_train_fwd(x, w, b, res)
    g0 = ops.layernorm_train_bwd(gy, x, w, m0, r0, res=res)[0]
    x[3, 5], x[17, 0] = float('nan'), float('inf')
    y, _, mean, rstd = ops.layernorm_train_fwd(x, w, b, res)
    gx = ops.layernorm_train_bwd(gy, x, w, mean, rstd, res=res)[0]
    rest = [i for i in range(40) if i not in (3, 17)]
    assert y[3].isnan().all() and y[17].isnan().all()
    assert torch.equal(y[rest], y0[rest]) and torch.equal(gx[rest], g0[rest])


def test_large_mean_small_spread():
    """A row around 1000 with a spread of 1: the centred form keeps u |mean| / spread, not u |mean|^2 / spread^2."""
    x, _, w, b, gy, _ = make(64, 512, F32, None, F32, offset=0.0)
    x = x + 1000
    y = ops.layernorm(x, w, b)
    f = formula(x, w, b, gy, None, 1e-5)
    close(y, f['y'], K * U * f['y_tol'])
    const = torch.full((3, 512), 7.25, device='cuda')
    assert torch.equal(ops.layernorm(const, w, b), b.expand(3, -1))               # variance 0: h = 0


def test_against_differences():
    x, res, w, b, gy, gs = (t if t is None else t.requires_grad_(True) if i < 4 else t for i, t in enumerate(make(6, 24, F32, F32, F32)))
    loss = lambda x_, r_, w_, b_: (torch.nn.functional.layer_norm(x_ + r_, (24,), w_, b_) * gy.double() + (x_ + r_) * gs.double()).sum()
    y, total = AddLayerNorm.apply(x, res, w, b, 1e-5, F32, True)
    ((y * gy).sum() + (total * gs).sum()).backward()
    wide = [t.detach().double() for t in (x, res, w, b)]
    h = 1e-6
    for i, t in enumerate((x, res, w, b)):
        d = torch.randn_like(wide[i])
        lo, hi = ([p + s * h * d if j == i else p for j, p in enumerate(wide)] for s in (-1, 1))
        diff = float(loss(*hi) - loss(*lo)) / (2 * h)
        # central differences in float64: h^2 and 1e-16 / h terms below 1e-8; the kernel's gradient: K u of the terms' sum
        scale = float((t.grad.double() * d).abs().sum()) + 1
        assert abs(float((t.grad.double() * d).sum()) - diff) <= 1e-6 * scale * 10, (i, diff)


def test_autograd_function_matches_the_module():
    x, res, w, b, gy, _ = make(150, 128, F32, F32, F32)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w, b)]
    AddLayerNorm.apply(leaves[0], leaves[1], leaves[2], leaves[3], 1e-5, F32, False).backward(gy)
    f = formula(x.double() + res.double(), w, b, gy, None, 1e-5)
    close(leaves[0].grad, f['gx'], 2 * K * U * f['gx_tol'])
    close(leaves[1].grad, f['gx'], 2 * K * U * f['gx_tol'])
    leaves[0].grad += 1                                             # the two leaves' gradients are not one buffer
    close(leaves[1].grad, f['gx'], 2 * K * U * f['gx_tol'])
    close(leaves[2].grad, f['gw'], 64 * U * (f['gw_tol'] + f['gw_rel']))
    # a frozen weight and a missing residual get no gradient
    p = x.clone().requires_grad_(True)
    AddLayerNorm.apply(p, None, w, b, 1e-5, F32, False).backward(gy)
    assert p.grad is not None and w.grad is None


def test_unused_outputs():
    """Only the sum, or only the normalised value, reaches the loss."""
    x, res, w, b, gy, gs = make(33, 64, F32, F32, F32)
    for use in (0, 1):
        leaves = [t.clone().requires_grad_(True) for t in (x, res, w, b)]
        out = AddLayerNorm.apply(*leaves, 1e-5, F32, True)
        (out[use] * (gy, gs)[use]).sum().backward()
        if use == 1:
            assert torch.equal(leaves[0].grad, gs) and torch.equal(leaves[1].grad, gs) and (leaves[2].grad is None or not leaves[2].grad.any())
        else:
            f = formula((x + res).double(), w, b, gy, None, 1e-5)
            close(leaves[0].grad, f['gx'], 2 * K * U * f['gx_tol'])


def test_other_stream_and_captured():
    x, res, w, b, gy, _ = make(500, 256, F16, F16, F32)
    gy = gy.half()
    def step():
        y, _, m, r = ops.layernorm_train_fwd(x, w, b, res)
        return (y,) + ops.layernorm_train_bwd(gy, x, w, m, r, res=res)
    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = []
    for _ in range(2):                                              # two graphs, each with its own workspace, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        x.copy_(torch.randn_like(x))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), i


def test_refusals():
    x, res, w, b, gy, _ = make(4, 32, F32, F32, F32)
    y, _, m, r = ops.layernorm_train_fwd(x, w, b, res)
    for bad in (lambda: ops.layernorm(x, w[:31], b), lambda: ops.layernorm(x, w, b, res[:3]), lambda: ops.layernorm(x, w, b, with_sum=True),
                lambda: ops.layernorm(x[:, :0], w[:0], b[:0]), lambda: ops.layernorm(x, w, b.half()),
                lambda: ops.layernorm_train_bwd(gy[:3], x, w, m, r), lambda: ops.layernorm_train_bwd(gy, x, w, m[:3], r),
                lambda: ops.layernorm(torch.zeros(2, 16385, device='cuda'), torch.zeros(16385, device='cuda'), torch.zeros(16385, device='cuda'))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.layernorm(x.double(), w.double(), b.double())
    with pytest.raises(ops._lib.HipLibraryError):
        ops.layernorm(x.half(), w.bfloat16(), b.bfloat16())          # two 16-bit types in one call
    with pytest.raises(ops._lib.HipLibraryError):
        ops.layernorm(x, w, b, out_dtype=F16)                        # a 16-bit result of a float32 input
