"""The formulas that the LayerNorm and attention Functions differentiate twice (autograd.attention_formula and the dropout decisions in torch's
operations), on the CPU in float32 against float64; the same through the kernels' Functions on the GPU: tests/test_token_training_gpu.py."""
import math

import torch

from deepinteraction_amd import autograd


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def test_attention_formula():
    B, L, S, H, Hk, D = 3, 5, 9, 4, 2, 8
    q, k, v = randn(B, L, H * D, seed=0), randn(B, S, Hk * D, seed=1), randn(B, S, Hk * D, seed=2)
    lengths, mask = torch.tensor([9, 4, 0]), torch.rand(B, S, generator=torch.Generator().manual_seed(3)) < 0.7
    allowed = torch.rand(B, L, S, generator=torch.Generator().manual_seed(4)) < 0.6
    allowed[0, 2] = False
    keep = allowed & mask[:, None] & (torch.arange(S) < lengths[:, None])[:, None]
    want = torch.zeros(B, L, H, D, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            for l in range(L):
                at = keep[b, l].nonzero()[:, 0]
                if len(at):
                    K, V = (t[b, at].double().view(-1, Hk, D)[:, h // (H // Hk)] for t in (k, v))
                    want[b, l, h] = torch.softmax(K @ q[b, l, h * D:(h + 1) * D].double() * 0.3, 0) @ V
    dead = ~(mask & (torch.arange(S) < lengths[:, None]))
    k, v = k.clone(), v.clone()
    k[dead], v[dead] = math.nan, math.inf                            # excluded keys and queries without keys may hold anything
    q = q.clone()
    q[0, 2] = math.nan
    for packed in (False, True):
        args = (torch.cat((k, v), -1), None) if packed else (k, v)
        got = autograd.attention_formula(q, *args, H, 0.3, lengths, mask, allowed)
        assert (got.double() - want.view(B, L, -1)).abs().max() <= 2.0 ** -20 * 8


def test_dropout_factors():
    f = autograd._dropout_factors(2, 3, 40, 101, 0.3, 12345678901234567890, None, 'cpu')
    drop = round(0.3 * 65536)
    assert f.shape == (2, 3, 40, 101) and set(f.unique().tolist()) == {0.0, torch.tensor(65536 / (65536 - drop)).item()}
    assert abs(float((f == 0).float().mean()) - 0.3) <= 5 * math.sqrt(0.21 / f.numel())
    word = torch.tensor([7])
    assert torch.equal(autograd._dropout_factors(1, 2, 9, 20, 0.5, 5, word, 'cpu'), autograd._dropout_factors(1, 2, 9, 20, 0.5, 12, None, 'cpu'))
    big = autograd._dropout_factors(1, 2, 9, 20, 0.5, 2 ** 64 - 3, word, 'cpu')      # the sum is taken modulo 2^64
    assert torch.equal(big, autograd._dropout_factors(1, 2, 9, 20, 0.5, 4, None, 'cpu'))


def test_formula_gradients_are_each_input_s_share():
    x = randn(4, seed=0).double().requires_grad_(True)
    y = x * x                                                        # an input that another one was computed from
    gx, none, gy = autograd._formula_grads(lambda x, c, y: x * c * y, (x, torch.tensor(3.0), y), (True, False, True), torch.ones(4).double())
    assert none is None and torch.equal(gx, 3 * y) and torch.equal(gy, 3 * x)
    assert torch.allclose(torch.autograd.grad(gx.sum(), x)[0], 6 * x)


def test_tokens_without_an_allowed_key():
    """`mha_tokens` in its torch formulation gives such a row the projection's bias and reaches no gradient through it, as on the GPU; the others
    are as with the rows left out."""
    from deepinteraction_amd.mmdet3d_plugin.models.utils import decoder_utils as du
    torch.manual_seed(0)
    m, H = du.MultiheadAttention(32, 4), 4
    torch.nn.init.normal_(m.in_proj_bias), torch.nn.init.normal_(m.out_proj.bias)
    allowed = torch.rand(2, 7, 7, generator=torch.Generator().manual_seed(1)) < 0.5
    allowed[..., 0] = True
    allowed[0, 2], allowed[1, 6] = False, False
    some = allowed.any(-1)
    grads = []
    for mask in (allowed, allowed | ~some[..., None]):               # the second: those rows attend, and are dropped afterwards
        x = randn(2, 7, 32, seed=3).requires_grad_(True)
        y = du.mha_tokens(x, x, x, m.in_proj_weight, m.in_proj_bias, m.out_proj, H, 0.0, mask)
        if mask is allowed:
            assert torch.equal(y[~some], m.out_proj.bias.expand(2, 32))
        kept = torch.where(some[..., None], y, torch.zeros_like(y))
        m.zero_grad()
        (kept * randn(2, 7, 32, seed=4)).sum().backward()
        grads.append([kept.detach(), x.grad] + [p.grad.clone() for p in m.parameters()])
    assert all(torch.allclose(a, b, rtol=0, atol=2.0 ** -20 * max(1.0, float(b.abs().max()))) for a, b in zip(*grads))
