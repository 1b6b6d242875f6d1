"""The training paths that the LayerNorm and attention operators carry, as modules: the decoder layer, a RoI block's masked attention, a
ray decoder layer; against the same modules in float64 on the CPU (torch formulation, materialised scores).

Tolerance: the float32 torch formulation of the same module on the GPU is the yardstick - two float32 evaluations of one chain differ
from float64 by errors of one size; the operators are given twice its largest error (and 2^-20 of the tensor's largest value, the level
of a dozen roundings, where the yardstick is exact).  Half precision the same, with 2^-10."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from deepinteraction_amd import autograd, ops
from deepinteraction_amd.mmdet3d_plugin.models.necks import fusion_transformerv4 as ft
from deepinteraction_amd.mmdet3d_plugin.models.utils import decoder_utils as du, transformer_bricks as tb


@pytest.fixture
def plain(monkeypatch):
    """Switches the modules to their torch formulation (and back with plain(False))."""
    def switch(on):
        if on:
            monkeypatch.setattr(du, 'cross_attention_usable', lambda *a: False)
            monkeypatch.setattr(ft, 'cross_attention_usable', lambda *a: False)
            monkeypatch.setattr(tb, '_norm_type', lambda *a: None)
        else:
            monkeypatch.undo()
    return switch


def grads(module, run, dev, dtype, amp=False):
    m = copy.deepcopy(module).to(dev, dtype)
    leaves, out = run(m, dev, dtype)
    g = torch.Generator().manual_seed(4)
    w = torch.randn(out.shape, generator=g).to(dev, torch.float64 if dtype == torch.float64 else torch.float32)
    with torch.autocast('cuda', enabled=False):
        (out.to(w.dtype) * w).sum().backward()
    named = {'out': out.detach()}
    named |= {f'd input {i}': t.grad for i, t in enumerate(leaves) if t.grad is not None}
    named |= {n: p.grad for n, p in m.named_parameters() if p.grad is not None}
    return {n: t.double().cpu() for n, t in named.items()}


def compare(module, run, plain, floor, amp=False):
    ref = grads(module, run, 'cpu', torch.float64)
    with torch.autocast('cuda', enabled=amp):
        plain(True)
        yard = grads(module, run, 'cuda', torch.float32)
        plain(False)
        calls = []
        fwd, norm = ops.cross_attention_train_fwd, ops.layernorm_train_fwd
        ops.cross_attention_train_fwd = lambda *a, **k: (calls.append('a'), fwd(*a, **k))[1]
        ops.layernorm_train_fwd = lambda *a, **k: (calls.append('n'), norm(*a, **k))[1]
        try:
            own = grads(module, run, 'cuda', torch.float32)
        finally:
            ops.cross_attention_train_fwd, ops.layernorm_train_fwd = fwd, norm
    assert set(own) == set(ref) == set(yard)
    for n, r in ref.items():
        top = float(r.abs().max())
        e, y = float((own[n] - r).abs().max()), float((yard[n] - r).abs().max())
        # a bias that feeds only a softmax's constant (the keys'), or a norm: exact gradient 0, round-off on both sides
        assert e <= 2 * y + floor * max(top, 1e-3), (n, e, y, top)
    return calls


def tokens(shape, dev, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dev, dtype)


def decoder_layer(dev, dropout=0.0):
    torch.manual_seed(0)
    return du.TransformerDecoderLayer(128, 8, 256, dropout, 'relu', self_posembed=du.PositionEmbeddingLearned(2, 128),
                                      cross_posembed=du.PositionEmbeddingLearned(2, 128)).train()


def run_decoder(m, dev, dtype):
    q, k = (tokens(s, dev, dtype, i).requires_grad_(True) for i, s in enumerate(((2, 128, 40), (2, 128, 600))))
    qp, kp = tokens((2, 40, 2), dev, dtype, 5), tokens((2, 600, 2), dev, dtype, 6)
    return (q, k), m(q, k, qp, kp)


@pytest.mark.parametrize('amp', [False, True])
def test_decoder_layer(plain, amp):
    calls = compare(decoder_layer('cpu'), run_decoder, plain, 2.0 ** -10 if amp else 2.0 ** -20, amp)
    assert calls.count('a') == 2 and calls.count('n') == 3


@pytest.mark.parametrize('amp', [False, True])
def test_ray_decoder_layer(plain, amp):
    torch.manual_seed(1)
    m = ft._RayDecoderLayer(128, 8, 256, dropout=0.0).train()

    def run(m, dev, dtype):
        t, mem = (tokens(s, dev, dtype, i).requires_grad_(True) for i, s in enumerate(((7, 60, 128), (7, 112, 128))))
        return (t, mem), m(t, mem)
    calls = compare(m, run, plain, 2.0 ** -10 if amp else 2.0 ** -20, amp)
    assert calls.count('a') == 2 and calls.count('n') == 3


def test_attention_among_the_queries_of_a_view(plain):
    """mha_tokens with the RoI blocks' mask; queries of no view have an empty row and are dropped, as by the blocks."""
    torch.manual_seed(2)
    m = du.MultiheadAttention(128, 8).train()
    view = torch.randint(-1, 3, (2, 50), generator=torch.Generator().manual_seed(3))
    allowed = (view[:, :, None] == view[:, None, :]) & (view[:, :, None] >= 0)

    def run(m, dev, dtype):
        x = tokens((2, 50, 128), dev, dtype, 1).requires_grad_(True)
        y = du.mha_tokens(x, x, x, m.in_proj_weight, m.in_proj_bias, m.out_proj, 8, 0.0, allowed.to(dev))
        return (x,), torch.where((view >= 0)[..., None].to(dev), y, torch.zeros_like(y))

    ref = grads(m, lambda m, dev, dtype: run(m, dev, dtype), 'cuda', torch.float32)
    assert all(torch.isfinite(t).all() for t in ref.values())
    # the torch formulation gives NaN for the empty rows, and NaN * 0 in its gradients: the oracle attends with one key for them
    ids = torch.arange(50)
    patched = allowed | ((view < 0)[:, :, None] & (ids[None, :, None] == ids[None, None, :]))

    def run_patched(m, dev, dtype):
        x = tokens((2, 50, 128), dev, dtype, 1).requires_grad_(True)
        y = du.mha_tokens(x, x, x, m.in_proj_weight, m.in_proj_bias, m.out_proj, 8, 0.0, patched.to(dev))
        return (x,), torch.where((view >= 0)[..., None].to(dev), y, torch.zeros_like(y))
    want = grads(m, run_patched, 'cpu', torch.float64)
    plain(True)
    yard = grads(m, run_patched, 'cuda', torch.float32)
    plain(False)
    for n, r in want.items():
        e, y = float((ref[n] - r).abs().max()), float((yard[n] - r).abs().max())
        assert e <= 2 * y + 2.0 ** -20 * max(float(r.abs().max()), 1e-3), (n, e, y)


def test_dropout_reaches_the_attention_and_its_seed_is_torch_s(plain):
    """Training with dropout: the same CPU seed gives the same step, another seed another; evaluation has none."""
    m = decoder_layer('cpu', dropout=0.3).cuda()

    def step(seed):
        torch.manual_seed(seed)
        for p in m.parameters():
            p.grad = None
        (q, _), out = run_decoder(m, 'cuda', torch.float32)
        out.square().sum().backward()
        return out.detach().clone(), q.grad.clone()
    a, b, c = step(1), step(1), step(2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], c[0])
    q = tokens((2, 30, 128), 'cuda', torch.float32, 0)
    kv = tokens((2, 90, 256), 'cuda', torch.float32, 1)
    torch.manual_seed(5)
    x = autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)
    y = autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)
    torch.manual_seed(5)
    assert torch.equal(x, autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)) and not torch.equal(x, y)


def test_packed_and_separate_projections_agree():
    q = tokens((2, 33, 64), 'cuda', torch.float16, 0)
    kv = tokens((2, 77, 64), 'cuda', torch.float16, 1)
    outs = []
    for packed in (True, False):
        a, b = q.clone().requires_grad_(True), kv.clone().requires_grad_(True)
        o = autograd.cross_attention(a, b, None, 4) if packed else autograd.cross_attention(a, *b.chunk(2, -1), 4)
        o.backward(tokens((2, 33, 64), 'cuda', torch.float16, 2))
        outs.append((o.detach(), a.grad, b.grad))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    with torch.no_grad():
        assert torch.equal(autograd.cross_attention(q, kv, None, 4), outs[0][0])


def test_captured_training_step_of_a_layer():
    """Forward and backward of the decoder layer in one graph, replayed with new inputs between eager steps."""
    m = decoder_layer('cpu').cuda()
    q, k = torch.empty(1, 128, 40, device='cuda'), torch.empty(1, 128, 600, device='cuda')
    qp, kp = tokens((1, 40, 2), 'cuda', torch.float32, 5), tokens((1, 600, 2), 'cuda', torch.float32, 6)
    params = [p for p in m.parameters()]

    def step():
        out = m(q, k, qp, kp)
        return (out,) + torch.autograd.grad(out.square().mean(), params, allow_unused=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    q.normal_(), k.normal_()
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = [None if t is None else t for t in step()]
    bn = [b for mod in m.modules() if isinstance(mod, torch.nn.BatchNorm1d) for b in (mod.running_mean, mod.running_var, mod.num_batches_tracked)]
    for n in range(3):
        q.normal_(), k.normal_()
        keep = [b.clone() for b in bn]
        graph.replay()
        torch.cuda.synchronize()
        got = [None if t is None else t.detach().clone() for t in static]
        for b, v in zip(bn, keep):
            b.copy_(v)
        for a, b in zip(got, step()):
            # library products may be chosen differently inside and outside a capture: a few roundings of the largest value
            assert (a is None) == (b is None) and (a is None or float((a - b).abs().max()) <= 2.0 ** -18 * max(float(b.abs().max()), 1e-6)), n


def test_dropout_in_a_captured_step_is_fresh_in_every_replay(monkeypatch):
    """Forward and backward of the attention in one graph: every replay has a mask of its own, the same in both directions - the one that the
    word drawn by that replay gives - and a generator that is seeded again repeats it."""
    q, kv, go = tokens((2, 37, 64), 'cuda', torch.float32, 0), tokens((2, 90, 128), 'cuda', torch.float32, 1), tokens((2, 37, 64), 'cuda', torch.float32, 2)
    q, kv = q.requires_grad_(True), kv.requires_grad_(True)

    def step():
        o = autograd.cross_attention(q, kv, None, 4, dropout_p=0.4)
        return (o.detach(),) + torch.autograd.grad(o, (q, kv), go)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    words, fwd = [], ops.cross_attention_train_fwd

    def keep(*a, **k):
        words.append(a[10])
        return fwd(*a, **k)
    monkeypatch.setattr(ops, 'cross_attention_train_fwd', keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    monkeypatch.undo()
    assert len(words) == 1 and words[0] is not None
    seen = []
    with torch.no_grad():
        k, v = kv.chunk(2, -1)
        for n in range(4):
            if n >= 2:
                torch.cuda.manual_seed(11)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            o, lse = ops.cross_attention_train_fwd(q, k, v, 4, dropout_p=0.4, seed=0, seed_word=words[0])
            gq, gk, gv = ops.cross_attention_train_bwd(q, k, v, o, go, lse, 4, dropout_p=0.4, seed=0, seed_word=words[0])
            assert all(torch.equal(a, b) for a, b in zip(got, (o, gq, torch.cat((gk, gv), -1)))), n
            seen.append((int(words[0]), got))
    assert len({w for w, _ in seen}) == 3 and not torch.equal(seen[0][1][0], seen[1][1][0])
    assert seen[2][0] == seen[3][0] and all(torch.equal(a, b) for a, b in zip(seen[2][1], seen[3][1]))


def test_dropout_follows_the_cuda_generator():
    """A saved and restored state of the device's generator repeats the mask; the CPU's generator is left alone."""
    q, kv = tokens((2, 30, 128), 'cuda', torch.float32, 0), tokens((2, 90, 256), 'cuda', torch.float32, 1)
    host, state = torch.get_rng_state(), torch.cuda.get_rng_state()
    a = autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)
    b = autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)
    torch.cuda.set_rng_state(state)
    assert torch.equal(a, autograd.cross_attention(q, kv, None, 8, dropout_p=0.5)) and not torch.equal(a, b)
    assert torch.equal(b, autograd.cross_attention(q, kv, None, 8, dropout_p=0.5))
    assert torch.equal(host, torch.get_rng_state())


def test_dropout_s_backward_keeps_the_word_of_its_forward():
    """A word that is registered for the forward alone, as around a capture, is the backward's as well."""
    q, kv = tokens((1, 30, 64), 'cuda', torch.float32, 0).requires_grad_(True), tokens((1, 70, 128), 'cuda', torch.float32, 1)
    word = torch.full((1,), 41, dtype=torch.int64, device='cuda')
    grads = []
    for cleared in (False, True):
        torch.manual_seed(3)
        ops.set_i2p_seed_tensor(word)
        try:
            o = autograd.cross_attention(q, kv, None, 4, dropout_p=0.5)
            if cleared:
                ops.set_i2p_seed_tensor(None)
            grads.append(torch.autograd.grad(o, q, torch.ones_like(o))[0])
        finally:
            ops.set_i2p_seed_tensor(None)
    assert torch.equal(*grads)


def test_hooks_and_subclasses_of_the_norms_are_called():
    """`post_norm` is the module's call for every norm that is more than its LayerNorm."""
    x, branch = tokens((2, 9, 128), 'cuda', torch.float32, 0).requires_grad_(True), tokens((2, 9, 128), 'cuda', torch.float32, 1)
    norm, seen = torch.nn.LayerNorm(128).cuda(), []
    want = tb.post_norm(norm, x, branch)
    for register in (norm.register_forward_hook, norm.register_forward_pre_hook, norm.register_full_backward_hook, norm.register_full_backward_pre_hook,
                     torch.nn.modules.module.register_module_forward_hook):
        handle = register(lambda *a: seen.append(register.__name__))
        out = tb.post_norm(norm, x, branch)
        out.sum().backward()
        handle.remove()
        assert seen and set(seen) == {register.__name__} and torch.allclose(out, want, atol=1e-5), register.__name__
        seen.clear()

    class Twice(torch.nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)
    assert torch.allclose(tb.post_norm(Twice(128).cuda(), x, branch), 2 * want, atol=1e-5)
    patched = torch.nn.LayerNorm(128).cuda()
    patched.forward = lambda x: x * 0
    assert not tb.post_norm(patched, x, branch).any()


def test_transforms_and_forward_mode_pass_the_modules():
    """torch.func's transforms and forward-mode differentiation of the attention and norm steps, as torch's own operations have them: against
    the float64 modules on the CPU (float32 chains of a dozen operations: 2^-16 of the largest value, or of 1.  The functional's gradient is
    a difference: with y = h, d sum y^2 = 2 rstd (h - h mean h^2) = 2 rstd h eps / (var + eps), about 1e-5, of terms 2 rstd h of 1 and more)."""
    torch.manual_seed(3)
    m = du.MultiheadAttention(128, 8).train()
    norm = torch.nn.LayerNorm(128)
    x, dx = tokens((3, 20, 128), 'cpu', torch.float64, 0), tokens((3, 20, 128), 'cpu', torch.float64, 1)

    def run(dev, dtype):
        a, n = copy.deepcopy(m).to(dev, dtype), copy.deepcopy(norm).to(dev, dtype)
        f = lambda t: tb.post_norm(n, t, du.mha_tokens(t, t, t, a.in_proj_weight, a.in_proj_bias, a.out_proj, 8))
        t, dt = x.to(dev, dtype), dx.to(dev, dtype)
        out = list(torch.func.jvp(f, (t,), (dt,)))
        out.append(torch.func.grad(lambda t: f(t).square().sum())(t))
        out.append(torch.func.vmap(lambda t: f(t[None])[0])(t))
        with torch.autograd.forward_ad.dual_level():
            out.append(torch.autograd.forward_ad.unpack_dual(f(torch.autograd.forward_ad.make_dual(t, dt))).tangent)
        return [o.detach().double().cpu() for o in out]
    for got, want in zip(run('cuda', torch.float32), run('cpu', torch.float64)):
        assert float((got - want).abs().max()) <= 2.0 ** -16 * max(float(want.abs().max()), 1.0)


def test_everything_dropped():
    """A dropout of 1, which torch's functions allow: out_proj's bias, and no gradient."""
    torch.manual_seed(4)
    m = du.MultiheadAttention(64, 4).cuda()
    x = tokens((2, 9, 64), 'cuda', torch.float32, 0).requires_grad_(True)
    y = du.mha_tokens(x, x, x, m.in_proj_weight, m.in_proj_bias, m.out_proj, 4, 1.0)
    assert torch.allclose(y, m.out_proj.bias.expand_as(y), atol=1e-6)
    y.sum().backward()
    assert not x.grad.any()


def second_order(f, inputs, seed):
    """[outputs, gradients, gradients of a functional of the gradients] of f(*inputs), every input a leaf."""
    leaves = [t.detach().clone().requires_grad_(True) for t in inputs]
    outs = f(*leaves)
    dt, dev = leaves[0].dtype, leaves[0].device
    gos = [tokens(o.shape, dev, dt, seed + i).requires_grad_(True) for i, o in enumerate(outs)]
    grads = torch.autograd.grad(outs, leaves, gos, create_graph=True)
    total = sum((g * tokens(g.shape, dev, dt, seed + 10 + i)).sum() for i, g in enumerate(grads))
    again = torch.autograd.grad(total, leaves + gos, allow_unused=True)
    return [t.detach().double().cpu() for t in list(outs) + list(grads)] + [None if t is None else t.double().cpu() for t in again]


def test_gradients_of_gradients():
    """create_graph through both Functions, against float64: float32 sums of up to a hundred terms, twice - 2^-14 of the largest value."""
    B, L, S, H, Hk, D = 2, 9, 30, 4, 2, 16
    lengths = torch.tensor([30, 11])
    allowed = torch.rand(B, L, S, generator=torch.Generator().manual_seed(0)) < 0.7
    allowed[:, 3] = False
    keep = allowed & (torch.arange(S) < lengths[:, None])[:, None]

    def plain(q, k, v):
        qh, kh, vh = q.view(B, L, H, D).transpose(1, 2), k.view(B, S, Hk, D).transpose(1, 2), v.view(B, S, Hk, D).transpose(1, 2)
        s = torch.matmul(qh, kh.repeat_interleave(H // Hk, 1).transpose(-1, -2)) * 0.3
        s = torch.where(keep.any(-1)[:, None, :, None], s.masked_fill(~keep[:, None], float('-inf')), torch.zeros_like(s))
        a = torch.softmax(s, -1) * keep[:, None]
        return (torch.matmul(a, vh.repeat_interleave(H // Hk, 1)).transpose(1, 2).reshape(B, L, -1),)

    def own(q, k, v):
        return (autograd.cross_attention(q, k, v, H, 0.3, lengths.cuda().int(), None, allowed.cuda()),)
    cases = [(plain, own, [(B, L, H * D), (B, S, Hk * D), (B, S, Hk * D)]),
             (lambda q, kv: plain(q, *kv.chunk(2, -1)), lambda q, kv: (autograd.cross_attention(q, kv, None, H, 0.3, lengths.cuda().int(), None, allowed.cuda()),),
              [(B, L, H * D), (B, S, 2 * Hk * D)])]
    ln = torch.nn.functional.layer_norm
    cases += [(lambda x, r, w, b: (ln(x + r, (24,), w, b, 1e-3),), lambda x, r, w, b: (autograd.AddLayerNorm.apply(x, r, w, b, 1e-3, None, False),),
               [(5, 7, 24), (5, 7, 24), (24,), (24,)]),
              (lambda x, w, b: (ln(x, (24,), w, b, 1e-3),), lambda x, w, b: (autograd.AddLayerNorm.apply(x, None, w, b, 1e-3, None, False),),
               [(5, 7, 24), (24,), (24,)]),
              (lambda x, r, w, b: (ln(x + r, (24,), w, b, 1e-3), x + r), lambda x, r, w, b: autograd.AddLayerNorm.apply(x, r, w, b, 1e-3, None, True),
               [(5, 7, 24), (5, 7, 24), (24,), (24,)]),
              # an input that another one is computed from
              (lambda x, w, b: (ln(x + x * x, (24,), w, b, 1e-3),), lambda x, w, b: (autograd.AddLayerNorm.apply(x, x * x, w, b, 1e-3, None, False),),
               [(5, 7, 24), (24,), (24,)])]
    for n, (f64, f, shapes) in enumerate(cases):
        inputs = [tokens(s, 'cpu', torch.float64, i) for i, s in enumerate(shapes)]
        want, got = second_order(f64, inputs, 20), second_order(f, [t.float().cuda() for t in inputs], 20)
        for i, (a, b) in enumerate(zip(got, want)):
            if a is None or b is None:
                assert all(t is None or not t.any() for t in (a, b)), (n, i)
            else:
                assert float((a - b).abs().max()) <= 2.0 ** -14 * max(float(b.abs().max()), 1.0), (n, i, float((a - b).abs().max()), float(b.abs().max()))


def test_the_formula_s_dropout_is_the_kernel_s():
    """The gradients of a backward with create_graph, which torch's operations compute, against the kernel's: the same decisions, heads shared
    and odd numbers of keys among them (float32 both: 2^-16 of the largest)."""
    for L, S, H, Hk, D, seed in ((5, 70, 4, 2, 32, 7), (90, 151, 8, 8, 16, 2 ** 63 + 5)):
        q, kv = tokens((2, L, H * D), 'cuda', torch.float32, 0).requires_grad_(True), tokens((2, S, 2 * Hk * D), 'cuda', torch.float32, 1).requires_grad_(True)
        go, word = tokens((2, L, H * D), 'cuda', torch.float32, 2), torch.full((1,), 3, dtype=torch.int64, device='cuda')
        for w in (None, word):
            o = autograd.CrossAttention.apply(q, kv, None, H, None, None, None, None, 0.3, seed, w)
            f = autograd.attention_formula(q, kv, None, H, dropout_p=0.3, seed=seed, seed_word=w)
            a = torch.autograd.grad(o, (q, kv), go, retain_graph=True)
            b = torch.autograd.grad(o, (q, kv), go, create_graph=True)
            for x, y in zip((o,) + a, (f,) + b):
                assert float((x - y).abs().max()) <= 2.0 ** -16 * float(y.abs().max())
            assert b[0].requires_grad and not a[0].requires_grad


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize('amp', [None, torch.float16, torch.bfloat16], ids=str)
def test_the_image_branch_s_norms_keep_their_types(monkeypatch, dtype, amp):
    """The Swin image branch with its norms in the kernels and as torch evaluates them, plain and under autocast (whose norms are float32): the
    same types, and values as far apart as a dozen blocks' roundings leave them - a norm in the other type, or a sum carried in 16 bits,
    doubles the count of those: 32 half steps of the largest value."""
    from deepinteraction_amd.mmdet3d_plugin.models.detectors import image_glue
    net = image_glue.FrozenSwinFPN(dtype=dtype)
    net.load_mmdet_state(*net.synthetic_state(seed=1))
    net = net.cuda()
    img = tokens((2, 3, 64, 96), 'cuda', torch.float32, 0)

    def run():
        with torch.autocast('cuda', dtype=amp or torch.float16, enabled=amp is not None):
            return net.stage_maps(img)
    calls, real = [], ops.layernorm
    monkeypatch.setattr(ops, 'layernorm', lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    got = run()
    assert len(calls) >= 20 or {dtype, amp} == {torch.float16, torch.bfloat16}
    monkeypatch.setattr(ops, 'layernorm_type', lambda *a: None)
    want = run()
    half = max(torch.finfo(t).eps for t in (dtype, amp or dtype)) / 2
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert float((a.float() - b.float()).abs().max()) <= max(32 * half, 2.0 ** -14) * float(b.float().abs().max())


def test_a_word_registered_later_does_not_reach_the_backward():
    q, kv = tokens((1, 30, 64), 'cuda', torch.float32, 0).requires_grad_(True), tokens((1, 70, 128), 'cuda', torch.float32, 1)
    word = torch.full((1,), 41, dtype=torch.int64, device='cuda')
    grads = []
    for registered in (None, word):
        torch.manual_seed(3)
        o = autograd.cross_attention(q, kv, None, 4, dropout_p=0.5)
        ops.set_i2p_seed_tensor(registered)
        try:
            grads.append(torch.autograd.grad(o, q, torch.ones_like(o))[0])
        finally:
            ops.set_i2p_seed_tensor(None)
    assert torch.equal(*grads)
