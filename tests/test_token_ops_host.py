"""Refusals of the LayerNorm and cross-attention entry points, at the C interface and in Python: every call here is turned down before
anything is launched, so none of it needs a GPU (and no pointer below is ever followed)."""
import ctypes

import pytest
import torch

from deepinteraction_amd import _lib, autograd, ops

L = _lib.lib()
P = 1 << 20                                    # a pointer on 16 bytes that nobody reads


def attention(**kw):
    t = _lib.Attention()
    t.q = t.k = t.v = P
    t.B, t.L, t.S, t.heads, t.kv_heads, t.head_dim, t.dtype = 2, 5, 9, 4, 2, 16, _lib.DI_F16
    t.q_bs, t.q_rs, t.k_bs, t.k_rs, t.v_bs, t.v_rs = 320, 64, 288, 32, 288, 32
    t.scale = 0.25
    for name, value in kw.items():
        setattr(t, name, value)
    return t


def said():
    return L.di_last_error().decode()


BAD = [(dict(dtype=_lib.DI_F16_HL), 'dtype'), (dict(dtype=7), 'dtype'), (dict(B=-1), 'negative'), (dict(L=-1), 'negative'), (dict(S=-2), 'negative'),
       (dict(heads=0), 'heads'), (dict(kv_heads=0), 'heads'), (dict(kv_heads=3), 'heads'), (dict(kv_heads=8), 'heads'), (dict(head_dim=0), 'head_dim'),
       (dict(head_dim=12), 'head_dim'), (dict(head_dim=136), 'head_dim'), (dict(scale=0.0), 'scale'), (dict(scale=-1.0), 'scale'),
       (dict(scale=float('inf')), 'scale'), (dict(scale=float('nan')), 'scale'), (dict(dropout_p=1.0), 'dropout'), (dict(dropout_p=-0.5), 'dropout'),
       (dict(dropout_p=float('nan')), 'dropout'), (dict(S=0x7fffffff), '2^30'), (dict(L=0x7fffffff), '2^30'), (dict(B=0x7fffffff), 'one launch'),
       (dict(heads=1 << 20, kv_heads=1 << 20), '16 MB'), (dict(q=0), 'q must'), (dict(q=P + 8), 'q must'), (dict(q_rs=60), 'q must'), (dict(q_bs=1), 'q must'),
       (dict(q_rs=1 << 23), 'q must'), (dict(k=0), 'k and v'), (dict(v=P + 2), 'k and v'), (dict(k_rs=-32), 'k and v'), (dict(v_rs=4), 'k and v'),
       (dict(v_bs=12), 'k and v')]


@pytest.mark.parametrize('change,word', BAD, ids=str)
def test_attention_refuses(change, word):
    t = attention(**change)
    ref = ctypes.addressof(t)
    assert L.di_attention_fwd(ref, P, None, P, None) == -1 and word in said()
    assert L.di_attention_bwd(ref, P, P, P, 320, 64, P, P, 288, 32, P, 288, 32, P, None) == -1 and word in said()
    assert L.di_attention_fwd_workspace_floats(ref) == -1 and word in said()
    assert L.di_attention_bwd_workspace_floats(ref) == -1 and word in said()


def test_attention_without_an_argument_block():
    assert L.di_attention_fwd(None, P, None, P, None) == -1 and 'null' in said()
    assert L.di_attention_bwd(None, P, P, P, 320, 64, P, P, 288, 32, P, 288, 32, P, None) == -1 and 'null' in said()
    assert L.di_attention_fwd_workspace_floats(None) == -1
    assert L.di_attention_bwd_workspace_floats(None) == -1


@pytest.mark.parametrize('out', [None, P + 8])
def test_attention_outputs_of_the_forward(out):
    assert L.di_attention_fwd(ctypes.addressof(attention()), out, None, P, None) == -1 and 'output' in said()


GRAD = dict(out=P, lse=P, go=P, go_bs=320, go_rs=64, gq=P, gk=P, gk_bs=288, gk_rs=32, gv=P, gv_bs=288, gv_rs=32, ws=P)


@pytest.mark.parametrize('change,word', [(dict(out=None), 'grad_out'), (dict(lse=None), 'grad_out'), (dict(go=None), 'grad_out'), (dict(go=P + 4), 'grad_out'),
                                         (dict(go_rs=62), 'grad_out'), (dict(go_bs=3), 'grad_out'), (dict(gq=None), 'grad_out'), (dict(gq=P + 8), 'grad_out'),
                                         (dict(gk=None), 'grad_k'), (dict(gv=None), 'grad_k'), (dict(gk=P + 8), 'grad_k'), (dict(gv_rs=-32), 'grad_k'),
                                         (dict(gk_rs=0), 'overlap'), (dict(gk_rs=24), 'overlap'), (dict(gv_rs=16), 'overlap'), (dict(gk_bs=0), 'overlap'),
                                         (dict(gv_bs=16), 'overlap'), (dict(ws=None), 'workspace'), (dict(ws=P + 4), 'workspace')], ids=str)
def test_attention_outputs_of_the_backward(change, word):
    assert L.di_attention_bwd(ctypes.addressof(attention()), *{**GRAD, **change}.values(), None) == -1 and word in said()


def test_nothing_to_do_is_no_error():
    for t in (attention(B=0, q=0, k=0, v=0), attention(L=0, q=0)):
        assert L.di_attention_fwd(ctypes.addressof(t), None, None, None, None) == 0
    t = attention(B=0, q=0, k=0, v=0)
    assert L.di_attention_bwd(ctypes.addressof(t), *[None if v == P else v for v in GRAD.values()], None) == 0
    t = attention(L=0, S=0, q=0, k=0, v=0)
    assert L.di_attention_bwd(ctypes.addressof(t), *[None if v == P else v for v in GRAD.values()], None) == 0
    assert L.di_layernorm_fwd(None, 8, 0, None, 0, 0, None, None, 0, None, 0, None, None, None, 0, 8, 1e-5, None) == 0


F, H, X = _lib.DI_F32, _lib.DI_F16, _lib.DI_BF16
FWD = dict(x=P, xs=8, xt=F, res=P, rs=8, rt=F, w=P, b=P, wt=F, y=P, yt=F, total=None, mean=None, rstd=None, rows=3, C=8, eps=1e-5)


@pytest.mark.parametrize('change,word', [(dict(C=0), 'columns'), (dict(C=16385), 'columns'), (dict(rows=-1), 'columns'), (dict(xt=_lib.DI_F16_HL), 'dtype'),
                                         (dict(rt=9), 'dtype'), (dict(wt=-1), 'dtype'), (dict(yt=4), 'dtype'), (dict(xt=H, rt=X), 'bfloat16'),
                                         (dict(xt=H, rt=H, wt=X), 'bfloat16'), (dict(yt=H), '16-bit output'), (dict(xt=H, yt=H), '16-bit output'),
                                         (dict(mean=P), 'together'), (dict(rstd=P), 'together'), (dict(x=None), 'null'), (dict(w=None), 'null'),
                                         (dict(b=None), 'null'), (dict(y=None), 'null')], ids=str)
def test_layernorm_refuses(change, word):
    assert L.di_layernorm_fwd(*{**FWD, **change}.values(), None) == -1 and word in said()


BWD = dict(gy=P, gs=8, yt=F, gsum=None, ss=8, x=P, xs=8, xt=F, res=P, rs=8, rt=F, w=P, wt=F, mean=P, rstd=P, gx=P, gxt=F, gres=P, gw=P, gb=P, ws=P, rows=3, C=8)


@pytest.mark.parametrize('change,word', [(dict(C=0), 'columns'), (dict(C=16385), 'columns'), (dict(rows=-1), 'columns'), (dict(xt=_lib.DI_F16_HL), 'dtype'),
                                         (dict(gxt=9), 'dtype'), (dict(xt=H, rt=X), 'bfloat16'), (dict(gxt=H, wt=X), 'bfloat16'), (dict(yt=H), '16-bit output'),
                                         (dict(res=None), 'not there'), (dict(gw=None), 'null'), (dict(gb=None), 'null'), (dict(gy=None), 'null'),
                                         (dict(x=None), 'null'), (dict(w=None), 'null'), (dict(mean=None), 'null'), (dict(rstd=None), 'null'),
                                         (dict(gx=None), 'null'), (dict(ws=None), 'null')], ids=str)
def test_layernorm_backward_refuses(change, word):
    assert L.di_layernorm_bwd(*{**BWD, **change}.values(), None) == -1 and word in said()


def test_layernorm_workspace_refuses():
    for rows, C in ((-1, 8), (3, 0), (3, 16385)):
        assert L.di_layernorm_bwd_workspace_floats(rows, C) == -1


def test_tensors_of_the_host_are_refused():
    q, kv, w = torch.zeros(1, 2, 32), torch.zeros(1, 3, 32), torch.ones(32)
    stat = torch.zeros(2)
    for call in (lambda: ops.cross_attention(q, kv, kv, 2), lambda: ops.cross_attention_train_fwd(q, kv, kv, 2),
                 lambda: ops.cross_attention_train_bwd(q, kv, kv, q, q, torch.zeros(1, 2, 2), 2), lambda: ops.layernorm(q, w, w),
                 lambda: ops.layernorm_train_fwd(q, w, w), lambda: ops.layernorm_train_bwd(q, q, w, stat, stat)):
        with pytest.raises(_lib.HipLibraryError):
            call()
    assert not autograd.cross_attention_usable(q, kv, 2)


def test_the_argument_block_s_layout():
    """Three pointers and six strides, five mask words and strides, seven ints, two floats, four bytes of padding, the seed."""
    A = _lib.Attention
    assert (A.q_bs.offset, A.key_lengths.offset, A.B.offset, A.scale.offset, A.seed.offset, ctypes.sizeof(A)) == (24, 72, 120, 148, 160, 168)


LARGE = [(True, dict(B=3 << 20, L=1, S=1, heads=8, kv_heads=8)), (True, dict(B=1 << 22, L=600, S=9, heads=1, kv_heads=1, head_dim=128)),
         (False, dict(B=1 << 20, L=1, S=4000, heads=1, kv_heads=1)), (False, dict(B=1 << 22, L=65, S=9, heads=2, kv_heads=2, head_dim=128, dropout_p=0.5)),
         (False, dict(B=1 << 20, L=1000, S=600, heads=8, kv_heads=1))]     # the last: the join of gq over three key blocks


@pytest.mark.parametrize('forward,sizes', LARGE, ids=str)
def test_attention_of_more_workgroups_than_a_launch_has(forward, sizes):
    """2^24 - 1 workgroups of 256 threads are the most that one launch takes."""
    t = attention(q_bs=0, k_bs=0, v_bs=0, q_rs=1024, k_rs=1024, v_rs=1024, **sizes)
    ref = ctypes.addressof(t)
    if forward:
        assert L.di_attention_fwd(ref, P, None, P, None) == -1 and 'one launch' in said()
        assert L.di_attention_fwd_workspace_floats(ref) == -1 and 'one launch' in said()
    else:
        assert L.di_attention_bwd(ref, P, P, P, 0, 1024, P, P, 1 << 22, 1024, P, 1 << 22, 1024, P, None) == -1 and 'one launch' in said()
        assert L.di_attention_bwd_workspace_floats(ref) == -1 and 'one launch' in said()


# rows of 32 elements (64 bytes), 2 samples of 9
OVERLAPS = [dict(gk_bs=32, gv=P + 4096), dict(gk_bs=64, gk_rs=64, gv=P + 4096), dict(gk_bs=256, gv=P + 4096), dict(gk_bs=-256, gv=P + 8192), dict(gv_bs=256, gv=P + 4096),
            dict(gv=P), dict(gv=P + 32), dict(gv=P + 64), dict(gv=P + 512), dict(gv=P + 576 + 64), dict(gk_rs=48, gk_bs=432, gv_rs=48, gv_bs=432, gv=P + 48),
            dict(gk_rs=64, gk_bs=576, gv_rs=64, gv_bs=576, gv=P + 96), dict(gk_rs=64, gk_bs=576, gv_rs=32, gv_bs=576, gv=P + 64)]


@pytest.mark.parametrize('change', OVERLAPS, ids=str)
def test_key_gradients_that_overlap(change):
    """Rows of two samples, or of the two gradients, in one place: the last writer would win."""
    assert L.di_attention_bwd(ctypes.addressof(attention()), *{**GRAD, **change}.values(), None) == -1 and 'overlap' in said()


APART = [dict(gv=P + 1152), dict(gk=P + 1152), dict(gk_bs=-288, gv=P + 1152), dict(gk_rs=64, gk_bs=576, gv_rs=64, gv_bs=576, gv=P + 64),       # behind it; halves
         dict(gk_bs=32, gk_rs=64, gv_bs=32, gv_rs=64, gv=P + 4096), dict(gk_bs=64, gk_rs=128, gv_bs=64, gv_rs=128, gv=P + 64),                  # sequence first
         dict(gk_bs=576, gv_bs=576, gv=P + 576)]                                                                                                  # (B, 2, S, E)


@pytest.mark.parametrize('change', APART, ids=str)
def test_key_gradients_side_by_side(change):
    """What is refused, if anything, is not the layout (without a GPU: the launch)."""
    assert L.di_attention_bwd(ctypes.addressof(attention(B=0)), *{**GRAD, **change}.values(), None) == 0
    if torch.cuda.is_available():
        return                                                       # the pointers must not be followed
    assert L.di_attention_bwd(ctypes.addressof(attention()), *{**GRAD, **change}.values(), None) != -1 or 'overlap' not in said()


def test_seed_words():
    q = torch.zeros(1, 2, 16)
    assert ops._seed_word(q, 0.0, None) is None and ops._seed_word(q, 0.5, None) is None
    word = torch.zeros(1, dtype=torch.int64)
    assert ops._seed_word(q, 0.5, word) is word and ops._seed_word(q, 0.0, word) is None
    for bad in (word.int(), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64, device='meta')):
        with pytest.raises(ValueError):
            ops._seed_word(q, 0.5, bad)
    assert ops._seed_word(q, 0.5, False) is None
