"""torch.autograd bindings of the gather operators (training step).

Forward = the inference kernels; backward = the float32-atomic scatter kernels of csrc/backward.hip.  Only
feature maps receive gradients: sampling coordinates are functions of points, metas and detached box
predictions, exactly as in the reference (F.grid_sample's grid at encoder_utils.py:195,:297 is built from
data; the RoI boxes come from deep-copied, decoded predictions, decoder_utils.py:672-679)."""
import torch
from torch.amp import custom_bwd, custom_fwd
from torch.autograd import forward_ad

from . import ops

# Mixed precision (torch.autocast): the gather kernels take fp16 or float32 maps as they come; `custom_fwd` / `custom_bwd` make
# a Function's backward run under the autocast state of its forward (PixelLinear's GEMMs then run in the forward's dtype).
_fwd = custom_fwd(device_type='cuda')
_bwd = custom_bwd(device_type='cuda')

import os
OWN_WGRAD = os.environ.get('DI_OWN_WGRAD', '1') != '0'       # float32 1x1 weight gradients through csrc/wgrad.hip (A/B switch)


class BEVWarpGather(torch.autograd.Function):
    """warped = bilinear(bev, unproject(depth)) masked to pc_range  (encoder_utils.py:183-196)."""

    @staticmethod
    @_fwd
    def forward(ctx, bev, depth, img2lidar, aug_fwd, xs, ys, pc_range):
        ctx.save_for_backward(depth, img2lidar, aug_fwd, xs, ys, pc_range)
        ctx.bev_hw, ctx.bev_dtype = tuple(bev.shape[-2:]), bev.dtype
        return ops.bevwarp_gather(bev, depth, img2lidar, aug_fwd, xs, ys, pc_range)

    @staticmethod
    @_bwd
    def backward(ctx, grad_out):
        depth, img2lidar, aug_fwd, xs, ys, pc_range = ctx.saved_tensors
        g = ops.bevwarp_gather_bwd(grad_out, depth, img2lidar, aug_fwd, xs, ys, pc_range, ctx.bev_hw)
        return g.to(ctx.bev_dtype), None, None, None, None, None, None


class RoIAlign(torch.autograd.Function):
    """detectron2 ROIAlign(7x7, ratio 2, aligned) on channels-last maps, output (R,49,C)."""

    @staticmethod
    @_fwd
    def forward(ctx, feat, rois, spatial_scale):
        ctx.save_for_backward(rois)
        ctx.shape, ctx.dtype, ctx.scale = tuple(feat.shape), feat.dtype, float(spatial_scale)
        return ops.roi_align(feat, rois, spatial_scale)

    @staticmethod
    @_bwd
    def backward(ctx, grad_out):
        (rois,) = ctx.saved_tensors
        g = ops.roi_align_bwd(grad_out, rois, ctx.shape, ctx.scale)
        return g.to(ctx.dtype), None, None


class PixelLinear(torch.autograd.Function):
    """y = x @ W^T + b for x = the (pixels, C) view of a feature map (a 1x1 convolution), pixels >> C.

    The weight gradient  dW = dy^T @ x  reduces over 10^5 pixels into a 128 x 128 result: as ONE GEMM the library
    launches 16 workgroups (no split-K: 370 us on 134 400 pixels).  float32 with channel counts that are multiples of 128:
    the own kernel of csrc/wgrad.hip (float32 matrix cores over pixel slabs + a fixed-order sum, bias gradient included).
    Otherwise (fp16 under autocast, other widths) the pixels are cut into S slabs, the slabs are a BATCHED GEMM (S x 16
    workgroups) and the S partial results are summed."""

    @staticmethod
    @_fwd
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    def _slabs(M):
        for S in (128, 100, 96, 81, 75, 64, 60, 50, 48, 40, 36, 32, 25, 24, 20, 16, 12, 10, 8, 6, 5, 4, 3, 2):
            if M % S == 0 and M // S >= 512:
                return S
        return 1

    @staticmethod
    @_bwd
    def backward(ctx, gy):
        x, weight = ctx.saved_tensors
        gx = gw = gb = None
        gy = gy.contiguous()
        if gy.dtype != weight.dtype:                 # autocast: the forward's GEMM ran in fp16
            weight = weight.to(gy.dtype)
        if x.dtype != gy.dtype:
            x = x.to(gy.dtype)
        if ctx.needs_input_grad[0]:
            gx = gy @ weight
        want_b = ctx.has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1]:
            M, S = x.shape[0], PixelLinear._slabs(x.shape[0])
            xc = x.contiguous()
            if OWN_WGRAD and M >= 4096 and ops.wgrad_supported(xc, gy):
                # float32: own kernel on the float32 matrix cores (csrc/wgrad.hip), 418 -> ~40 us on the image maps
                gw, gb = ops.wgrad(xc, gy, bias=want_b)
                want_b = False
            elif S > 1:
                gw = torch.bmm(gy.view(S, M // S, -1).transpose(1, 2), xc.view(S, M // S, -1)).sum(0)
            else:
                gw = gy.t() @ x
        if want_b:
            gb = gy.sum(0)
        return gx, gw, gb


class WideLinear(torch.autograd.Function):
    """y = x @ W^T + b for a FEW rows and VERY MANY outputs (DynamicConv's parameter generator: 200 tokens x 128 -> 32 768,
    reference decoder_utils.py:584-600).  The input gradient  dx = dy @ W  reduces over the 32 768 outputs into a 200 x 128
    result: as one GEMM the library launches a handful of workgroups without split-K (94 us per call for 8 MB of weights);
    here the reduction is cut into S slabs, the slabs are a batched GEMM and the partial results are summed."""

    @staticmethod
    @_fwd
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @_bwd
    def backward(ctx, gy):
        x, weight = ctx.saved_tensors
        gx = gw = gb = None
        gy = gy.contiguous()
        if gy.dtype != weight.dtype:
            weight = weight.to(gy.dtype)
        if x.dtype != gy.dtype:
            x = x.to(gy.dtype)
        N, K = gy.shape
        if ctx.needs_input_grad[0]:
            S = next((s_ for s_ in (64, 32, 16, 8) if K % s_ == 0 and K // s_ >= 256), 1)
            if S > 1:
                gx = torch.bmm(gy.view(N, S, K // S).transpose(0, 1), weight.view(S, K // S, -1)).sum(0)
            else:
                gx = gy @ weight
        if ctx.needs_input_grad[1]:
            gw = gy.t() @ x
        if ctx.has_bias and ctx.needs_input_grad[2]:
            gb = gy.sum(0)
        return gx, gw, gb


class I2PAttention(torch.autograd.Function):
    """ctx[cell] = sum_j d_j softmax_j(<qfold[cell], s_j>) s_j over the pillar's valid image keys
    (encoder_utils.py:257-320 with the single-head attention folded, see MMRI_I2P), d_j the attention dropout factor.
    Returns (ctx, valid, mass): mass = sum_j d_j p_j, the kept probability mass (= valid without dropout) - the folded
    value bias enters the module's output scaled by it, and its gradient flows back into the scores."""

    @staticmethod
    @_fwd
    def forward(ctx, img, qfold, pillars, coors, num_points, proj, aug_rev, ori_hw, dropout_p, seed, keys=None):
        ctx.save_for_backward(img, qfold, pillars, coors, num_points, proj, aug_rev)
        ctx.ori_hw, ctx.dropout_p, ctx.seed = ori_hw, float(dropout_p), int(seed)
        out, valid, mass = ops.i2p_attention(img, qfold, pillars, coors, num_points, proj, aug_rev, ori_hw, dropout_p,
                                             seed, keys, with_mass=True)
        ctx.mark_non_differentiable(valid)
        return out, valid, mass

    @staticmethod
    @_bwd
    def backward(ctx, grad_ctx, _grad_valid, grad_mass):
        img, qfold, pillars, coors, num_points, proj, aug_rev = ctx.saved_tensors
        g_img, g_q = ops.i2p_attention_bwd(img, qfold, grad_ctx, pillars, coors, num_points, proj, aug_rev,
                                           ctx.ori_hw, ctx.dropout_p, ctx.seed, grad_mass=grad_mass)
        return g_img.to(img.dtype), g_q.to(qfold.dtype), None, None, None, None, None, None, None, None, None


def _formula_grads(formula, inputs, needs, grad_out):
    """Gradients of formula(*inputs) that can be differentiated again (a backward with create_graph): through torch's operations on views
    of the inputs, so that each gradient is its own input's share even where one input was computed from another."""
    with torch.enable_grad(), torch.autocast('cuda', enabled=False):
        views = [t.view_as(t) if need else t for t, need in zip(inputs, needs)]
        grads = iter(torch.autograd.grad(formula(*views), [t for t, need in zip(views, needs) if need], grad_out, create_graph=True, allow_unused=True))
    return [next(grads) if need else None for need in needs]


class AddLayerNorm(torch.autograd.Function):
    """y = LayerNorm(x + res) (csrc/layernorm.hip, layernorm_bwd.hip; res may be None), or (y, x + res) with `with_sum`: the post-norm
    and pre-norm steps of a training forward.  x and res are kept, not their sum; with_sum keeps the sum instead.  (Neither this Function nor
    CrossAttention calls anything that autocast changes: without custom_fwd / custom_bwd a forward and backward take 10 us of the host less.)"""

    @staticmethod
    def forward(ctx, x, res, weight, bias, eps, out_dtype, with_sum):
        y, total, mean, rstd = ops.layernorm_train_fwd(x, weight, bias, res, eps, with_sum, out_dtype)
        ctx.save_for_backward(x if total is None else total, res if total is None else None, weight, mean, rstd)
        ctx.types, ctx.eps = (x.dtype, None if res is None else res.dtype), eps
        ctx.set_materialize_grads(False)
        return (y, total) if with_sum else y

    @staticmethod
    def _formula_backward(ctx, gy, gsum):
        """`backward` for create_graph: through the formula (float32, as the kernels)."""
        x, res, weight, _, _ = ctx.saved_tensors
        xt, rt = ctx.types
        need = ctx.needs_input_grad
        both = rt is not None and res is None                      # x is the sum: its gradient is the residual's as well
        wants = [need[0] or (both and need[1]), res is not None and need[1], need[2]]
        gx = gres = gw = gb = None
        if gy is not None:
            def formula(x, res, weight):
                s = x.float() if res is None else x.float() + res.float()
                return torch.nn.functional.layer_norm(s, s.shape[-1:], weight.float(), None, ctx.eps)
            gx, gres, gw = _formula_grads(formula, (x, res, weight), wants, gy.float())
            gb = gy.float().reshape(-1, gy.shape[-1]).sum(0).to(weight.dtype) if need[3] else None
        if gsum is not None:
            gx = gsum if gx is None else gx + gsum
        if both and need[1] and gx is not None:
            gres = gx.to(rt)
        return gx.to(xt) if need[0] and gx is not None else None, gres, gw, gb, None, None, None

    @staticmethod
    def backward(ctx, gy, gsum=None):
        if torch.is_grad_enabled():
            return AddLayerNorm._formula_backward(ctx, gy, gsum)
        x, res, weight, mean, rstd = ctx.saved_tensors
        xt, rt = ctx.types
        need = ctx.needs_input_grad
        if gy is None:                                   # only the sum went on
            gx, gw, gb = gsum, None, None
        else:
            gx, gres, gw, gb = ops.layernorm_train_bwd(gy, x, weight, mean, rstd, res=res, grad_sum=gsum)
        if gx is None:
            return (None,) * 7
        if gy is None or res is None:
            gres = None if rt is None else gx.to(rt)
        return (gx.to(xt) if need[0] else None, gres if need[1] else None, gw if need[2] else None, gb if need[3] else None,
                None, None, None)


class CrossAttention(torch.autograd.Function):
    """softmax(scale q k^T) v per head (csrc/attention*.hip); k alone, (B, S, 2 Ek), is [K | V] of one projection and receives one
    packed gradient.  Gradients: q, k, v; lengths and masks have none."""

    @staticmethod
    def forward(ctx, q, k, v, num_heads, scale, key_lengths, key_mask, allowed, dropout_p, seed, seed_word=None):
        Ek = k.shape[-1] // 2
        ks, vs = (k[..., :Ek], k[..., Ek:]) if v is None else (k, v)
        seed_word = ops._seed_word(q, dropout_p, seed_word)        # the backward's as well, whatever is registered by then
        out, lse = ops.cross_attention_train_fwd(q, ks, vs, num_heads, scale, key_lengths, key_mask, allowed, dropout_p, seed,
                                                 False if seed_word is None else seed_word)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths, key_mask, allowed, seed_word)
        ctx.args = (num_heads, scale, dropout_p, seed)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        q, k, v, out, lse, key_lengths, key_mask, allowed, seed_word = ctx.saved_tensors
        num_heads, scale, dropout_p, seed = ctx.args
        if torch.is_grad_enabled():                                # create_graph: through the formula
            def formula(q, k, v):
                return attention_formula(q, k, v, num_heads, scale, key_lengths, key_mask, allowed, dropout_p, seed, seed_word)
            need = [t is not None and n for t, n in zip((q, k, v), ctx.needs_input_grad)]
            return tuple(_formula_grads(formula, (q, k, v), need, grad_out)) + (None,) * 8
        Ek = k.shape[-1] // 2
        packed = None if v is not None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        ks, vs = (k[..., :Ek], k[..., Ek:]) if v is None else (k, v)
        gq, gk, gv = ops.cross_attention_train_bwd(q, ks, vs, out, grad_out, lse, num_heads, scale, key_lengths, key_mask, allowed,
                                                   dropout_p, seed,
                                                   grads_kv=None if packed is None else (packed[..., :Ek], packed[..., Ek:]),
                                                   seed_word=False if seed_word is None else seed_word)
        return (gq, gk if packed is None else packed, gv if packed is None else None) + (None,) * 8


def _dropout_factors(B, H, L, S, p, seed, seed_word, device):
    """(B, H, L, S) float32: 0 or the reciprocal of the kept share - the decisions of csrc/attention.h's hash, in torch's operations."""
    M = 0xFFFFFFFF

    def mix(x):
        x = ((x ^ (x >> 16)) * 0x7FEB352D) & M
        x = ((x ^ (x >> 15)) * 0x846CA68B) & M
        return x ^ (x >> 16)
    seed = seed & 0xFFFFFFFFFFFFFFFF
    seed = torch.full((1,), seed - (1 << 64) if seed >> 63 else seed, dtype=torch.int64, device=device)
    if seed_word is not None:
        seed = seed + seed_word
    row = torch.arange(B * H * L, device=device)
    h = mix(mix(((seed & M) + (row & M) * 0x9E3779B9) & M) ^ ((seed >> 32) & M) ^ (((row >> 32) * 0x85EBCA6B) & M))[:, None]
    x = mix(h ^ (torch.arange((S + 3) // 4, device=device) * 0xC2B2AE35 & M))
    y = mix((x + 0x68BC21EB) & M)
    numbers = torch.stack((x & 0xFFFF, x >> 16, y & 0xFFFF, y >> 16), -1).view(B, H, L, -1)[..., :S]
    drop = min(int(p * 65536 + 0.5), 65535)
    return (numbers >= drop).float() * (65536 / (65536 - drop))


def attention_formula(q, k, v, num_heads, scale=None, key_lengths=None, key_mask=None, allowed=None, dropout_p=0.0, seed=0, seed_word=None):
    """What `ops.cross_attention_train_fwd` computes, in torch's operations (float32, scores materialised) and differentiable as often as
    those are; v None: k is [K | V]."""
    if v is None:
        k, v = k.chunk(2, -1)
    (B, L, E), S = q.shape, k.shape[1]
    D = E // num_heads
    Hk = k.shape[-1] // D
    G = num_heads // Hk
    keep = torch.ones((B, 1, S), dtype=torch.bool, device=q.device)
    if key_lengths is not None:
        keep = keep & (torch.arange(S, device=q.device) < key_lengths[:, None])[:, None]
    if key_mask is not None:
        keep = keep & (key_mask != 0)[:, None]
    zero = q.new_zeros((), dtype=torch.float32)
    kh, vh = (torch.where(keep.view(B, 1, S, 1), t.float().view(B, S, Hk, D).transpose(1, 2), zero) for t in (k, v))       # whatever lies there
    if allowed is not None:
        keep = keep & (allowed != 0)
    some = keep.any(-1).view(B, 1, 1, -1, 1)                           # rows with a key at all: the others are zeros, whatever they hold
    qh = torch.where(some, q.float().view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4), zero).reshape(B, Hk, G * L, D)
    s = torch.matmul(qh, kh.transpose(-1, -2).contiguous()).view(B, Hk, G, L, S) * (D ** -0.5 if scale is None else scale)
    a = torch.softmax(s.masked_fill(~(keep[:, None, None] | ~some), float('-inf')), -1)
    if dropout_p > 0:
        a = a * _dropout_factors(B, num_heads, L, S, dropout_p, seed, seed_word, q.device).view(B, Hk, G, L, S)
    o = torch.matmul(a.view(B, Hk, G * L, S), vh).view(B, Hk, G, L, D)
    return torch.where(some, o, zero).permute(0, 3, 1, 2, 4).reshape(B, L, E).to(q.dtype)


def _dropout_seed(like):
    """(seed, device word or None) of one call's dropout mask.  From the CUDA generator of `like`'s device, whose state a saved and restored step
    repeats: outside a capture its seed and offset, which moves on (mixed by splitmix64: Steele, Lea and Flood, 2014); inside one a word drawn
    there, so that every replay draws its own.  Where a word is registered (`ops.set_i2p_seed_tensor`), that one with a seed of torch's CPU
    generator."""
    word = ops._I2P_SEED_REF[0]
    if word is not None:
        return int(torch.randint(0, 2 ** 62, (1,)).item()), word
    if ops._on_device(like, torch.cuda.is_current_stream_capturing):
        return 0, torch.randint(0, 2 ** 62, (1,), dtype=torch.int64, device=like.device)
    gen = torch.cuda.default_generators[like.get_device()]
    at = gen.get_offset()
    gen.set_offset(at + 4)                               # philox: four numbers a step
    z = (gen.initial_seed() + (at // 4 + 1) * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & 0xFFFFFFFFFFFFFFFF
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & 0xFFFFFFFFFFFFFFFF
    return z ^ (z >> 31), None


def transformed(*tensors):
    """Whether torch.func's transforms or forward-mode differentiation act on a call: they know torch's own operations only."""
    if torch._C._are_functorch_transforms_active():
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def cross_attention_usable(q, k, num_heads, v=None, dropout_p=0.0):
    """Whether `cross_attention` takes these projections: on the GPU, one of float32 / float16 / bfloat16, a head dim of 8 .. 128 in
    steps of 8, weights that are not all dropped, outside of torch's transforms."""
    if transformed(q, k, v) or not dropout_p < 1:
        return False
    D = q.shape[-1] // num_heads
    return q.is_cuda and q.dtype == k.dtype and q.dtype in (torch.float32, torch.float16, torch.bfloat16) and D % 8 == 0 and 8 <= D <= 128


def cross_attention(q, k, v, num_heads, scale=None, key_lengths=None, key_mask=None, allowed=None, dropout_p=0.0):
    """`ops.cross_attention`, differentiable where a gradient is asked for; v None: k is [K | V] of one projection.  dropout_p: of the
    attention weights, a fresh mask in every call and in every replay of a captured one (`_dropout_seed`)."""
    ops._same_device(q)
    if dropout_p > 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v))):
        seed, word = _dropout_seed(q) if dropout_p > 0 else (0, None)
        return CrossAttention.apply(q, k, v, num_heads, scale, key_lengths, key_mask, allowed, dropout_p, seed, word)
    if v is None:
        k, v = k.chunk(2, -1)
    return ops.cross_attention(q, k, v, num_heads, scale, key_lengths, key_mask, allowed)


# ---------------------------------------------------------------------------------- DeepInteraction++ samplers
class MSDeformAttn(torch.autograd.Function):
    """mmcv MultiScaleDeformableAttention core on the packed [offsets | logits] projection (csrc/plusplus.hip /
    plusplus_bwd.hip).  Gradients: value, packed projection.  Reference points are constants."""

    @staticmethod
    @_fwd
    def forward(ctx, value, proj, ref, level_hw, n_points):
        L = len(level_hw)
        n_off = 8 * L * n_points * 2
        ctx.save_for_backward(value, proj, ref)
        ctx.level_hw, ctx.n_points, ctx.n_off = list(level_hw), n_points, n_off
        return ops.ms_deform_attn(value, proj[..., :n_off], proj[..., n_off:], ref, level_hw, n_points)

    @staticmethod
    @_bwd
    def backward(ctx, grad_out):
        value, proj, ref = ctx.saved_tensors
        n_off = ctx.n_off
        gv, gp = ops.ms_deform_attn_bwd(value, proj[..., :n_off], proj[..., n_off:], ref, ctx.level_hw, grad_out,
                                        ctx.n_points)
        return gv.to(value.dtype), gp, None, None, None


class GridGather(torch.autograd.Function):
    """out[g, n] = bilinear(feat[g // per_feat], grid[g, n]) + add[n]; gradient w.r.t. feat only (the grid is
    geometry, the additive term a constant encoding)."""

    @staticmethod
    @_fwd
    def forward(ctx, feat, grid, add, grids_per_feat):
        ctx.save_for_backward(grid)
        ctx.shape, ctx.dtype, ctx.per = tuple(feat.shape), feat.dtype, grids_per_feat
        return ops.grid_gather(feat, grid, add, grids_per_feat)

    @staticmethod
    @_bwd
    def backward(ctx, grad_out):
        (grid,) = ctx.saved_tensors
        return ops.grid_gather_bwd(grid, grad_out, ctx.shape, ctx.per).to(ctx.dtype), None, None, None


class PolarBEVSample(torch.autograd.Function):
    """out = mean over seeing cameras of bilinear(polar[cam], loc(cell, cam)) + bev  (fusion_transformerv4.py:581-640)."""

    @staticmethod
    @_fwd
    def forward(ctx, polar, bev, proj, aug_rev, cam_xy, params):
        ctx.save_for_backward(proj, aug_rev, cam_xy, params)
        ctx.shape, ctx.dtype = tuple(polar.shape), polar.dtype
        return ops.polar_bev_sample(polar, bev, proj, aug_rev, cam_xy, params)

    @staticmethod
    @_bwd
    def backward(ctx, grad_out):
        proj, aug_rev, cam_xy, params = ctx.saved_tensors
        gp = ops.polar_bev_sample_bwd(grad_out, proj, aug_rev, cam_xy, params, ctx.shape)
        return gp.to(ctx.dtype), grad_out, None, None, None, None
