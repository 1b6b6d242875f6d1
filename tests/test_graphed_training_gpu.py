"""The captured training step (graphed.GraphedTrainingModule): every replay's outputs and gradients against the same module run eagerly, with
other work and synchronisations between the replays; memset nodes replaced by kernels."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

from deepinteraction_amd import _lib, graphed, ops, synth, train_step

# (query, key) grids, rows of a wide sum: sizes at which torch's sums run over many workgroups and clear counters first
SUMS = [(32400, 128), (134400, 64), (5000, 7)]


def captured(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        out = fn()
    return g, out


def memsets(g):
    return int(_lib.lib().di_graph_fill_by_kernels(int(g.raw_cuda_graph()), 0))


def test_library_sums_in_a_graph():
    xs = [torch.empty(s, device='cuda') for s in SUMS]
    g, outs = captured(lambda: [x.sum(0) for x in xs])
    assert memsets(g) > 0                                            # otherwise this test shows nothing
    nodes = _lib.lib().di_graph_node_count(int(g.raw_cuda_graph()))
    graphed._without_memsets(g)
    assert memsets(g) == 0 and _lib.lib().di_graph_node_count(int(g.raw_cuda_graph())) == nodes
    for n in range(5):
        for x in xs:
            x.normal_()
        want = [x.sum(0) for x in xs]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), n


def test_memset_nodes_of_every_kind():
    """Bytes, 16- and 32-bit values, rows apart, odd addresses and sizes; what lies beside them stays."""
    hip = ctypes.CDLL('libamdhip64.so')
    buf, want = torch.empty(1 << 16, dtype=torch.uint8, device='cuda'), torch.full((1 << 16,), 7, dtype=torch.uint8)
    at, p = buf.data_ptr(), ctypes.c_void_p

    def fn():
        s = p(torch.cuda.current_stream().cuda_stream)
        rc = [hip.hipMemsetAsync(p(at), 3, ctypes.c_size_t(16), s), hip.hipMemsetAsync(p(at + 33), 0x85, ctypes.c_size_t(1), s),
              hip.hipMemsetAsync(p(at + 101), 0xff, ctypes.c_size_t(4099), s), hip.hipMemsetD16Async(p(at + 8194), ctypes.c_ushort(0x1234), ctypes.c_size_t(51), s),
              hip.hipMemsetD32Async(p(at + 12288), 0x01020304, ctypes.c_size_t(1000), s),
              hip.hipMemset2DAsync(p(at + 20000), ctypes.c_size_t(128), 9, ctypes.c_size_t(30), ctypes.c_size_t(17), s),
              hip.hipMemset2DAsync(p(at + 30001), ctypes.c_size_t(64), 5, ctypes.c_size_t(64), ctypes.c_size_t(3), s)]
        assert rc == [0] * 7
    want[:16], want[33], want[101:101 + 4099] = 3, 0x85, 0xff
    want[8194:8194 + 102] = torch.tensor([0x34, 0x12], dtype=torch.uint8).repeat(51)
    want[12288:12288 + 4000] = torch.tensor([4, 3, 2, 1], dtype=torch.uint8).repeat(1000)
    for row in range(17):
        want[20000 + 128 * row:20030 + 128 * row] = 9
    want[30001:30001 + 192] = 5
    g, _ = captured(fn)
    assert memsets(g) == 7
    graphed._without_memsets(g)
    assert memsets(g) == 0
    for n in range(3):
        buf.fill_(7)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf.cpu(), want), n


def test_a_graph_that_is_none_is_refused():
    assert _lib.lib().di_graph_fill_by_kernels(None, 1) == -2


def no_dropout(*modules):
    for root in modules:
        for m in root.modules():
            if isinstance(m, torch.nn.Dropout):
                m.p = 0.0
            elif isinstance(getattr(m, 'dropout', None), float):
                m.dropout = 0.0


@pytest.mark.parametrize('amp', [False, True])
def test_every_replay_s_gradients_of_the_hot_path(amp):
    """The captured forward and backward of the hot path, replayed six times - one of them with a huge gradient, whose infinities must not
    stay - against the same module run eagerly.

    Bounds: outputs and gradients of two eager passes differ by the order of the scatter kernels' float32 atomics and by the ReLU gates that
    those roundings flip; as in `test_training_step_gradients_match_oracle` no element is off by more than 5 % of its tensor's largest (a
    sum that was not cleared is off by its whole size).  Exact zeros (a bias in front of a BatchNorm) are what is left of summands of up to
    some tens: a hundred roundings of 2^-24, or under autocast of 2^-11 (of values that add up in float32), of 16."""
    torch.backends.cudnn.deterministic = True
    tr = train_step.GraphedTrainer(synth.SHAPE_TINY, 24, torch.device('cuda'), 1, pool=1, amp=amp, prepare_model=no_dropout)
    tr.h.load(tr.records[0])
    named = [(n, p) for m in (tr.enc, tr.dec) for n, p in m.named_parameters()]
    weights, gen = [], torch.Generator().manual_seed(3)
    zero = 100 * 16 * 2.0 ** -24 if not amp else 16 * 2.0 ** -11 * 4

    def step(run, scale=1.0):
        for _, p in named:
            p.grad = None
        outs = run(tr.h.img_feats, tr.h.pts_feats)
        if not weights:
            weights.extend(torch.randn(o.shape, generator=gen).cuda() for o in outs)
        sum((o * w).sum() * scale for o, w in zip(outs, weights) if o.requires_grad).backward()
        torch.cuda.synchronize()
        return [o.detach().clone() for o in outs], {n: p.grad.detach().float().clone() for n, p in named if p.grad is not None}
    outs, grads = step(tr.module)
    assert len(grads) > 380 and all(torch.isfinite(g).all() for g in grads.values())
    for n in range(6):
        if n == 3:
            step(tr.graphed, 2.0 ** 60)
        got, g = step(tr.graphed)
        torch.randn(1 << 20, device='cuda').sum()
        for a, b in zip(outs, got):
            assert float((a - b).abs().max()) <= 5e-2 * float(a.abs().max()) + zero, n
        assert set(g) == set(grads)
        bad = [(k, float((g[k] - r).abs().max()), float(r.abs().max())) for k, r in grads.items()
               if not float((g[k] - r).abs().max()) <= 5e-2 * float(r.abs().max()) + zero]
        assert not bad, (n, len(bad), bad[:5])


def test_the_inference_captures_hold_no_memset():
    from deepinteraction_amd import harness
    enc, dec = harness.build_models(synth.SHAPE_TINY, 24, torch.float16, 'cuda')
    d = harness.to_device(synth.make_inputs(1, synth.SHAPE_TINY, seed=3), 'cuda', torch.float16)
    h = graphed.GraphedHotPath(enc, dec, d)
    probe = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.no_grad(), torch.cuda.graph(probe):
        h._forward()
    assert memsets(probe) == 0


def test_a_capture_with_the_voxeliser_is_replayed_without_memsets(monkeypatch):
    """The capture that starts from the points holds a memset node of a library call: what is replayed does not."""
    from deepinteraction_amd import harness
    from deepinteraction_amd.mmdet3d_plugin import PointGlue
    counted, real = [], graphed._without_memsets

    def count(graph):
        counted.append(memsets(graph))
        real(graph)
        counted.append(memsets(graph))
        return graph
    monkeypatch.setattr(graphed, '_without_memsets', count)
    shape = synth.SHAPE_R
    (Hb, Wb), rng = shape['bev_hw'], list(synth.PC_RANGE)
    glue = PointGlue(dict(max_num_points=20, max_voxels=(30000, 60000), point_cloud_range=rng,
                          voxel_size=[(rng[3] - rng[0]) / Wb, (rng[4] - rng[1]) / Hb, rng[5] - rng[2]])).eval()
    enc, dec = harness.build_models(shape, 200, torch.float16, 'cuda')
    d = harness.to_device(synth.make_inputs(1, shape, seed=3), 'cuda', torch.float16)
    with torch.no_grad():
        g = graphed.GraphedHotPath(enc, dec, d, glue=glue)
        assert len(counted) == 2 and counted[0] > 0 and counted[1] == 0
        first = {k: v.clone() for k, v in g()[0][0].items()}
        for _ in range(3):
            torch.randn(1 << 22, device='cuda').sum()
            out = g()[0][0]
            torch.cuda.synchronize()
            assert all(torch.equal(out[k], v) for k, v in first.items())
