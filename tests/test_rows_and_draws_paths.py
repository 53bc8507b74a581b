"""The paths that use rows in 8 or 4 bits and draws from scores: the exchange with quantised records (CPU: gloo, two
processes, the codec restated by the oracle; GPU: the kernels, two clouds in two threads), checkpoints, pixel draws of the
frame loops, and all of them after one another as a mapped frame uses them."""
import os
import socket
import threading

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from oracle import rows_oracle as RO
from tests.helpers import base_cfg, load_decoders

gpu = pytest.mark.gpu
FORMATS = ["int8", "e4m3", "int4"]


def _stands_for(pair, fmt):
    """What a pair of feature rows [n, 2, 32] is worth after the wire."""
    if pair.shape[0] == 0:
        return pair
    return torch.from_numpy(RO.values(*RO.quantize(pair.numpy(), fmt, 32)))


class _HostWire:
    """point_slam_amd.dist._RowWire with the oracle for a codec: host tensors have no kernels."""

    def __init__(self, fmt):
        from point_slam_amd import row_store
        self.fmt = fmt
        self.codes, self.scales = row_store.record_floats(2, 32, fmt)
        self.floats = self.codes + self.scales

    def put(self, rec, col, pair):
        if pair.shape[0] == 0:
            return
        q, s = RO.quantize(pair.numpy(), self.fmt, 32)
        q = torch.from_numpy(q).reshape(-1, 64)
        if self.fmt == "e4m3":
            b = q.to(torch.float8_e4m3fn).view(torch.uint8)
        elif self.fmt == "int8":
            b = q.to(torch.int8).view(torch.uint8)
        else:
            i = q.to(torch.int32) & 15
            b = (i[:, 0::2] | (i[:, 1::2] << 4)).to(torch.uint8)
        rec[:, col:col + self.codes] = b.contiguous().view(torch.float32)
        rec[:, col + self.codes:col + self.floats] = torch.from_numpy(s).reshape(-1, 2)

    def get(self, rec, col):
        b = rec[:, col:col + self.codes].contiguous().view(torch.uint8)
        if self.fmt == "e4m3":
            q = b.view(torch.float8_e4m3fn).float()
        elif self.fmt == "int8":
            q = b.view(torch.int8).float()
        else:
            q = torch.stack([b & 15, b >> 4], -1).flatten(-2).to(torch.int8)
            q = torch.where(q > 7, q - 16, q).float()
        return q.reshape(-1, 2, 32) * rec[:, col + self.codes:col + self.floats].reshape(-1, 2, 1)


def _gloo_worker(rank, world, port, q, fmt):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from point_slam_amd import dist as PD
    from tests.test_dist_gloo import FakeCloud, _triplets
    PD._RowWire = _HostWire
    g = torch.Generator().manual_seed(100)
    base, bg, bc = torch.rand(10, 3, generator=g) + 5.0, torch.randn(10, 32, generator=g), torch.randn(10, 32, generator=g)
    cloud = FakeCloud(base, bg.clone(), bc.clone())
    sync = PD.FrameParallelSync(cloud, None, wire=fmt)
    gr = torch.Generator().manual_seed(rank + 1)
    c0 = torch.tensor([[1.0, 1.0, 1.0]])
    new = _triplets(c0 if rank == 0 else torch.cat([c0 + 0.01, torch.tensor([[2.0, 2.0, 2.0]])]))
    n = new.shape[0]
    mine = torch.randn(n, 2, 32, generator=gr)
    sync.note_rows(cloud, torch.tensor([0, 1, 5]) if rank == 0 else torch.tensor([1, 2]))
    change = torch.randn(10, 2, 32, generator=gr) * 0.1
    rows = [0, 1] if rank == 0 else [1, 2]
    before = torch.stack([bg, bc], 1)
    for r in rows:
        cloud.geo[r] += change[r, 0]; cloud.col[r] += change[r, 1]
    moved = torch.stack([cloud.geo[:10], cloud.col[:10]], 1) - before
    cloud.append_points(new, mine[:, 0], mine[:, 1])
    counts = sync.exchange(cloud)
    q.put(tuple(x.numpy() if torch.is_tensor(x) else x for x in
                (rank, counts, cloud.pos, torch.stack([cloud.geo, cloud.col], 1), cloud.rad, mine, moved, before)))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("fmt", FORMATS)
def test_exchange_with_quantised_records_world2(fmt):
    s = socket.socket(); s.bind(("127.0.0.1", 0)); port = s.getsockname()[1]; s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_gloo_worker, args=(r, 2, port, q, fmt)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=120) for _ in range(2)], key=lambda x: x[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    _check_exchange(res, fmt)


def _check_exchange(res, fmt):
    (_, c0, pos0, f0, rad0, m0, d0, before), (_, c1, pos1, f1, rad1, m1, d1, _) = [[torch.from_numpy(x) if isinstance(x, np.ndarray) else x for x in r] for r in res]
    assert c0 == c1 == [3, 6]
    assert torch.equal(pos0, pos1) and torch.equal(f0, f1) and torch.equal(rad0, rad1)        # identical replicas
    nb = before.shape[0]
    assert pos0.shape[0] == nb + 6                                                             # rank 1's first location is a duplicate
    # new points: what the codes stand for, on the rank that made them too; position and radius as they were
    assert torch.equal(f0[nb:nb + 3], _stands_for(m0, fmt)) and torch.equal(f0[nb + 3:], _stands_for(m1[3:], fmt))
    assert (rad0[nb:] == 0.04).all()
    # touched rows: snapshot + mean of the changes as sent; the others untouched
    q0, q1 = _stands_for(d0, fmt), _stands_for(d1, fmt)
    want = before.clone()
    want[0] += q0[0]; want[1] += (q0[1] + q1[1]) / 2; want[2] += q1[2]
    assert torch.allclose(f0[:nb], want, rtol=0, atol=4 * 2.0 ** -24 * float(want.abs().max()))      # three fp32 additions, in either order
    assert torch.equal(f0[3:nb], before[3:])


def test_wire_and_record_refusals():
    from point_slam_amd import dist as PD, row_store
    with pytest.raises(ValueError):
        PD._RowWire("fp4")
    assert PD._RowWire(None).floats == 64 and PD._RowWire("int8").floats == 18 and PD._RowWire("int4").floats == 10
    v = torch.zeros(3, 2, 32)
    for rec, cc, sc in ((torch.zeros(3, 20).double(), 2, 18), (torch.zeros(2, 20), 2, 18), (torch.zeros(3, 40)[:, ::2], 2, 18),
                        (torch.zeros(3, 20), 4, 18), (torch.zeros(3, 20), 2, 17), (torch.zeros(3, 20), -1, 18), (torch.zeros(3, 19), 2, 18)):
        with pytest.raises(ValueError):
            row_store.write_records(rec, v, "int8", cc, sc)
    with pytest.raises(ValueError):
        row_store.record_floats(1, 3, "int8")


def test_score_sampling_is_refused_where_the_loop_cannot_take_it():
    from point_slam_amd.slam import HipSLAM
    cfg = base_cfg()
    cfg["mapping"]["score_sampling"] = {"temperature": 0.7}
    with pytest.raises(NotImplementedError):
        HipSLAM(cfg, dict(H=120, W=160, fx=100.0, fy=100.0, cx=80.0, cy=60.0), engine="dropin")


# ------------------------------------------------------------------------------------------------ GPU
def _cloud(cfg, n=4000, seed=3, max_points=50000):
    from point_slam_amd import synthetic as syn
    from point_slam_amd.neural_point import HipNeuralPointCloud
    cfg = dict(cfg, mapping=dict(cfg["mapping"], device="cuda:0"))
    npc = HipNeuralPointCloud(cfg, max_points=max_points, device="cuda:0")
    base = syn.seed_cloud(syn.intrinsics(320, 240), n, n_views=4, seed=seed)
    g = torch.Generator().manual_seed(9)
    npc.set_points(base.cuda(), (torch.randn(base.shape[0], 32, generator=g) * 0.1).cuda(), (torch.randn(base.shape[0], 32, generator=g) * 0.1).cuda())
    return npc


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_records_match_the_oracle(fmt):
    from point_slam_amd import row_store
    v = torch.randn(777, 2, 32) * 0.1
    cw, sw = row_store.record_floats(2, 32, fmt)
    for code_col, width in ((4, 4 + cw + sw), (1, 1 + cw + sw), (0, cw + sw), (3, 9 + cw + sw)):
        rec = torch.full((777, width), 7.0, device="cuda")
        row_store.write_records(rec, v.cuda(), fmt, code_col, code_col + cw)
        host = rec.cpu()
        want = torch.zeros(777, width)
        w = _HostWire(fmt)
        w.put(want, code_col, v)
        span = slice(code_col, code_col + w.floats)
        assert torch.equal(host[:, span].contiguous().view(torch.int32), want[:, span].contiguous().view(torch.int32))
        keep = torch.ones(width, dtype=torch.bool); keep[span] = False
        assert (host[:, keep] == 7.0).all()
        assert torch.equal(row_store.read_records(rec, 2, 32, fmt, code_col, code_col + cw).cpu(), _stands_for(v, fmt))


class _ThreadTransport:
    """all-gather-v between two threads of one process."""

    def __init__(self, rank, box, barrier):
        self.rank, self.box, self.barrier = rank, box, barrier

    def allgather_v(self, rec):
        torch.cuda.synchronize()
        self.box[self.rank] = rec.clone()
        torch.cuda.synchronize()
        self.barrier.wait(60)
        out, counts = torch.cat([self.box[0], self.box[1]]), [self.box[0].shape[0], self.box[1].shape[0]]
        torch.cuda.synchronize()
        self.barrier.wait(60)
        return out, counts


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_exchange_with_quantised_records_on_the_real_cloud(fmt, monkeypatch):
    from point_slam_amd import dist as PD
    from tests.test_dist_gloo import _triplets
    me = threading.local()
    monkeypatch.setattr(PD.dist, "get_rank", lambda group=None: me.rank)
    monkeypatch.setattr(PD, "make_transport", lambda npc, group=None, kind=None: None)
    box, barrier, res, errors = [None, None], threading.Barrier(2), [None, None], []

    def work(rank):
        try:
            me.rank = rank
            npc = clouds[rank]
            nb = npc.pts_num()
            sync = PD.FrameParallelSync(npc, None, wire=fmt)
            sync.transport = _ThreadTransport(rank, box, barrier)
            before = torch.stack([npc.get_geo_feats(), npc.get_col_feats()], 1).clone()
            gr = torch.Generator().manual_seed(rank + 1)
            c0 = torch.tensor([[30.0, 1.0, 1.0]])
            new = _triplets(c0 if rank == 0 else torch.cat([c0 + 0.01, torch.tensor([[40.0, 2.0, 2.0]])]))
            mine, change = torch.randn(new.shape[0], 2, 32, generator=gr), torch.randn(3, 2, 32, generator=gr) * 0.1
            sync.note_rows(npc, torch.tensor([0, 1, 5] if rank == 0 else [1, 2], device="cuda"))
            for r in ([0, 1] if rank == 0 else [1, 2]):
                npc.get_geo_feats()[r] += change[r, 0].cuda(); npc.get_col_feats()[r] += change[r, 1].cuda()
            moved = torch.stack([npc.get_geo_feats(), npc.get_col_feats()], 1) - before
            npc.append_points(new.cuda(), mine[:, 0].cuda(), mine[:, 1].cuda(), radius=torch.full((new.shape[0],), 0.04, device="cuda"))
            counts = sync.exchange(npc)
            torch.cuda.synchronize()
            res[rank] = (rank, counts, npc.cloud_pos(), torch.stack([npc.get_geo_feats(), npc.get_col_feats()], 1).cpu(),
                         torch.cat([torch.zeros(nb), npc.point_radius(nb).cpu()]), mine, moved.cpu(), before.cpu())
        except Exception as e:
            errors.append(e)
            barrier.abort()

    clouds = [_cloud(base_cfg()) for _ in range(2)]
    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors, errors
    _check_exchange(res, fmt)


def _slam(cfg, n=12000):
    from point_slam_amd import synthetic as syn
    from point_slam_amd.decoders import PointDecoders
    from point_slam_amd.slam import Frame, HipSLAM
    cam = syn.intrinsics(320, 240)
    s = HipSLAM(cfg, cam, max_points=200000, decoders=PointDecoders(cfg).load_reference_state(load_decoders("replica")))
    s.seed_points(syn.seed_cloud(cam, n, n_views=4, seed=3))
    frames = []
    for k, t in enumerate((0.0, 4.0, 8.0)):
        c2w = syn.pose(t, "cuda:0")
        depth, color = syn.render_frame(cam, c2w)
        depth = depth.clone(); depth[100:120, 50:90] = 0.0                 # a sensor hole
        r_add, r_query = syn.dynamic_radii(color, cfg)
        frames.append(Frame(k, depth, color, r_add, r_query, c2w=c2w))
    return cam, s, frames


@gpu
def test_checkpoint_with_quantised_rows(tmp_path):
    from point_slam_amd import checkpoint as CK
    cam, s, _ = _slam(base_cfg())
    geo, col = s.npc.get_geo_feats().clone(), s.npc.get_col_feats().clone()
    sizes = {}
    for fmt in [None] + FORMATS:
        path = str(tmp_path / f"{fmt}.tar")
        s.save_checkpoint(path, idx=3, positions_as_list=False, feature_format=fmt)
        sizes[fmt] = os.path.getsize(path)
        ck = torch.load(path, map_location="cuda:0", weights_only=True)
        npc = _cloud(base_cfg(), n=100)
        assert CK.load_neural_point_cloud(npc, ck) == s.npc.pts_num()
        pair = torch.stack([geo, col], 1).cpu()
        want = pair if fmt is None else _stands_for(pair, fmt)
        assert torch.equal(torch.stack([npc.get_geo_feats(), npc.get_col_feats()], 1).cpu(), want)
        assert torch.equal(npc.cloud_pos(), s.npc.cloud_pos())
        if fmt is None:
            assert "feature_rows" not in ck and torch.equal(ck["geo_feats"], geo)
    n = s.npc.pts_num()
    assert sizes[None] - sizes["int8"] > 0.99 * n * (256 - 72) and sizes["int8"] - sizes["int4"] > 0.99 * n * 32


@gpu
def test_score_draws_take_valid_pixels_by_their_weight():
    cam, s, frames = _slam(base_cfg())
    torch.manual_seed(0)
    n = 300000
    cut = {"temperature": 0.8, "top_p": 0.95}
    idx = s.score_draws(frames, n, cut, edge_h=10, edge_w=15)
    assert idx.shape == (3, n) and idx.dtype == torch.int32
    from oracle import draw_oracle as DO
    for f, i in zip(frames, idx.cpu().long()):
        v, u = i // cam["W"], i % cam["W"]
        assert (v >= 10).all() and (v < cam["H"] - 10).all() and (u >= 15).all() and (u < cam["W"] - 15).all()
        d = f.depth.cpu()
        assert (d[v, u] > 0).all()
        mask = torch.zeros_like(d, dtype=torch.bool); mask[10:-10, 15:-15] = True
        w = DO.kept_weights(f.grad_scores[1].cpu().double().numpy(), mask=(mask & (d > 0)).reshape(-1).numpy(), **cut).astype(float)
        got = np.bincount(i.numpy(), minlength=w.size)
        assert (got[w == 0] == 0).all()
        # counts of 64 groups of pixels: binomial, standard deviation below sqrt(n p); six of them
        p = np.add.reduceat(w, np.arange(0, w.size, w.size // 64)) / w.sum()
        c = np.add.reduceat(got, np.arange(0, w.size, w.size // 64))
        assert (np.abs(c - n * p) <= 6 * np.sqrt(n * p) + 1).all()


@gpu
def test_a_frame_without_depth_draws_a_pixel_the_loops_filter():
    cam, s, frames = _slam(base_cfg())
    frames[0].depth.zero_()
    assert (s.score_draws(frames[:1], 50, {}) == 0).all()


@gpu
def test_the_frame_loops_run_on_score_draws():
    """tracking / mapping with score_sampling: the same loops, other pixels.  The draws they use are the ones that
    score_draws gives; handing those in as `draws` must give the same losses."""
    cfg = base_cfg()
    cfg["tracking"].update(score_sampling={"temperature": 1.0, "top_k": 20000}, iters=4, pixels=150)
    cfg["mapping"].update(score_sampling={"temperature": 0.7, "top_p": 0.9, "floor": 1e-2}, iters=6, pixels=300, pixels_adding=200)
    from point_slam_amd.slam import camera_tensor_from_c2w
    cam, s, frames = _slam(cfg)
    for f in frames[:2]:
        s.map(f, f.c2w, n_iters=6, fixed_iters=True)
        assert torch.isfinite(s.last_losses).all()
        s.keyframes.append(f)
    cam0 = camera_tensor_from_c2w(frames[2].c2w)
    torch.manual_seed(5)
    best = s.track(frames[2], cam0)
    first = s.last_losses.clone()
    assert torch.isfinite(best).all() and torch.isfinite(first).all()
    torch.manual_seed(5)
    idx = s.score_draws(frames[2:], 4 * 150, cfg["tracking"]["score_sampling"], 20, 20).reshape(4, 150)
    fb = torch.zeros(4, 2, 32, device="cuda").normal_(mean=0, std=0.01)
    tr = cfg["tracking"].pop("score_sampling")
    cfg["tracking"]["sample_with_color_grad"] = True          # draws handed in are full-image indices
    s._track_native(frames[2], cam0, 4, 150, draws=(idx, fb))
    # the first iteration's loss sums 150 rays in fp32, in any order: 150 * 2^-24
    assert abs(float(first[0, 0] - s.last_losses[0, 0])) <= 150 * 2.0 ** -24 * float(first[0, 0]), (first, s.last_losses, tr)


@gpu
def test_a_mapped_frame_end_to_end():
    """Scores -> drawn pixels -> points at those pixels -> their rows held in 8 bits -> read back into a second map that
    renders."""
    from point_slam_amd import host_ops as H
    from point_slam_amd.row_store import QuantizedRows
    cam, s, frames = _slam(base_cfg())
    f = frames[0]
    torch.manual_seed(1)
    idx = s.score_draws([f], 3000, {"temperature": 0.7, "top_p": 0.95})[0].long()
    nb = s.npc.pts_num()
    added = s._add_batch(f, f.c2w, idx, False)
    n = s.npc.pts_num()
    assert added > 0 and n == nb + 3 * added
    st = QuantizedRows(s.npc._max_points, 2, 32, "int8")
    st.write(torch.stack([s.npc.get_geo_feats()[:nb], s.npc.get_col_feats()[:nb]], 1))
    st.write(torch.stack([s.npc.get_geo_feats()[nb:], s.npc.get_col_feats()[nb:]], 1), first=nb)
    back = st.read(count=n)
    pair = torch.stack([s.npc.get_geo_feats(), s.npc.get_col_feats()], 1)
    assert torch.equal(back.cpu(), _stands_for(pair.cpu(), "int8"))
    step = pair.abs().amax(-1, keepdim=True) / 254
    assert ((back - pair).abs() <= step * (1 + 2.0 ** -20)).all()
    u, v = H.pixels_from_flat_index(idx[:500], 0, cam["H"], 0, cam["W"])
    ro, rd = H.get_rays_from_uv(u, v, f.c2w, cam["fx"], cam["fy"], cam["cx"], cam["cy"])
    gd, rq = f.depth[v.long(), u.long()], f.r_query[v.long(), u.long()]

    def render(geo, col):
        s.renderer.fixed_fallback = (torch.zeros(32, device="cuda"), torch.zeros(32, device="cuda"))
        with torch.no_grad():
            return s.renderer.render_batch_ray(s.npc, s.decoders, rd, ro, "cuda:0", "color", gt_depth=gd, npc_geo_feats=geo,
                                               npc_col_feats=col, is_tracker=False, dynamic_r_query=rq)[:3]
    full, q8 = render(pair[:, 0].contiguous(), pair[:, 1].contiguous()), render(back[:, 0].contiguous(), back[:, 1].contiguous())
    # a rendered depth is a weighted mean of samples at 0.98 .. 1.02 of the sensor depth, whatever the features are
    assert (full[0] - q8[0]).abs().max() <= 0.041 * gd.max() and torch.isfinite(q8[2]).all()
    assert not torch.equal(full[2], q8[2])


def _small_slam(tracking=None, mapping=None, **kw):
    from point_slam_amd.slam import HipSLAM
    cfg = base_cfg()
    if tracking is not None:
        cfg["tracking"]["score_sampling"] = tracking
    if mapping is not None:
        cfg["mapping"]["score_sampling"] = mapping
    return HipSLAM(cfg, dict(H=120, W=160, fx=100.0, fy=100.0, cx=80.0, cy=60.0), **kw)


def test_score_sampling_with_nothing_but_defaults_is_score_sampling():
    """{} names no parameter and takes every default; only an absent key, None and False mean uniform draws."""
    from point_slam_amd.slam import score_cut
    assert score_cut({}) is None and score_cut({"score_sampling": None}) is None and score_cut({"score_sampling": False}) is None
    assert score_cut({"score_sampling": {}}) == {} and score_cut({"score_sampling": {"top_p": 0.9}}) == {"top_p": 0.9}
    for bad in (True, 0.7, "top_p", [("top_p", 0.9)], {"topp": 0.9}, {"mask": None}, {"with_prob": True}):
        with pytest.raises(ValueError, match="score_sampling"):
            score_cut({"score_sampling": bad})
    for where in ("tracking", "mapping"):
        with pytest.raises(NotImplementedError):
            _small_slam(**{where: {}}, engine="dropin")
        with pytest.raises(ValueError, match="score_sampling"):
            _small_slam(**{where: True})


@gpu
def test_the_loops_draw_by_score_with_nothing_but_defaults(monkeypatch):
    cfg = base_cfg()
    cfg["tracking"].update(score_sampling={}, iters=2, pixels=100)
    cfg["mapping"].update(score_sampling={}, iters=3, pixels=200, pixels_adding=200)
    from point_slam_amd.slam import HipSLAM, camera_tensor_from_c2w
    cam, s, frames = _slam(cfg)
    calls = []
    draws = HipSLAM.score_draws
    monkeypatch.setattr(HipSLAM, "score_draws", lambda self, *a, **kw: calls.append(a[2]) or draws(self, *a, **kw))
    s.map(frames[0], frames[0].c2w, n_iters=3, fixed_iters=True)
    assert calls == [{}]
    s.track(frames[1], camera_tensor_from_c2w(frames[1].c2w))
    assert calls == [{}, {}] and torch.isfinite(s.last_losses).all()


@gpu
def test_a_frame_with_depth_in_its_border_only_draws_a_pixel_the_loops_filter():
    cam, s, frames = _slam(base_cfg())
    f = frames[0]
    f.depth[10:-10, 15:-15] = 0.0
    assert float(f.depth[0, 0]) > 0                          # a pixel of the border, which the loops would take
    idx = s.score_draws([f], 50, {"temperature": 0.7}, edge_h=10, edge_w=15)
    assert (f.depth.reshape(-1)[idx.long()] == 0).all()
    v, u = idx // cam["W"], idx % cam["W"]
    assert (v >= 10).all() and (v < cam["H"] - 10).all() and (u >= 15).all() and (u < cam["W"] - 15).all()


@gpu
def test_the_floor_of_flat_pixels():
    cam, s, frames = _slam(base_cfg())
    for floor in (-1e-3, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="floor"):
            s.score_draws(frames[:1], 5, {"floor": floor})
    f = frames[0]
    f.color[:, :160] = 0.5                                   # flat but for the half that is not
    flat = (s.grad_mag(f) == 0).reshape(-1)
    assert int(flat.sum()) > 1000
    idx = s.score_draws([f], 5000, {"floor": 0.0}).long()
    assert not flat[idx].any() and (f.depth.reshape(-1)[idx] > 0).all()
    assert flat[s.score_draws([f], 5000, {"floor": 10.0}).long()].any()
    frames[1].color.fill_(0.5)                               # no gradient anywhere: every pixel with depth alike
    for floor in (0.0, 1e-3):
        idx = s.score_draws(frames[1:2], 2000, {"floor": floor, "top_p": 0.9}).long()
        assert (frames[1].depth.reshape(-1)[idx] > 0).all() and idx.unique().numel() > 1000


@gpu
def test_a_border_that_leaves_no_pixel_is_refused():
    cam, s, frames = _slam(base_cfg())
    for eh, ew in ((cam["H"] // 2, 0), (0, cam["W"] // 2), (cam["H"], cam["W"]), (-1, 0)):
        with pytest.raises(ValueError, match="border"):
            s.score_draws(frames[:1], 5, {}, edge_h=eh, edge_w=ew)


def _owner_worker(rank, world, port, q, fmt):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from point_slam_amd import dist as PD
    from tests.test_dist_gloo import FakeCloud
    PD._RowWire = _HostWire
    g = torch.Generator().manual_seed(100)
    cloud = FakeCloud(torch.rand(10, 3, generator=g) + 5.0, torch.randn(10, 32, generator=g), torch.randn(10, 32, generator=g))
    before = torch.stack([cloud.geo, cloud.col], 1).clone()
    theta = torch.arange(6.0)
    sync = PD.FrameParallelSync(cloud, theta, n_color=4, wire=fmt, merge="owner")
    gr = torch.Generator().manual_seed(rank + 1)
    rows = [0, 1] if rank == 0 else [1, 2]
    sync.note_rows(cloud, torch.tensor(rows))
    for r in rows:
        cloud.geo[r] += torch.randn(32, generator=gr) * 0.1; cloud.col[r] += torch.randn(32, generator=gr) * 0.1
    moved = torch.stack([cloud.geo[:10], cloud.col[:10]], 1) - before
    theta += rank + 1
    counts = sync.exchange(cloud, theta)                     # no new points: the records of that half are empty
    q.put(tuple(x.numpy() if torch.is_tensor(x) else x for x in (rank, counts, torch.stack([cloud.geo, cloud.col], 1), moved, before, theta)))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("fmt", FORMATS)
def test_owner_writes_with_quantised_records_world2(fmt):
    """Of a row of the seed map that both ranks trained the lowest rank's change counts, as sent; the decoder stays fp32."""
    s = socket.socket(); s.bind(("127.0.0.1", 0)); port = s.getsockname()[1]; s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_owner_worker, args=(r, 2, port, q, fmt)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=120) for _ in range(2)], key=lambda x: x[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    (_, c0, f0, d0, before, t0), (_, c1, f1, d1, _, t1) = [[torch.from_numpy(x) if isinstance(x, np.ndarray) else x for x in r] for r in res]
    assert c0 == c1 == [0, 0] and torch.equal(f0, f1) and torch.equal(t0[:4], t1[:4]) and torch.equal(t0[:4], torch.arange(4.0) + 1.5)
    want = before.clone()
    q0, q1 = _stands_for(d0, fmt), _stands_for(d1, fmt)
    want[0] += q0[0]; want[1] += q0[1]; want[2] += q1[2]
    assert torch.equal(f0, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_records_of_halves_match_the_oracle(fmt, dtype):
    """bf16 and fp16 values into records, several groups to a head, the codes where a row of records begins on a multiple of 4 bytes only."""
    from point_slam_amd import row_store
    v = (torch.randn(301, 3, 64) * 0.1).to(dtype)
    for group in (64, 16):
        cw, sw = row_store.record_floats(3, 64, fmt, group)
        q, s = RO.quantize(v.float().numpy(), fmt, group)
        for code_col, scale_col, width in ((0, cw, cw + sw), (sw + 1, 1, cw + sw + 4), (2, cw + 5, cw + sw + 5)):
            rec = torch.full((301, width), 7.0, device="cuda")
            row_store.write_records(rec, v.cuda(), fmt, code_col, scale_col, group)
            back = row_store.read_records(rec, 3, 64, fmt, code_col, scale_col, group).cpu()
            assert torch.equal(back, torch.from_numpy(RO.values(q, s)))
            host = rec.cpu()
            assert torch.equal(host[:, scale_col:scale_col + sw], torch.from_numpy(s).reshape(301, sw))
            keep = torch.ones(width, dtype=torch.bool); keep[code_col:code_col + cw] = False; keep[scale_col:scale_col + sw] = False
            assert (host[:, keep] == 7.0).all()


@gpu
@pytest.mark.parametrize("temperature", [0.5, 1.0, 4.0])
def test_a_floor_of_zero_keeps_flat_pixels_out_whatever_u_is(temperature, monkeypatch):
    """u = 0 takes the first pixel that weighs anything at all: the flat ones in front of it must not."""
    cam, s, frames = _slam(base_cfg())
    f = frames[0]
    f.color[:, :160] = 0.5
    flat = (s.grad_mag(f) == 0).reshape(-1)
    live = (f.depth.reshape(-1) > 0)
    assert bool((flat & live)[:100].any()) and int((flat & live).nonzero()[0]) < int((~flat & live).nonzero()[0])
    monkeypatch.setattr(torch, "rand", lambda *size, **kw: torch.zeros(*size, **kw))
    idx = s.score_draws([f], 70, {"floor": 0.0, "temperature": temperature})
    assert (idx == int((~flat & live).nonzero()[0])).all()
