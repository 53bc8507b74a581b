"""Draws of indices from scores under temperature, top-k, top-p and min-p (psl_draw_indices, frame_ops.draw_indices): refusals
and the oracle's known answers on the CPU, the kernels against the extended-precision oracle on the GPU.

Indices have to be equal: both sides decide by sums whose relative error is below 2^-45 (2^20 fp64 additions at worst, in
practice 2^-50), so a random u falls between them with a chance below 1e-7 for each test here.  Where u or a limit is put ON
a border, weights are equal powers of two and every sum is exact.  prob: fp64 to its last rounding, so half an fp32 step of
the value, 2^-24, and the sums' 2^-45 beside it; 1.001 * 2^-24 is asserted."""
import ctypes as C
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import draw_oracle as DO
from point_slam_amd import _lib, frame_ops
from tests.helpers import ROOT

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_known_answers():
    s = np.log(np.array([4.0, 1, 2, 1]))
    assert np.allclose(DO.kept_weights(s).astype(float), [1, .25, .5, .25])
    assert np.allclose(DO.kept_weights(s, top_k=3).astype(float), [1, .25, .5, 0])       # a tie goes to the lower index
    assert np.allclose(DO.kept_weights(s, top_p=0.7).astype(float), [1, 0, .5, 0])
    assert np.allclose(DO.kept_weights(s, min_p=0.4).astype(float), [1, 0, .5, 0])
    assert np.allclose(DO.kept_weights(s, top_k=3, top_p=0.8).astype(float), [1, 0, .5, 0])      # 0.8 of what top-k left
    assert np.allclose(DO.kept_weights(s, temperature=0).astype(float), [1, 0, 0, 0])
    idx, p = DO.draws(np.zeros(8), np.arange(8) / 8)
    assert list(idx) == list(range(8)) and np.allclose(p, 1 / 8)
    assert DO.draws([-np.inf, np.nan], [0.5])[0][0] == -1
    assert list(DO.draws([0, np.inf, 1, np.inf], [0.0, 0.6])[0]) == [1, 3]


def _args(**kw):
    buf = (C.c_char * 8192)()
    p = C.addressof(buf)
    p += -p % 256
    L = _lib.lib()
    a = dict(n_rows=1, n_cols=16, n_draws=2, dtype=0, scores=p, score_stride=16, u=p + 64, u_stride=2, idx=p + 128, prob=None,
             temperature_all=1.0, top_p_all=1.0, min_p_all=0.0, top_k_all=0, ws=p + 256, ws_bytes=L.psl_draw_ws_bytes(1, 16))
    a.update(kw)
    r = _lib.psl_draw_args(**a)
    r._buf = buf
    return r


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(n_rows=-1), dict(n_rows=65536), dict(n_cols=-1), dict(n_cols=0x7fffffff), dict(n_draws=-1), dict(n_rows=65535, n_draws=1 << 30),
    dict(scores=None), dict(u=None), dict(idx=None), dict(ws=None), dict(ws_bytes=16), dict(score_stride=-1), dict(u_stride=-1),
    dict(mask_stride=-1), dict(ws=264), dict(scores=258), dict(idx=258), dict(temperature=257), dict(top_k=258),
    dict(temperature_all=float("nan")), dict(top_p_all=float("nan")), dict(min_p_all=float("nan"))])
def test_bad_arguments_are_refused(bad):
    L = _lib.lib()
    assert L.psl_draw_indices(C.byref(_args(**bad)), None) == -1 and b"psl_draw_indices" in L.psl_last_error()


def test_workspace_sizes_and_nothing_to_do():
    L = _lib.lib()
    assert L.psl_draw_ws_bytes(-1, 5) < 0 and L.psl_draw_ws_bytes(5, -1) < 0 and L.psl_draw_ws_bytes(70000, 5) < 0
    assert L.psl_draw_ws_bytes(0, 0) >= 0 and L.psl_draw_ws_bytes(1, 0) > 0
    assert L.psl_draw_ws_bytes(12, 816000) < 12 * 816000 * 8          # below one double to an entry
    assert L.psl_draw_ws_bytes(65535, 0x7f000000) > 1 << 40
    assert L.psl_draw_indices(None, None) == -1
    assert L.psl_draw_indices(C.byref(_args(n_rows=0, scores=None)), None) == 0
    assert L.psl_draw_indices(C.byref(_args(n_draws=0, u=None)), None) == 0


def test_python_refusals():
    s, u = torch.zeros(2, 8), torch.zeros(2, 3)
    for kw in (dict(scores=s.double()), dict(scores=s[None]), dict(u=u.double()), dict(u=u[:1]), dict(u=u[None]),
               dict(mask=torch.ones(2, 7, dtype=torch.bool)), dict(mask=torch.ones(2, 8)), dict(temperature=torch.ones(3)),
               dict(temperature=torch.ones(2, dtype=torch.float64)), dict(top_k=torch.ones(2)), dict(top_p=torch.ones(2, 1)),
               dict(min_p=torch.ones(1)), dict(temperature=float("nan")), dict(top_p=float("nan"))):
        a = dict(scores=s, u=u)
        a.update(kw)
        with pytest.raises(ValueError):
            frame_ops.draw_indices(**a)
    for S, U in (((1, 2 ** 32 + 5), (1, 3)), ((1, 5), (1, 2 ** 32 + 5)), ((65536, 5), (65536, 1))):      # sizes that a 32-bit field would wrap
        with pytest.raises(ValueError, match="up to 65535 rows"):
            frame_ops.draw_indices(torch.zeros(1, 1).expand(S), torch.zeros(1, 1).expand(U))
    with pytest.raises(_lib.PslError):
        frame_ops.draw_indices(s, u)                                  # no host fallback


def test_struct_layout_matches_ctypes(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    names = [f for f, _ in _lib.psl_draw_args._fields_]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pointslam_hip.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof(psl_draw_args, {f}));\n' for f in names)
                   + '  printf("%zu", sizeof(psl_draw_args)); return 0; }\n')
    exe = tmp_path / "l"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got == [getattr(_lib.psl_draw_args, f).offset for f in names] + [C.sizeof(_lib.psl_draw_args)]
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "pointslam_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct psl_draw_args \{(.*?)\} psl_draw_args;", hdr, flags=re.S).group(1)
    assert sum(st.count(",") + 1 for st in body.split(";") if st.strip()) == len(names)


# ------------------------------------------------------------------------------------------------ GPU
def _scores(R, V, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * spread).to(DT[dtype])


def _check(scores, u, mask=None, where="", dev="cuda", **par):
    """One call against the oracle, row by row.  par: numbers, or tensors [R]."""
    dpar = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in par.items()}
    idx, prob = frame_ops.draw_indices(scores.to(dev), u.to(dev), mask=None if mask is None else mask.to(dev), with_prob=True, **dpar)
    idx, prob = idx.cpu().numpy(), prob.cpu().double().numpy()
    for r in range(scores.shape[0]):
        cut = {k: (v[r].item() if torch.is_tensor(v) else v) for k, v in par.items()}
        m = None if mask is None else (mask if mask.dim() == 1 else mask[r]).numpy()
        want, p = DO.draws(scores[r].double().numpy(), u[r].numpy(), mask=m, **cut)
        bad = np.flatnonzero(idx[r] != want)
        assert bad.size == 0, (where, r, bad[:5], idx[r][bad[:5]], want[bad[:5]], u[r][bad[:5]], cut)
        # half a step is 2^-24 of the value down to 2^-126; below, where fp32's steps are 2^-149 wide, it is 2^-150
        assert np.all(np.abs(prob[r] - p) <= 1.001 * np.maximum(2.0 ** -24 * p, 2.0 ** -150)), (where, r)
    return idx


CUTS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=7), dict(top_p=0.9), dict(top_p=0.3, temperature=1.5), dict(min_p=0.05),
        dict(top_k=50, top_p=0.8, min_p=0.01, temperature=0.8), dict(top_k=300, top_p=0.999), dict(temperature=0.0), dict(top_p=0.0)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 2, 15, 16, 17, 255, 1000, 4096, 4097, 12289])
def test_cuts_and_lengths(dtype, V):
    R = 3
    s, u = _scores(R, V, dtype, seed=V), torch.rand(R, 65, generator=torch.Generator().manual_seed(V + 1))
    mask = torch.rand(R, V, generator=torch.Generator().manual_seed(V + 2)) < 0.7
    mask[0, 0] = True
    for cut in CUTS:
        _check(s, u, where=str(cut), **cut)
        _check(s, u, mask=mask, where=f"masked {cut}", **cut)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,V,n", [(1, 307200, 3000), (5, 131072, 1), (2, 50021, 257), (300, 500, 2), (40, 70000, 3)])
def test_long_rows_and_many_rows(dtype, R, V, n):
    s, u = _scores(R, V, dtype, seed=3), torch.rand(R, n, generator=torch.Generator().manual_seed(4))
    for cut in (dict(), dict(top_k=V // 4, temperature=0.7), dict(top_p=0.95), dict(top_k=2000, top_p=0.5, min_p=1e-3), dict(top_p=0.9999, temperature=2.0)):
        _check(s, u, where=str(cut), **cut)


@gpu
def test_parameters_of_each_row():
    R, V = 24, 5000
    g = torch.Generator().manual_seed(0)
    s, u = _scores(R, V, "f32"), torch.rand(R, 40, generator=g)
    par = dict(temperature=torch.rand(R, generator=g) * 2, top_k=torch.randint(-1, 400, (R,), generator=g, dtype=torch.int32),
               top_p=torch.rand(R, generator=g) * 1.2, min_p=torch.rand(R, generator=g) * 0.1 - 0.02)
    par["temperature"][0], par["temperature"][1], par["top_p"][2], par["min_p"][3] = 0.0, -1.0, -0.5, 1.0
    par["top_k"][4], par["min_p"][5], par["top_p"][6] = 1 << 30, 3.0, 1.0
    _check(s, u, **par)
    par["temperature"][7] = float("nan")
    idx = frame_ops.draw_indices(s.cuda(), u.cuda(), **{k: v.cuda() for k, v in par.items()})
    assert (idx[7].cpu() == s[7].argmax()).all()


@gpu
def test_ties_and_borders_are_exact():
    for V in (8, 64, 4096, 65536):
        s = torch.full((1, V), 0.25)
        u = (torch.arange(V) / V)[None].float()
        assert (_check(s, u)[0] == np.arange(V)).all()
        for k in (1, 3, V // 2):
            idx = _check(s, u, top_k=k, where="k")
            assert idx.max() == k - 1                            # ties: the lowest indices
        for p in (0.5, 0.25, 0.125):
            assert _check(s, u, top_p=p, where="p").max() == int(V * p) - 1
        assert _check(s, u, top_k=V // 2, top_p=0.5).max() == V // 4 - 1
        assert _check(s, u, min_p=1.0).max() == V - 1
    g = torch.Generator().manual_seed(1)
    s = torch.randint(0, 5, (4, 20000), generator=g).float()      # five scores, thousands of ties each
    u = torch.rand(4, 500, generator=g)
    for cut in (dict(top_k=5000), dict(top_k=17), dict(top_p=0.5), dict(top_p=0.97), dict(top_k=9000, top_p=0.6), dict(min_p=0.1)):
        _check(s, u, where=str(cut), **cut)
        _check(s.flip(0).bfloat16(), u, where=str(cut), **cut)
    z = torch.zeros(2, 100); z[:, ::2] = -0.0
    assert _check(z, torch.rand(2, 50), top_k=10).max() == 9      # -0 and +0 tie
    # u at 0, at the largest below 1, outside and NaN
    s = _scores(1, 3000, "f32")
    _check(s, torch.tensor([[0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), 1e-45]]), top_k=11)
    _check(s, torch.tensor([[0.0, 1 - 2.0 ** -24, 1.0]]))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_special_scores_and_empty_rows(dtype):
    V = 700
    lowest = torch.finfo(DT[dtype]).min
    s = _scores(12, V, dtype)
    inf, nan = float("inf"), float("nan")
    mask = torch.rand(12, V, generator=torch.Generator().manual_seed(5)) < 0.5
    s[0] = -inf
    s[1] = nan
    s[2, ::2], s[2, 1::2] = nan, -inf
    s[3, 100], s[3, 600] = inf, inf
    s[4, :] = lowest
    s[5, :300] = lowest
    s[6, 17] = nan
    s[7][~mask[7]] = nan
    s[8][~mask[8]] = inf
    mask[9] = False
    s[10] = -inf; s[10, 699] = 1.0
    s[11] = torch.finfo(DT[dtype]).max; s[11, 5] = lowest
    u = torch.rand(12, 30)
    for cut in (dict(), dict(top_k=5), dict(top_p=0.8), dict(top_k=200, top_p=0.5, min_p=0.1), dict(temperature=0.0), dict(temperature=1e-3), dict(temperature=1e30), dict(temperature=inf), dict(temperature=1e-320)):
        idx = _check(s, u, mask=mask, where=str(cut), **cut)
        assert (idx[[0, 1, 2, 9]] == -1).all()
        live = [3, 4, 5, 6, 7, 8, 11]
        assert all(mask[r, idx[r]].all() for r in live)
        idx = _check(s, u, where=str(cut), **cut)
        assert (idx[[0, 1, 2]] == -1).all() and set(idx[3]) <= {100, 600} and (idx[10] == 699).all()


@gpu
def test_strides_shared_masks_and_vectors():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 1100, generator=g)
    u = torch.rand(6, 20, generator=g)
    mask = torch.rand(1001, generator=g) < 0.5
    for off in (0, 1, 2, 3):
        for t in (torch.float32, torch.bfloat16):
            w = wide.to(t)
            want = _check(w[:, off:off + 1001].contiguous(), u, mask=mask, top_k=100)
            got = frame_ops.draw_indices(w.cuda()[:, off:off + 1001], u.cuda(), mask=mask.cuda(), top_k=100)
            assert (got.cpu().numpy() == want).all()
    want = _check(wide, u, top_p=0.7)
    assert (frame_ops.draw_indices(wide.t().contiguous().cuda().t(), u.cuda(), top_p=0.7).cpu().numpy() == want).all()
    assert (frame_ops.draw_indices(wide.cuda(), u.t().contiguous().cuda().t(), top_p=0.7).cpu().numpy() == want).all()
    one = frame_ops.draw_indices(wide[2].cuda(), u[2].cuda(), top_p=0.7)
    assert one.shape == (20,) and (one.cpu().numpy() == want[2]).all()
    same = frame_ops.draw_indices(wide[2].cuda().expand(6, -1), u.cuda(), top_p=0.7)
    assert (same[2].cpu().numpy() == want[2]).all()
    m8 = (mask.to(torch.uint8) * 7).cuda()
    assert torch.equal(frame_ops.draw_indices(wide.cuda()[:, :1001], u.cuda(), mask=m8), frame_ops.draw_indices(wide.cuda()[:, :1001], u.cuda(), mask=mask.cuda()))


@gpu
def test_nothing_to_draw_from_or_to_draw():
    assert frame_ops.draw_indices(torch.zeros(0, 5, device="cuda"), torch.zeros(0, 3, device="cuda")).shape == (0, 3)
    assert frame_ops.draw_indices(torch.zeros(2, 5, device="cuda"), torch.zeros(2, 0, device="cuda")).shape == (2, 0)
    idx, prob = frame_ops.draw_indices(torch.zeros(2, 0, device="cuda"), torch.rand(2, 3, device="cuda"), with_prob=True, top_k=3, top_p=0.5)
    assert (idx == -1).all() and (prob == 0).all()


@gpu
def test_draws_follow_the_distribution():
    """u on a regular grid: each index is drawn n * p times, give or take one."""
    s = _scores(1, 3000, "f32", spread=1.0)
    n = 200000
    u = ((torch.arange(n) + 0.5) / n).float()[None]
    for cut in (dict(), dict(top_k=700, top_p=0.9, temperature=0.8)):
        idx = frame_ops.draw_indices(s.cuda(), u.cuda(), **cut)[0].cpu().numpy()
        w = DO.kept_weights(s[0].double().numpy(), **cut).astype(float)
        assert np.abs(np.bincount(idx, minlength=3000) - n * w / w.sum()).max() <= 1.1


@gpu
def test_the_answer_does_not_change_from_run_to_run():
    s, u = _scores(4, 200000, "f32").cuda(), torch.rand(4, 50000).cuda()
    first = frame_ops.draw_indices(s, u, top_k=50000, top_p=0.9, with_prob=True)
    for _ in range(5):
        again = frame_ops.draw_indices(s, u, top_k=50000, top_p=0.9, with_prob=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@gpu
def test_another_stream_and_captured_graphs():
    s, u = _scores(3, 9000, "bf16").cuda(), torch.rand(3, 40).cuda()
    par = dict(top_k=500, top_p=0.9, min_p=0.001, temperature=0.7)
    want = frame_ops.draw_indices(s, u, **par)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = frame_ops.draw_indices(s, u, **par)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)
    s1, u1, s2, u2 = s.clone(), u.clone(), s.clone(), u.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = frame_ops.draw_indices(s1, u1, with_prob=True, **par)
    with torch.cuda.graph(g2):
        o2 = frame_ops.draw_indices(s2, u2, with_prob=True)
    for k in range(4):
        s1.copy_(_scores(3, 9000, "bf16", seed=10 + k)); u1.uniform_(); s2.copy_(_scores(3, 9000, "bf16", seed=20 + k)); u2.uniform_()
        g1.replay(); g2.replay()
        e1, e2 = frame_ops.draw_indices(s1, u1, with_prob=True, **par), frame_ops.draw_indices(s2, u2, with_prob=True)
        torch.cuda.synchronize()
        assert torch.equal(o1[0], e1[0]) and torch.equal(o1[1], e1[1]) and torch.equal(o2[0], e2[0]) and torch.equal(o2[1], e2[1])


@gpu
def test_captured_draws_from_long_rows_follow_their_inputs():
    """Scores and limits change between the replays, and with them the way a row takes: from a list, by sums over the row, empty."""
    R, V, n = 4, 40000, 50
    s, u, mask = _scores(R, V, "f32").cuda(), torch.rand(R, n).cuda(), torch.ones(R, V, dtype=torch.bool, device="cuda")
    k, p = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.ones(R, device="cuda")
    kw = dict(top_k=k, top_p=p, temperature=0.9, mask=mask, with_prob=True)
    frame_ops.draw_indices(s, u, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        idx, prob = frame_ops.draw_indices(s, u, **kw)
    limits = [([50, 0, 20000, 1], [0.9, 0.5, 1.0, 1.0]), ([0, 0, 0, 0], [1.0, 1.0, 1.0, 1.0]), ([30000, 700, 5, 0], [0.99, 1.0, 0.3, 0.999]),
              ([1024, 1025, 2000, 1], [1.0, 0.9, 0.9, 0.0])]
    for j, (kk, pp) in enumerate(limits + limits[:2]):
        s.copy_(_scores(R, V, "f32", seed=30 + j)); u.uniform_()
        k.copy_(torch.tensor(kk, dtype=torch.int32)); p.copy_(torch.tensor(pp))
        mask.fill_(True)
        mask[j % R] = False if j % 2 else True
        g.replay()
        want = frame_ops.draw_indices(s, u, **kw)
        torch.cuda.synchronize()
        assert torch.equal(idx, want[0]) and torch.equal(prob, want[1]), j
        _check(s.cpu(), u.cpu(), mask=mask.cpu(), where=str(j), top_k=k.cpu(), top_p=p.cpu(), temperature=0.9)


@gpu
def test_rows_longer_than_a_thousand_tiles_and_offsets_past_32_bits():
    V = 5_000_001
    s, u = _scores(2, V, "f32"), torch.rand(2, 300)
    _check(s, u)
    _check(s, u, top_k=1_000_000, top_p=0.9)
    store = torch.empty((1 << 32) + 5000, dtype=torch.float16, device="cuda")      # 8.6 GB
    far = torch.as_strided(store, (3, 1000), (1 << 31, 1))
    near = _scores(3, 1000, "f16")
    far.copy_(near)
    assert torch.equal(frame_ops.draw_indices(far, u[:1].expand(3, -1).cuda(), top_k=90), frame_ops.draw_indices(near.cuda(), u[:1].expand(3, -1).cuda(), top_k=90))


@gpu
def test_tensors_of_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    s, u = _scores(2, 3000, "f32"), torch.rand(2, 20)
    _check(s, u, dev="cuda:1", top_k=30)
    with pytest.raises(ValueError):
        frame_ops.draw_indices(s.to("cuda:1"), u.to("cuda:0"))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_equal_scores_in_a_long_row(dtype):
    """More candidates in the deciding bin than its list holds (a quarter of the row), and just fewer."""
    V = 60000
    g = torch.Generator().manual_seed(4)
    for share in (0.1, 0.24, 0.26, 0.6):
        s = torch.randn(2, V, generator=g)
        flat = torch.rand(2, V, generator=g) < share
        s[flat] = 0.5
        s = s.to(DT[dtype])
        u = torch.rand(2, 200, generator=g)
        above = int((s[0] > 0.5).sum())
        for cut in (dict(top_k=above + 1), dict(top_k=above + int(share * V / 3)), dict(top_p=0.7), dict(top_p=0.6, top_k=above + int(share * V / 2)),
                    dict(top_k=V - 5), dict(top_p=0.99, temperature=0.5), dict(top_p=0.2, top_k=above)):
            _check(s, u, where=f"{share} {cut}", **cut)


@gpu
def test_wide_and_narrow_ranges():
    """Scores that fill one bin, a few, or mostly the last one."""
    V = 30011
    g = torch.Generator().manual_seed(6)
    u = torch.rand(1, 300, generator=g)
    base = torch.randn(1, V, generator=g)
    for s in (base * 1e-6, base * 1e-30, base * 1e4, base * 1e30, base.exp().exp(), torch.cat([base[:, :V - 1] * 1e-3, torch.tensor([[50.0]])], 1),
              torch.where(base > 2.5, base, torch.full_like(base, torch.finfo(torch.float32).min))):
        for cut in (dict(top_k=1000), dict(top_p=0.9), dict(top_k=20000, top_p=0.99), dict(top_p=0.5, temperature=1e-3), dict(top_k=5000, temperature=1e4), dict(top_p=1 - 1e-9), dict(top_k=V - 1)):
            _check(s, u, where=str(cut), **cut)
    for scale, t in ((1e-37, 1e-37), (1e-40, 1e-41), (1e-38, 1e-30), (1e30, 1e35), (1e-30, 1e-320), (1e37, 1e-300)):
        for cut in (dict(top_p=0.9), dict(top_k=700, top_p=0.5), dict(top_k=25000)):
            _check(base * scale, u, where=f"{scale} {t} {cut}", temperature=t, **cut)
    s = base.clone(); s[0, ::1000] = float("inf")
    for t in (1.0, float("inf"), 1e-300, 1e300):
        for cut in (dict(top_p=0.5), dict(top_k=7), dict(top_k=3000, top_p=0.9)):
            _check(s, u, where=f"inf {t} {cut}", temperature=t, **cut)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_entries_kept_of_long_rows(dtype):
    """Rows of which up to 1 024 entries are in question, and just over that: a limit on the count, on the mass of a sharp row, both,
    a floor, no temperature; with masks; ties that straddle the limit; few draws and very many."""
    R, V = 9, 30011
    s = _scores(R, V, dtype, seed=5, spread=3.0)
    s[7] = torch.randint(0, 40, (V,), generator=torch.Generator().manual_seed(6)).to(s.dtype)       # some 750 entries to a score
    s[8, :] = -4.0
    s[8, 17::101] = 2.0                                                                             # 297 equal ones above the rest
    mask = torch.rand(R, V, generator=torch.Generator().manual_seed(7)) < 0.5
    mask[3] = False
    mask[4] = False
    mask[4, 29999] = True
    u = torch.rand(R, 33, generator=torch.Generator().manual_seed(8))
    u[:, 0], u[:, 1] = 0.0, 1.0 - 2.0 ** -24
    k = torch.tensor([1, 2, 200, 1024, 1025, 900, 0, 760, 300], dtype=torch.int32)
    p = torch.tensor([0.9, 0.5, 0.95, 1.0, 1.0, 0.999, 0.6, 0.97, 0.5])
    t = torch.tensor([1.0, 0.7, 0.9, 1.3, 0.8, 2.0, 0.2, 0.9, 1.0])
    m = torch.tensor([0.0, 0.1, 0.02, 0.0, 0.0, 1e-4, 0.0, 0.0, 0.0])
    for kw in (dict(top_k=k, temperature=t), dict(top_k=k, top_p=p, temperature=t, min_p=m), dict(top_p=p, temperature=0.15), dict(top_k=297), dict(top_k=298),
               dict(top_k=V, top_p=p), dict(temperature=0.0), dict(top_k=5000, top_p=0.9)):
        few = _check(s, u, where=str(kw), **kw)
        _check(s, u, mask=mask, where="masked " + str(kw), **kw)
        for times in (150, 600):                     # from the list still, and by sums over the row
            many, _ = frame_ops.draw_indices(s.cuda(), u.repeat(1, times).cuda(), with_prob=True, **{a: b.cuda() if torch.is_tensor(b) else b for a, b in kw.items()})
            assert np.array_equal(many[:, -33:].cpu().numpy(), few) and np.array_equal(many[:, :33].cpu().numpy(), few), kw


@gpu
@pytest.mark.parametrize("V,n", [(2048, 1024), (2048, 1025), (16384, 4096), (16384, 4097), (16385, 1), (40000, 622), (40000, 626), (40000, 16384), (40000, 16385)])
def test_both_sides_of_each_limit_between_forms(V, n):
    s, u = _scores(2, V, "f32", seed=V), torch.rand(2, n, generator=torch.Generator().manual_seed(n))
    for cut in (dict(), dict(top_k=90), dict(top_p=0.9), dict(top_k=2000, top_p=0.99, min_p=1e-4)):
        _check(s, u, where=str(cut), **cut)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [16385, 300000])
def test_the_smallest_u_where_the_first_entries_weigh_next_to_nothing(V, dtype):
    """Leading entries 100 and 700 temperatures below the rest -- 4e-44 and 1e-304 of its weight, below what fp32 holds -- and in
    front of them entries that are not to be drawn: u = 0 (and what is turned into it) takes the first that is."""
    u = torch.tensor([[0.0, -1.0, float("nan"), 1e-45, 2.0 ** -24, 0.5, 1 - 2.0 ** -24]] * 5)
    for below in (100.0, 700.0):
        for lead in (16, 40, 2000):
            s = _scores(5, V, dtype, seed=V + lead, spread=0.5)
            s[:, :lead] = -below
            mask = torch.ones(5, V, dtype=torch.bool)
            mask[0, 0] = False
            s[1, :3] = -float("inf")
            s[2, :17] = float("nan")
            mask[3, ::16] = False
            s[4, 0] = float("inf")
            mask[4, :lead - 1] = False                      # one light entry in its block
            for cut in (dict(), dict(top_k=V - 5), dict(min_p=1e-306)):
                first = _check(s, u, mask=mask, where=f"{below} {lead} {cut}", **cut)[:, 0]
                if cut != dict(top_k=V - 5):
                    assert first.tolist() == [1, 3, 17, 1, lead - 1], (below, lead, cut)
            many = frame_ops.draw_indices(s.cuda(), torch.zeros(5, 20000, device="cuda"), mask=mask.cuda())      # places of every group
            assert (many.cpu() == torch.tensor([1, 3, 17, 1, lead - 1])[:, None]).all()


@gpu
def test_u_on_the_border_of_a_chunk_that_begins_with_light_entries():
    """Three fifths of a row are equal weights whose sums are exact; u = 1/8 is their sum in front of the second 4 096 entries, where 15
    entries of e^-100 or e^-700 follow one that is masked."""
    for below in (100.0, 700.0):
        s = torch.zeros(1, 5 * 8192)
        mask = torch.ones(1, 5 * 8192, dtype=torch.bool)
        s[0, 4096:4112], mask[0, 4096] = -below, False
        mask[0, 4112 + 28672:] = False                      # 32 768 entries of weight 1
        idx, prob = frame_ops.draw_indices(s.cuda(), torch.tensor([[0.125]], device="cuda"), mask=mask.cuda(), with_prob=True)
        # any entry that lies within rounding of the border, and none that is masked
        assert 4095 <= int(idx) <= 4112 and bool(mask[0, int(idx)]), (below, int(idx))
        w = 1.0 if int(idx) in (4095, 4112) else np.exp(-below)
        assert abs(float(prob) - w / 32768) <= 1.001 * max(2.0 ** -24 * w / 32768, 2.0 ** -150)


@gpu
@pytest.mark.parametrize("how", ["masked", "-inf", "nan"])
def test_u_on_a_border_with_nothing_to_draw_behind_it(how):
    """Rows of two equal halves with 56 empty blocks between them, the first entry of every block excluded: u = 0.5 lies within
    rounding of the border, and the running sums of empty blocks are off by a last place in one row of eight.  The draw is the last entry
    in front or the first behind."""
    R, V = 400, 20000
    g = torch.Generator().manual_seed(12)
    half = torch.randn(R, 1600, generator=g)
    s, ok = torch.zeros(R, V), torch.zeros(R, V, dtype=torch.bool)
    for at in (0, 2496):
        s[:, at:at + 1600], ok[:, at:at + 1600] = half, True
    ok[:, ::16] = False
    s[~ok] = {"masked": 3.0, "-inf": -float("inf"), "nan": float("nan")}[how]
    u = torch.full((R, 3), 0.5)
    idx = frame_ops.draw_indices(s.cuda(), u.cuda(), mask=ok.cuda() if how == "masked" else None).cpu()
    assert bool(((idx == 1599) | (idx == 2497)).all()), idx[(idx != 1599) & (idx != 2497)].unique()


def test_a_call_asks_for_the_workspace_it_uses():
    L = _lib.lib()

    def need(R, V, n, **kw):
        return L.psl_draw_call_ws_bytes(C.byref(_args(n_rows=R, n_cols=V, n_draws=n, **kw)))
    some = C.c_float(0.0)
    for R, V, n, kw in ((1, 2048, 1, {}), (4096, 2048, 1, dict(top_k_all=50)), (65535, 2048, 1, {}), (3, 16384, 1024, {}), (3, 16384, 4096, dict(top_p_all=0.9)),
                        (3, 0, 7, {}), (2, 500, 4096, dict(temperature=C.addressof(some))), (2, 500, 4096, dict(temperature_all=0.0))):
        assert need(R, V, n, **kw) == 256, (R, V, n, kw)
    for R, V, n, kw in ((3, 16384, 1025, {}), (3, 16384, 4097, dict(top_p_all=0.9)), (3, 16385, 1, {}), (3, 2048, 1025, dict(min_p_all=0.1)), (2, 816000, 5, dict(top_k_all=9))):
        assert need(R, V, n, **kw) == L.psl_draw_ws_bytes(R, V), (R, V, n, kw)
    assert L.psl_draw_ws_bytes(4096, 2048) < 4096 * 64 * 1024
    assert need(-1, 5, 1) == -1 and need(5, -1, 1) == -1 and need(65536, 5, 1) == -1 and L.psl_draw_call_ws_bytes(None) == -1
    for kw in (dict(ws_bytes=255), dict(n_draws=2000, ws_bytes=L.psl_draw_ws_bytes(1, 16) - 1)):
        assert L.psl_draw_indices(C.byref(_args(**kw)), None) == -1 and b"workspace" in L.psl_last_error()


@gpu
@pytest.mark.parametrize("R,V,n,k", [(7, 2048, 5, 50), (7, 16384, 1024, 0), (2, 700, 4096, 300), (2, 700, 4097, 300), (3, 3000, 1025, 0), (3, 16385, 2, 900),
                                     (3, 16385, 20000, 9000), (2, 50021, 3, 0)])
def test_nothing_behind_the_workspace_is_written(R, V, n, k):
    s, u = _scores(R, V, "f32").cuda(), torch.rand(R, n).cuda()
    want = frame_ops.draw_indices(s, u, top_k=k)
    idx = torch.empty(R, n, dtype=torch.int32, device="cuda")
    a = _lib.psl_draw_args(n_rows=R, n_cols=V, n_draws=n, scores=s.data_ptr(), score_stride=V, u=u.data_ptr(), u_stride=n, idx=idx.data_ptr(),
                           temperature_all=1.0, top_p_all=1.0, top_k_all=k)
    a.ws_bytes = _lib.lib().psl_draw_call_ws_bytes(C.byref(a))
    ws = torch.full((a.ws_bytes + 4096,), 0xa5, dtype=torch.uint8, device="cuda")
    a.ws = ws.data_ptr()
    _lib.call_on(s.device, "psl_draw_indices", a)
    assert torch.equal(idx, want) and (ws[a.ws_bytes:] == 0xa5).all()


@gpu
def test_many_short_rows_take_no_workspace_to_speak_of():
    s, u = _scores(4096, 2048, "bf16").cuda(), torch.rand(4096, 1, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    idx = frame_ops.draw_indices(s, u, top_k=40, top_p=0.9)
    assert torch.cuda.max_memory_allocated() - before <= 1 << 20
    for r in (0, 1, 2047, 4095):
        want, _ = DO.draws(s[r].double().cpu().numpy(), u[r].cpu().numpy(), top_k=40, top_p=0.9)
        assert int(idx[r, 0]) == want[0]


@gpu
def test_as_many_rows_as_a_call_takes():
    R = 65535
    for V, kw in ((2100, dict(top_k=50, top_p=0.9)), (16385, dict()), (16385, dict(top_k=90, top_p=0.9))):
        s = _scores(1, V, "bf16", seed=V).cuda()
        u = torch.rand(R, 1, device="cuda")
        idx, prob = frame_ops.draw_indices(s.expand(R, V), u, with_prob=True, **kw)
        one, p1 = frame_ops.draw_indices(s, u.t().contiguous()[:, :1000], with_prob=True, **kw)
        want, p = DO.draws(s[0].double().cpu().numpy(), u[:, 0].cpu().numpy(), **kw)
        assert np.array_equal(idx[:, 0].cpu().numpy(), want) and torch.equal(idx[:1000, 0], one[0]) and torch.equal(prob[:1000, 0], p1[0])
        assert np.all(np.abs(prob[:, 0].cpu().double().numpy() - p) <= 1.001 * 2.0 ** -24 * p)


@gpu
def test_calls_on_several_streams_at_once():
    jobs = [(_scores(3, V, "f32", seed=V).cuda(), torch.rand(3, n).cuda(), kw) for V, n, kw in
            ((200000, 20000, dict(top_p=0.95)), (40000, 5, dict(top_k=300, top_p=0.9)), (3000, 100, dict(top_k=50)), (120000, 3000, dict(min_p=1e-3)))]
    want = [frame_ops.draw_indices(s, u, with_prob=True, **kw) for s, u, kw in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(5):
        for k, (s, u, kw) in enumerate(jobs):
            with torch.cuda.stream(streams[k]):
                got[k].append(frame_ops.draw_indices(s, u, with_prob=True, **kw))
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        for g in got[k]:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1]), k
