"""Per-frame image operators in front of the render/optimise path, on the device.

Mirrors of host code the reference runs with skimage / scipy / numpy once per frame:
  * dynamic_radius_maps        <- src/Tracker.py:235-250, src/Mapper.py:686-701
  * get_selected_index_with_grad <- src/common.py:116-159
  * keyframe_overlap / keyframe_selection_overlap <- src/Mapper.py:170-235
All three call libpointslam_hip.so (psl_frame_radii, psl_topgrad_select_sync, psl_keyframe_overlap_sync); there is
no torch fallback.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib


def dynamic_radius_maps(color: torch.Tensor, cfg: dict, with_grad_mag: bool = False):
    """color [H,W,3] float32 on the device -> (r_add [H,W] f32, r_query [H,W] f32[, grad_mag [H,W] f64])."""
    pc = cfg["pointcloud"]
    H, W = int(color.shape[0]), int(color.shape[1])
    col = color.detach().float().contiguous()
    r_add = torch.empty(H, W, device=col.device, dtype=torch.float32)
    r_query = torch.empty(H, W, device=col.device, dtype=torch.float32)
    gm = torch.empty(H, W, device=col.device, dtype=torch.float64) if with_grad_mag else None
    _lib.check(_lib.lib().psl_frame_radii(_lib.ptr(col), H, W, float(pc["color_grad_threshold"]),
                                          float(pc["radius_add_max"]), float(pc["radius_add_min"]),
                                          float(pc["radius_query_ratio"]), _lib.ptr(gm), _lib.ptr(r_add),
                                          _lib.ptr(r_query), _lib.stream_ptr()), "psl_frame_radii")
    return (r_add, r_query, gm) if with_grad_mag else (r_add, r_query)


def get_selected_index_with_grad(npc, H0, H1, W0, W1, n, image, ratio=15, gt_depth=None, depth_limit=False,
                                 grad_mag=None, cfg=None):
    """common.get_selected_index_with_grad (src/common.py:116-159): flat indices (sorted, int64, on the device) of
    the pixels among the top ratio*n by colour-gradient magnitude that lie in the region and have sensor depth;
    also returns the gradient-magnitude image (float64).  `npc` supplies the native context (scratch)."""
    H, W = int(image.shape[0]), int(image.shape[1])
    if grad_mag is None:
        col = image.detach().float().contiguous()
        grad_mag = torch.empty(H, W, device=col.device, dtype=torch.float64)
        _lib.check(_lib.lib().psl_frame_radii(_lib.ptr(col), H, W, 0.15, 0.08, 0.02, 2.0, _lib.ptr(grad_mag), None, None,
                                              _lib.stream_ptr()), "psl_frame_radii")
    k = min(int(ratio * n), H * W)
    sel = torch.empty(max(k, 1), device=grad_mag.device, dtype=torch.int32)
    n_sel = C.c_int(0)
    dep = gt_depth.detach().float().contiguous() if gt_depth is not None else None
    _lib.check(_lib.lib().psl_topgrad_select_sync(npc.handle, _lib.ptr(grad_mag), _lib.ptr(dep), H, W, k, int(H0), int(H1),
                                                  int(W0), int(W1), 5.0 if depth_limit else 0.0, _lib.ptr(sel),
                                                  C.byref(n_sel), _lib.stream_ptr()), "psl_topgrad_select_sync")
    return torch.sort(sel[:n_sel.value].long()).values, grad_mag


_DRAW_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def draw_indices(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None, with_prob=False):
    """Draws of indices from rows of scores (psl_draw_indices; no reference counterpart: the reference takes pixels uniformly
    or from the hard top-k of get_selected_index_with_grad).

    scores [R, V] (fp32, bf16 or fp16; pixels of a frame, entries of a vocabulary), u [R, n] fp32 in [0, 1): n draws from
    each row, with replacement -- the random numbers are the caller's, as everywhere in this package.  An entry weighs
    exp((score - max) / temperature); top_k (0: off), top_p (1: off) and min_p (0: off) cut the tail, in that order, ties to
    the lower index; temperature or a limit may be a number or a tensor [R].  `mask` (bool or uint8, [R, V] or [V]): entries
    that may be drawn -- what the others hold, NaN included, does not matter.  A vector of scores and a vector u make one row.
    Returns indices int32 [R, n] (-1 where a row has nothing to draw) and, with_prob, their probabilities fp32 [R, n] under
    the cut distribution (what an importance weight divides by).  Probabilities are numbers, not part of an autograd graph: no
    gradient reaches scores through them, whether scores require one or not."""
    one = scores.dim() == 1
    if one:
        scores, u = scores.unsqueeze(0), u.unsqueeze(0)
        mask = mask.unsqueeze(0) if mask is not None and mask.dim() == 1 else mask
    if scores.dim() != 2 or scores.dtype not in _DRAW_DTYPES:
        raise ValueError(f"scores: [rows, entries] in float32, bfloat16 or float16, got {tuple(scores.shape)} {scores.dtype}")
    R, V = scores.shape
    dev = scores.device
    if u.dim() != 2 or u.dtype != torch.float32 or u.shape[0] != R or u.device != dev:
        raise ValueError(f"u: float32 [{R}, draws] on {dev}, got {tuple(u.shape)} {u.dtype} on {u.device}")
    n = u.shape[1]
    if R > 65535 or V > 0x7f000000 or n > 0x7fffffff:
        raise ValueError(f"{R} rows of {V} entries, {n} draws: up to 65535 rows of {0x7f000000} entries, {0x7fffffff} draws")
    if V > 1 and scores.stride(1) != 1:
        scores = scores.contiguous()
    if n > 1 and u.stride(1) != 1:
        u = u.contiguous()
    a = _lib.psl_draw_args(n_rows=R, n_cols=V, n_draws=n, dtype=_DRAW_DTYPES[scores.dtype], scores=scores.data_ptr(),
                           score_stride=scores.stride(0), u=u.data_ptr(), u_stride=u.stride(0))
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.device != dev or tuple(mask.shape) not in ((R, V), (V,)):
            raise ValueError(f"mask: bool or uint8 [{R}, {V}] or [{V}] on {dev}, got {tuple(mask.shape)} {mask.dtype} on {mask.device}")
        mask = mask.expand(R, V)
        if V > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
        a.mask, a.mask_stride = mask.data_ptr(), mask.stride(0)
    keep = []
    for name, x, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                        ("min_p", min_p, torch.float32)):
        if torch.is_tensor(x):
            if tuple(x.shape) != (R,) or x.device != dev or x.dtype != dt:
                raise ValueError(f"{name}: a number or {dt} [{R}] on {dev}, got {tuple(x.shape)} {x.dtype} on {x.device}")
            x = x.contiguous()
            keep.append(x)
            setattr(a, name, x.data_ptr())
        elif name == "top_k":
            a.top_k_all = max(0, min(int(x), 0x7fffffff))
        elif x != x:
            raise ValueError(f"{name} is NaN")
        else:
            setattr(a, name + "_all", float(x))
    if dev.type != "cuda":
        raise _lib.PslError(f"psl_draw_indices: tensors on {dev}; the kernels run on the GPU and have no host fallback")
    idx = torch.empty(R, n, dtype=torch.int32, device=dev)
    prob = torch.empty(R, n, dtype=torch.float32, device=dev) if with_prob else None
    if R and n:
        a.ws_bytes = _lib.check(_lib.lib().psl_draw_call_ws_bytes(C.byref(a)), "psl_draw_call_ws_bytes")
        ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=dev)
        a.idx, a.prob, a.ws = idx.data_ptr(), prob.data_ptr() if with_prob else None, ws.data_ptr()
        _lib.call_on(dev, "psl_draw_indices", a)
    if one:
        idx, prob = idx[0], prob[0] if with_prob else None
    return (idx, prob) if with_prob else idx


def keyframe_overlap(rays_o, rays_d, gt_depth, keyframe_c2w, cam: dict, n_samples=8, edge=20):
    """percent_inside per keyframe (src/Mapper.py:197-229). keyframe_c2w: list of [4,4] (or [3,4]) poses, tensors or host
    float lists.  Rays with gt_depth <= 0 are skipped by the kernel (get_samples' depth_filter, Mapper.py:190-192): the
    caller may pass the uncompacted draw."""
    n_kf = len(keyframe_c2w)
    if n_kf == 0:
        return np.zeros(0, dtype=np.float32)
    flat = []
    for c in keyframe_c2w:
        if isinstance(c, (list, tuple)):       # 12 (3x4) or 16 host floats, row-major: Frame.c2w_host() -- no device copy
            h = [float(x) for x in c]
            flat += h[:12] + [0.0, 0.0, 0.0, 1.0]
            continue
        m = torch.eye(4)
        cc = c.detach().float().cpu()
        m[:cc.shape[0], :] = cc
        flat += m.reshape(-1).tolist()
    host = (C.c_float * (16 * n_kf))(*flat)
    out = (C.c_float * n_kf)()
    ro = rays_o.detach().float().contiguous()
    rd = rays_d.detach().float().contiguous()
    gd = gt_depth.detach().float().reshape(-1).contiguous()
    intr = _lib.psl_cam_intr(H=cam["H"], W=cam["W"], fx=cam["fx"], fy=cam["fy"], cx=cam["cx"], cy=cam["cy"])
    _lib.check(_lib.lib().psl_keyframe_overlap_sync(_lib.ptr(ro), _lib.ptr(rd), _lib.ptr(gd), int(ro.shape[0]),
                                                    int(n_samples), host, n_kf, intr, float(edge), out,
                                                    _lib.stream_ptr()), "psl_keyframe_overlap_sync")
    return np.array(list(out), dtype=np.float32)


def keyframe_selection_overlap(rays_o, rays_d, gt_depth, keyframe_c2w, cam: dict, k, n_samples=8, rng=None):
    """Mapper.keyframe_selection_overlap (src/Mapper.py:170-235): keyframes with any overlap, in random order, the
    first k of them (np.random.permutation on the host, as in the reference)."""
    pct = keyframe_overlap(rays_o, rays_d, gt_depth, keyframe_c2w, cam, n_samples)
    order = sorted(range(len(pct)), key=lambda i: pct[i], reverse=True)
    sel = [i for i in order if pct[i] > 0.0]
    perm = (rng or np.random).permutation(np.array(sel, dtype=np.int64)) if sel else np.zeros(0, dtype=np.int64)
    return list(perm[:k])


def image_metrics(gt_color, gt_depth, color, depth):
    """(psnr, ms_ssim, depth_l1) of one rendered frame as the end-of-run evaluation computes them
    (src/Mapper.py:861-879).  Images [H,W,3] / [H,W] on the device."""
    H, W = int(gt_depth.shape[0]), int(gt_depth.shape[1])
    out = (C.c_double * 3)()
    a, b = gt_color.detach().float().contiguous(), color.detach().float().contiguous()
    c, d = gt_depth.detach().float().contiguous(), depth.detach().float().contiguous()
    _lib.check(_lib.lib().psl_image_metrics_sync(_lib.ptr(a), _lib.ptr(c), _lib.ptr(b), _lib.ptr(d), H, W, out,
                                                 _lib.stream_ptr()), "psl_image_metrics_sync")
    return float(out[0]), float(out[1]), float(out[2])
