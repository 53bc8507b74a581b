"""ctypes binding of libpointslam_hip.so (include/pointslam_hip.h).

The library is the product; there is NO Python/CPU fallback: if the shared
object is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
# PSL_LIB=<path>: load another build of the same ABI (A/B measurements of two builds on ONE box, tools/gpu_round.sh)
LIB_PATH = os.environ.get("PSL_LIB") or os.path.join(_HERE, "libpointslam_hip.so")


class PslError(RuntimeError):
    pass


ABI_VERSION = 9     # include/pointslam_hip.h: psl_abi_version(); v2: psl_render_args.z_vals; v3: exposure blocks,
#                     full-image pixel indices in psl_track_args, step0_params in psl_map_args; v4: psl_dedupe_count / psl_dedupe_blocks,
#                     psl_comm_* / psl_allgather_new_points (RCCL inside the library), psl_map_args refinement fields;
#                     v5: psl_allgather_decide (rank-invariant capacity decision), psl_selftest_math; v6: psl_comm_reserve, psl_pose_const_speed, psl_selftest_traffic;
#                     v8: psl_rows_write / psl_rows_read (feature rows in 8 or 4 bits), psl_draw_ws_bytes / psl_draw_indices (draws from scores);
#                     v9: psl_draw_call_ws_bytes
EXPOSURE_DIM, EXPOSURE_MLP_FLOATS = 8, 2700


class psl_config(C.Structure):
    _fields_ = [("n_surface", C.c_int32), ("nn_num", C.c_int32), ("c_dim", C.c_int32), ("min_nn_num", C.c_int32),
                ("near_end_surface", C.c_float), ("far_end_surface", C.c_float), ("radius_query", C.c_float),
                ("max_query_radius", C.c_float), ("encode_rel_pos", C.c_int32), ("max_points", C.c_int32), ("nn_weighting", C.c_int32)]


class psl_render_args(C.Structure):
    _fields_ = [("n_rays", C.c_int32), ("flags", C.c_int32), ("sigmoid_coef", C.c_float),
                ("rays_o", C.c_void_p), ("rays_d", C.c_void_p), ("gt_depth", C.c_void_p), ("r_query", C.c_void_p),
                ("geo_feats", C.c_void_p), ("col_feats", C.c_void_p), ("params", C.c_void_p),
                ("col_embed_B", C.c_void_p), ("fallback_geo", C.c_void_p), ("fallback_col", C.c_void_p),
                ("exposure_affine", C.c_void_p), ("ws", C.c_void_p),
                ("depth", C.c_void_p), ("var", C.c_void_p), ("rgb", C.c_void_p), ("valid_ray", C.c_void_p),
                ("z_vals", C.c_void_p)]


class psl_render_grads(C.Structure):
    _fields_ = [("g_depth", C.c_void_p), ("g_var", C.c_void_p), ("g_rgb", C.c_void_p),
                ("g_geo_feats", C.c_void_p), ("g_col_feats", C.c_void_p), ("feat_row_map", C.c_void_p),
                ("g_params", C.c_void_p), ("g_rays_o", C.c_void_p), ("g_rays_d", C.c_void_p),
                ("g_exposure_affine", C.c_void_p)]


class psl_cam_intr(C.Structure):
    _fields_ = [("H", C.c_int32), ("W", C.c_int32), ("fx", C.c_float), ("fy", C.c_float), ("cx", C.c_float),
                ("cy", C.c_float)]


class psl_frame_view(C.Structure):
    _fields_ = [("depth", C.c_void_p), ("color", C.c_void_p), ("r_query", C.c_void_p), ("c2w", C.c_float * 12)]


class psl_exposure_args(C.Structure):
    _fields_ = [("mlp", C.c_void_p), ("feats", C.c_void_p), ("adam", C.c_void_p), ("lr_mlp", C.c_float),
                ("lr_feat", C.c_float), ("step0", C.c_int32)]


class psl_track_args(C.Structure):
    _fields_ = [("cam", psl_cam_intr), ("edge_h", C.c_int32), ("edge_w", C.c_int32), ("n_iters", C.c_int32),
                ("n_pix", C.c_int32), ("pix_idx", C.c_void_p), ("fallback", C.c_void_p), ("frame", psl_frame_view),
                ("cam_tensor", C.c_void_p), ("adam_state", C.c_void_p), ("step0", C.c_int32), ("lr_T", C.c_float),
                ("lr_quat", C.c_float), ("w_color", C.c_float), ("handle_dynamic", C.c_int32),
                ("use_color", C.c_int32), ("sigmoid_coef", C.c_float), ("geo_feats", C.c_void_p),
                ("col_feats", C.c_void_p), ("params", C.c_void_p), ("col_embed_B", C.c_void_p), ("ws", C.c_void_p),
                ("loss_out", C.c_void_p), ("best_out", C.c_void_p), ("pix_full_image", C.c_int32),
                ("exposure", C.POINTER(psl_exposure_args))]


class psl_map_args(C.Structure):
    _fields_ = [("cam", psl_cam_intr), ("n_frames", C.c_int32), ("pix_per_frame", C.c_int32), ("n_iters", C.c_int32),
                ("n_geo_iters", C.c_int32), ("frames", C.POINTER(psl_frame_view)), ("pix_idx", C.c_void_p),
                ("fallback", C.c_void_p), ("geo_feats", C.c_void_p), ("col_feats", C.c_void_p), ("params", C.c_void_p),
                ("col_embed_B", C.c_void_p), ("sel_rows", C.c_void_p), ("row_map", C.c_void_p), ("n_sel", C.c_int32),
                ("g_geo", C.c_void_p), ("g_col", C.c_void_p), ("adam_geo", C.c_void_p), ("adam_col", C.c_void_p),
                ("adam_params", C.c_void_p), ("step0_geo", C.c_int32), ("step0_col", C.c_int32),
                ("train_decoder", C.c_int32), ("lr_geo_geo_stage", C.c_float), ("lr_geo_color_stage", C.c_float),
                ("lr_col", C.c_float), ("lr_decoder", C.c_float), ("w_color", C.c_float), ("sigmoid_coef", C.c_float),
                ("ws", C.c_void_p), ("loss_out", C.c_void_p), ("exposure", C.POINTER(psl_exposure_args)),
                ("step0_params", C.c_int32)]


class psl_rows_args(C.Structure):
    _fields_ = [("format", C.c_int32), ("dtype", C.c_int32), ("heads", C.c_int32), ("dim", C.c_int32), ("group", C.c_int32),
                ("rows_bits", C.c_int32), ("n", C.c_int64), ("capacity", C.c_int64), ("first", C.c_int64),
                ("rows", C.c_void_p), ("values", C.c_void_p), ("value_row_stride", C.c_int64),
                ("value_head_stride", C.c_int64), ("codes", C.c_void_p), ("codes_row_stride", C.c_int64),
                ("scales", C.c_void_p), ("scales_row_stride", C.c_int64), ("owner", C.c_void_p)]


class psl_draw_args(C.Structure):
    _fields_ = [("n_rows", C.c_int32), ("n_cols", C.c_int32), ("n_draws", C.c_int32), ("dtype", C.c_int32),
                ("scores", C.c_void_p), ("score_stride", C.c_int64), ("mask", C.c_void_p), ("mask_stride", C.c_int64),
                ("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p), ("min_p", C.c_void_p),
                ("temperature_all", C.c_double), ("top_p_all", C.c_double), ("min_p_all", C.c_double),
                ("top_k_all", C.c_int32), ("reserved", C.c_int32), ("u", C.c_void_p), ("u_stride", C.c_int64),
                ("idx", C.c_void_p), ("prob", C.c_void_p), ("ws", C.c_void_p), ("ws_bytes", C.c_int64)]


# psl_dtype, psl_row_format
F32, BF16, F16 = 0, 1, 2
ROWS_INT8, ROWS_E4M3, ROWS_INT4 = 0, 1, 2

# psl_render_flags
STAGE_COLOR, PTS_GRAD, PARAM_GRAD, FEAT_GRAD, NO_SIGMOID, HAS_AFFINE = 1, 2, 4, 8, 16, 32

_SIGS = {
    "psl_create": (C.c_int, [C.c_int, C.POINTER(psl_config), C.POINTER(C.c_void_p)]),
    "psl_destroy": (None, [C.c_void_p]),
    "psl_last_error": (C.c_char_p, []),
    "psl_abi_version": (C.c_int, []),
    "psl_param_count": (C.c_int, []),
    "psl_param_color_count": (C.c_int, []),
    "psl_param_entry": (C.c_int, [C.c_int, C.c_char_p, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int),
                                  C.POINTER(C.c_int)]),
    "psl_param_master_floats": (C.c_int, []),
    "psl_points_reset": (C.c_int, [C.c_void_p]),
    "psl_points_append": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]),
    "psl_points_truncate": (C.c_int, [C.c_void_p, C.c_int]),
    "psl_points_count": (C.c_int, [C.c_void_p]),
    "psl_points_download": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]),
    "psl_points_download_range": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p]),
    "psl_index_build": (C.c_int, [C.c_void_p, C.c_void_p]),
    "psl_knn": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_float, C.c_int, C.c_void_p, C.c_void_p,
                          C.c_void_p, C.c_void_p]),
    "psl_dedupe_count": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_float, C.c_int, C.c_int, C.c_void_p, C.c_void_p]),
    "psl_dedupe_blocks": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p]),
    "psl_comm_unique_id": (C.c_int, [C.c_void_p]),
    "psl_selftest_traffic": (C.c_int, [C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]),
    "psl_pose_const_speed": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "psl_comm_reserve": (C.c_int, [C.c_void_p, C.c_int]),
    "psl_comm_init": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int]),
    "psl_comm_destroy": (C.c_int, [C.c_void_p]),
    "psl_allgather_new_points": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int,
                                           C.POINTER(C.c_int32), C.c_void_p]),
    "psl_allgather_decide": (C.c_int, [C.POINTER(C.c_int32), C.c_int, C.POINTER(C.c_int32), C.POINTER(C.c_longlong), C.POINTER(C.c_int)]),
    "psl_selftest_math": (C.c_int, [C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]),
    "psl_frame_radii": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_float, C.c_float, C.c_float, C.c_void_p,
                                  C.c_void_p, C.c_void_p, C.c_void_p]),
    "psl_topgrad_select_sync": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                          C.c_int, C.c_int, C.c_float, C.c_void_p, C.POINTER(C.c_int), C.c_void_p]),
    "psl_keyframe_overlap_sync": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.POINTER(C.c_float),
                                            C.c_int, psl_cam_intr, C.c_float, C.POINTER(C.c_float), C.c_void_p]),
    "psl_image_metrics_sync": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                         C.POINTER(C.c_double), C.c_void_p]),
    "psl_near_pcl_hits": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int,
                                    C.c_float, C.c_void_p, C.c_void_p]),   # ctx o d n z_steps step_row n_steps r hits stream
    "psl_add_points_sync": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_float, C.c_int,
                                      C.c_float, C.c_float, C.c_void_p, C.POINTER(C.c_int), C.c_void_p]),
    "psl_render_ws_floats": (C.c_int64, [C.c_int, C.c_int]),
    "psl_render_fwd": (C.c_int, [C.c_void_p, C.POINTER(psl_render_args), C.c_void_p]),
    "psl_render_bwd": (C.c_int, [C.c_void_p, C.POINTER(psl_render_args), C.POINTER(psl_render_grads), C.c_void_p]),
    "psl_composite_fwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_float, C.c_void_p, C.c_void_p, C.c_void_p,
                                    C.c_void_p, C.c_void_p]),
    "psl_adam_step": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_float,
                                C.c_float, C.c_float, C.c_float, C.c_int, C.c_void_p]),
    "psl_adam_step_rows": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                     C.c_float, C.c_float, C.c_float, C.c_float, C.c_int, C.c_void_p]),
    "psl_track_ws_floats": (C.c_int64, [C.c_int]),
    "psl_track_iters": (C.c_int, [C.c_void_p, C.POINTER(psl_track_args), C.c_void_p]),
    "psl_map_ws_floats": (C.c_int64, [C.c_int, C.c_int]),
    "psl_map_iters": (C.c_int, [C.c_void_p, C.POINTER(psl_map_args), C.c_void_p]),
    "psl_frustum_select_sync": (C.c_int, [C.c_void_p, C.POINTER(C.c_float), psl_cam_intr, C.c_void_p, C.c_float,
                                          C.c_float, C.c_void_p, C.c_void_p, C.POINTER(C.c_int), C.c_void_p]),
    "psl_rows_write": (C.c_int, [C.POINTER(psl_rows_args), C.c_void_p]),
    "psl_rows_read": (C.c_int, [C.POINTER(psl_rows_args), C.c_void_p]),
    "psl_draw_ws_bytes": (C.c_int64, [C.c_int32, C.c_int32]),
    "psl_draw_call_ws_bytes": (C.c_int64, [C.POINTER(psl_draw_args)]),
    "psl_draw_indices": (C.c_int, [C.POINTER(psl_draw_args), C.c_void_p]),
    "psl_sync": (C.c_int, [C.c_void_p, C.c_void_p]),
    "psl_profile_enable": (C.c_int, [C.c_void_p, C.c_int]),
    "psl_knn_candidates": (C.c_int64, [C.c_void_p]),
    "psl_debug_option": (C.c_int, [C.c_char_p, C.c_int]),
    "psl_profile_classes": (C.c_int, []),
    "psl_profile_read": (C.c_int, [C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_int), C.POINTER(C.c_double), C.c_int]),
    "psl_profile_name": (C.c_char_p, [C.c_int]),
}

EXPORTED_SYMBOLS = tuple(_SIGS.keys())
_lib = None


def lib():
    """Load the shared library (once).  Raises PslError when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise PslError(f"{LIB_PATH} not found: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                           "(there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        missing = []
        for name, (res, args) in _SIGS.items():
            try:
                fn = getattr(L, name)   # AttributeError if the symbol is missing
            except AttributeError:
                if os.environ.get("PSL_LIB"):     # an older build loaded for an A/B run: newer entry points are absent
                    missing.append(name)
                    continue
                raise
            fn.restype = res
            fn.argtypes = args
        ver = int(L.psl_abi_version())
        if ver != ABI_VERSION or missing:
            # struct layouts and signatures belong to ONE ABI version: a silent mismatch measures garbage
            msg = (f"{LIB_PATH}: psl_abi_version() = {ver}, this binding is ABI {ABI_VERSION}"
                   + (f"; entry points absent from the library: {', '.join(missing)}" if missing else ""))
            if not os.environ.get("PSL_LIB") or os.environ.get("PSL_LIB_ALLOW_ABI_MISMATCH") != "1":
                raise PslError(msg + " (an A/B run of an older build: set PSL_LIB_ALLOW_ABI_MISMATCH=1 once the struct layouts "
                                     "of the calls it makes are known to be unchanged)")
            import sys
            print("[point_slam_amd._lib] WARNING " + msg, file=sys.stderr, flush=True)
        _lib = L
    return _lib


def check(rc: int, what: str = ""):
    if rc < 0:
        msg = lib().psl_last_error().decode()
        raise PslError(f"{what or 'psl call'} failed ({rc}): {msg}")
    return rc


def ptr(t):
    """data_ptr of a torch tensor (or None)."""
    if t is None:
        return None
    return C.c_void_p(t.data_ptr())


def stream_ptr():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def call_on(device, entry: str, args):
    """entry(args, the current stream of `device`) with that device current: tensors may live on another device than the
    current one.  The raw stream is asked for directly; a torch.cuda.Stream object per call costs as much as a launch."""
    import torch
    fn = getattr(lib(), entry)
    here = torch.cuda.current_device()
    if device.index is None or device.index == here:
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        stream = raw(here) if raw is not None else torch.cuda.current_stream().cuda_stream
        return check(fn(C.byref(args), stream), entry)
    with torch.cuda.device(device):
        return check(fn(C.byref(args), torch.cuda.current_stream().cuda_stream), entry)
