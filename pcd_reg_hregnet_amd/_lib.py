"""ctypes binding of ``libhregnet_amd.so`` (the C ABI in include/hregnet_amd.h).

The HIP library is the product path: there is no CPU or PyTorch fallback.
If the library is missing or no GPU is visible, every op raises.
``torch`` is imported first so the process shares PyTorch's HIP runtime
(libamdhip64.so.7) with the library; tensors pass as raw device pointers and
work is enqueued on PyTorch's current stream.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import switches

_HERE = os.path.dirname(os.path.abspath(__file__))
# HREG_LIB: an alternative build of the same library (A/B timing experiments only)
LIB_PATH = os.environ.get("HREG_LIB") or os.path.join(_HERE, "libhregnet_amd.so")

HREG_OK = 0
HREG_STATUS_FPS_TIMEOUT = 1
_ERRORS = {1: "invalid argument", 2: "kernel launch failed", 3: "unsupported shape"}

HREG_EPI_AFFINE = 0
HREG_EPI_COSINE = 1
HREG_HEAD_SOFTPLUS = 0
HREG_HEAD_SIGMOID = 1
HREG_TWIST_UNIFORM = 0
HREG_TWIST_GAUSSIAN = 1
HREG_TWIST_INVERSE_GAUSSIAN = 2
HREG_REDUCE_NONE = 0
HREG_REDUCE_MEAN = 1
HREG_REDUCE_SUM = 2
MAX_SEGS = 4

_vp = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64


class Seg(ctypes.Structure):
    _fields_ = [("base", _vp), ("gather", _vp), ("rowscale", _vp), ("batch_stride", _i64),
                ("ld", _i), ("k0", _i), ("kc", _i), ("row_div", _i)]


class Gemm(ctypes.Structure):
    _fields_ = [("seg", Seg * MAX_SEGS), ("nseg", _i), ("R", _i), ("N", _i), ("K", _i),
                ("batch", _i), ("ldw", _i), ("w_batch_stride", _i64), ("W", _vp),
                ("scale", _vp), ("shift", _vp), ("relu", _i), ("epi", _i), ("rnorm", _vp),
                ("cnorm", _vp), ("rnorm_batch_stride", _i64), ("cnorm_batch_stride", _i64),
                ("out", _vp), ("ldo", _i), ("out_batch_stride", _i64),
                ("add", Seg * 2), ("nadd", _i)]


_u32 = ctypes.c_uint32
_u64 = ctypes.c_uint64
TOK_F32, TOK_BF16 = 0, 1
TOK_MAX_BUCKETS, TOK_MAX_THRESH, TOK_MAX_DISTANCE = 128, 64, 1024


class TokAttn(ctypes.Structure):
    # (the header's stride arrays as scalars: setting them takes a tenth of the time)
    _fields_ = [("dtype", _i), ("B", _i), ("Nq", _i), ("Nk", _i), ("H", _i), ("Hk", _i), ("D", _i),
                ("causal", _i), ("align_end", _i), ("scale", ctypes.c_float), ("q", _vp), ("k", _vp),
                ("v", _vp), ("out", _vp),
                *((f"{t}_{d}", _i64) for t in ("qs", "ks", "vs", "os") for d in "bnh"),
                ("lse", _vp), ("out_rest", _vp), ("q_len", _vp), ("k_len", _vp), ("key_mask", _vp),
                ("mask_sb", _i64), ("bias", _vp), ("bias_dtype", _i), ("num_buckets", _i),
                ("max_distance", _i), ("both", _i), ("nthresh", _i),
                ("thresh", ctypes.c_int32 * TOK_MAX_THRESH), ("dout", _vp),
                ("dos_b", _i64), ("dos_n", _i64), ("dos_h", _i64),
                ("dq", _vp), ("dk", _vp), ("dv", _vp), ("dbias", _vp), ("ws", _vp),
                ("ws_bytes", ctypes.c_size_t)]


class TokBlock(ctypes.Structure):
    _fields_ = [("dtype", _i), ("param_dtype", _i), ("R", _i), ("C", _i), ("gate_rows", _i),
                ("post", _i), ("pre", _i), ("scale", ctypes.c_float), ("eps", ctypes.c_float),
                ("step", _u32), ("site", _u32), ("seed", _u64), ("seed_dev", _vp), ("x", _vp),
                ("f", _vp), ("gate", _vp), ("post_w", _vp), ("post_b", _vp), ("pre_w", _vp),
                ("pre_b", _vp), ("y", _vp), ("h", _vp), ("stats", _vp), ("dy", _vp), ("dh", _vp),
                ("dx", _vp), ("df", _vp), ("dgate", _vp), ("dpost_w", _vp), ("dpost_b", _vp),
                ("dpre_w", _vp), ("dpre_b", _vp), ("ws", _vp), ("ws_bytes", ctypes.c_size_t)]


_SIGS = {
    "hreg_tok_attn_fwd": [ctypes.POINTER(TokAttn), _vp],
    "hreg_tok_attn_bwd": [ctypes.POINTER(TokAttn), _vp],
    "hreg_tok_dropout": [_vp, _vp, _i64, _i, _u32, _u64, _vp, _u32, _vp],
    "hreg_tok_block_fwd": [ctypes.POINTER(TokBlock), _vp],
    "hreg_tok_block_bwd": [ctypes.POINTER(TokBlock), _vp],
    "hreg_furthest_point_sampling": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_fps_bounded": [_i, _i, _i, _vp, _vp, _vp, _vp, _i, _vp],
    "hreg_weighted_furthest_point_sampling": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_gather_points": [_i, _i, _i, _i, _vp, _vp, _vp, _vp],
    "hreg_gather_points_grad": [_i, _i, _i, _i, _vp, _vp, _vp, _vp],
    "hreg_knn_points": [_vp, _vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_knn_gather": [_vp, _vp, _i, _i, _i, _i, _i, _vp, _vp],
    "hreg_knn_group": [_vp, _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp],
    "hreg_spatial_index": [_vp, _i, _i, _vp, _vp],
    "hreg_knn_group_indexed": [_vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp],
    "hreg_gemm": [ctypes.POINTER(Gemm), _vp],
    "hreg_gemm6": [ctypes.POINTER(Gemm), _vp],
    "hreg_gemm_grouped": [ctypes.POINTER(Gemm), _i, _vp],
    "hreg_attend": [_vp, _i, _i, _i, _i, _vp, _vp, _vp, _i, _i, _vp, _i, _vp, _vp, _vp],
    "hreg_group_max": [_vp, _i, _i, _i, _i, _vp, _i, _vp],
    "hreg_head_out": [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_row_norms": [_vp, _i, _i, _i, _vp, _vp],
    "hreg_sim_gather": [_vp, _i, _i, _i, _vp, _i, _vp, _vp, _i, _vp],
    "hreg_pair_feats": [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _vp, _i, _vp, _vp,
                        _vp],
    "hreg_weighted_svd": [_vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_weighted_svd_grouped": [_vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_fps_indexed": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_fps_indexed_lean": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_weighted_svd_tr": [_vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp],
    "hreg_transform_points": [_vp, _vp, _vp, _i, _i, _vp, _vp],
    "hreg_transformation_loss": [_vp, _vp, _vp, _vp, _i, ctypes.c_float, _vp, _vp, _vp, _vp, _vp,
                                 _vp],
    "hreg_group_l1_6": [_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp],
    "hreg_group_l1_6g": [_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp],
    "hreg_group6_l2": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group6_l3": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_split6_l2": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_split6_l3": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_split6j_l3": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_fine_head": [_vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_fine_head_table_floats": [_i],
    "hreg_nbr_head": [_vp, _vp, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_fine_head6": [_vp, _i, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_nbr_head6": [_vp, _vp, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_nbr_head6s": [_vp, _vp, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_head6_table_floats": [_i],
    "hreg_corr_head6_table_floats": [_i],
    "hreg_coarse_head6": [_vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_corr_head6": [_vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp],
    "hreg_corr_head6x": [_vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _vp],
    "hreg_nbr_head6sx": [_vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _vp],
    "hreg_mlp_head": [_vp, _i, _vp, _i, _i, _i, _i, _vp, _vp, _vp],
    "hreg_mlp_head_table_floats": [_i],
    "hreg_mlp_head6": [_vp, _i, _vp, _i, _i, _i, _i, _vp, _vp, _vp],
    "hreg_mlp_head6x": [_vp, _i, _vp, _i, _i, _i, _i, _vp, _vp, _i, _vp],
    "hreg_mlp_head6_table_floats": [_i],
    "hreg_sigma_weights": [_vp, _i, _i, _vp, _vp],
    "hreg_se3_exp": [_vp, _i, _vp, _vp],
    "hreg_se3_log": [_vp, _i, _vp, _vp],
    "hreg_twists_from_samples": [_vp, _vp, _i, _i, _vp, _vp],
    "hreg_perturb_clouds": [_vp, _vp, _i, _i, _vp, _vp, _vp, _vp],
    "hreg_range_filter": [_vp, _vp, _i, _i, ctypes.c_float, _vp, _vp, _vp, _vp],
    "hreg_chamfer": [_vp, _vp, _i, _i, _i, ctypes.c_float, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_js_loss": [_vp, _vp, _i, _vp, _vp, _vp, _vp],
    "hreg_rowdot": [_vp, _i, _i, _vp, _vp, _i, _vp, _vp],
    "hreg_rowdot_bwd": [_vp, _vp, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_relu_bwd": [_vp, _vp, ctypes.c_size_t, _vp, _vp],
    "hreg_debug_fps_stamps": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_debug_fps_floor": [_i, _i, _vp, _vp, _vp, _vp],
    "hreg_debug_wfps_floor": [_i, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_debug_fps_cluster": [_i, _i, _i, _vp, _vp, _vp, _vp, _i, ctypes.c_uint, _vp],
    "hreg_device_status": [ctypes.POINTER(ctypes.c_int), _i],
    "hreg_bn_stats": [_vp, _i, _i, ctypes.c_float, _vp, _vp, _vp, _vp, _vp],
    "hreg_bn_apply": [_vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp],
    "hreg_bn_backward": [_vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _vp],
    "hreg_bn_running_update": [_vp, _vp, _i, ctypes.c_float, _vp, _vp, _vp],
    "hreg_col_sum": [_vp, _i, _i, _vp, _vp, _i, _vp],
    "hreg_gemm_tn": [_vp, _i, _vp, _i, _i, _i, _i, ctypes.c_float, _vp, _vp, _vp],
    "hreg_debug_gemm_tn_s": [_vp, _i, _vp, _i, _i, _i, _i, ctypes.c_float, _vp, _vp, _vp, _i],
    "hreg_ts_gemm_supported": [_i, _i, _i, _i],
    "hreg_ts_gemm": [_vp, _i, _i, _i, _vp, _i, _i, _vp, _vp, _i, _vp, _i, _vp],
    "hreg_copy_many": [_i, _vp, _vp, _vp, _vp],
    "hreg_ts_gemm_split_out": [_vp, _i, _i, _i, _vp, _i, _i, _vp, _i, _i, _vp, _i, _i, _vp, _i, _vp],
    "hreg_ts_gemm_bn_tail": [_vp, _i, _vp, _i, _vp, _i, _i, _vp, _i, _vp, _vp, _i, ctypes.c_float, ctypes.c_float,
                             _vp, _vp, _vp, _vp,
                             _vp, _vp, _vp],
    "hreg_gemm_tn_tail": [_vp, _i, _vp, _i, _vp, _i, _vp, _i, _i, _i, ctypes.c_float, _vp, _vp, _vp],
    "hreg_ts_gemm_bn": [_vp, _i, _i, _i, _vp, _i, _i, _vp, _vp, _i, ctypes.c_float, ctypes.c_float, _vp,
                        _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_ts_gemm_pre_supported": [_i, _i, _i],
    "hreg_ts_gemm_bn_pre": [_vp, _i, _i, _i, _vp, _i, _vp, _vp, _i, ctypes.c_float, ctypes.c_float, _vp,
                            _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp],
    "hreg_gemm_tn_pre": [_vp, _i, _vp, _i, _i, _i, _i, ctypes.c_float, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp],
    "hreg_transpose": [_vp, _i, _i, _vp, _vp],
    "hreg_add_into": [_vp, _vp, ctypes.c_size_t, _vp],
    "hreg_adam_step": [_vp, _vp, _vp, _vp, ctypes.c_size_t, ctypes.c_float, ctypes.c_float,
                       ctypes.c_float, ctypes.c_float, _i, _vp],
    "hreg_adam_step_dev": [_vp, _vp, _vp, _vp, ctypes.c_size_t, ctypes.c_float, ctypes.c_float,
                           ctypes.c_float, ctypes.c_float, _vp, _vp],
    "hreg_copy_rows": [_vp, _i, _i, _i, _i, _vp, _i, _i, _vp],
    "hreg_group_sum": [_vp, _i, _i, _i, _i, _vp, _i, _i, _vp],
    "hreg_gather_rows": [_vp, _i, _vp, _i, _i, _vp, _i, _vp],
    "hreg_csr_build": [_vp, _i, _i, _vp, _vp],
    "hreg_scatter_rows": [_vp, _i, _vp, _i, _i, _i, _vp, _i, _i, _vp],
    "hreg_geom_rows": [_vp, _vp, _i, _i, _vp, _i, _vp],
    "hreg_geom_rows_bwd": [_vp, _i, _vp, _i, _vp, _i, _i, _vp, _vp, _vp],
    "hreg_attention_fwd": [_vp, _i, _i, _vp, _i, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp,
                           _i, _vp],
    "hreg_attention_bwd": [_vp, _i, _i, _vp, _i, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp,
                           _i, _i, _vp, _i, _vp, _i, _vp, _vp],
    "hreg_group_max_arg": [_vp, _i, _i, _i, _i, _vp, _i, _vp, _vp],
    "hreg_attention_fwd_pre": [_vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp],
    "hreg_attention_bwd_pre": [_vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _i, _vp,
                               _i, _vp, _vp],
    "hreg_group_max_arg_pre": [_vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_max_bwd": [_vp, _i, _vp, _i, _i, _i, _vp, _i, _i, _vp],
    "hreg_head_out_bwd": [_vp, _i, _i, _vp, _vp, _vp, _i, _i, _vp, _vp, _i, _vp],
    "hreg_sim_stats": [_vp, _i, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_sim_feats": [_vp, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _i, _vp],
    "hreg_sim_feats_bwd": [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp,
                           _vp, _i, _vp, _vp, _vp, _vp],
    "hreg_weighted_svd_bwd": [_vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_transform_points_bwd": [_vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_compose_se3": [_i, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_compose_se3_bwd": [_i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hreg_transformation_loss_bwd": [_vp, _vp, _vp, _vp, _i, ctypes.c_float, ctypes.c_float, _vp,
                                     _vp, _vp, _vp],
    "hreg_index_offset": [_vp, _i, _i, _i, _vp, _vp],
    "hreg_calib_metrics": [_vp, _vp, _i, _vp, _vp, _vp],
    "hreg_icp_init": [_vp, _vp, _i, _i, _i, _vp, _vp, _vp],
    "hreg_icp_iterate": [_vp, _i, _i, _i, ctypes.c_float, ctypes.c_double, ctypes.c_double, _i, _i,
                         _vp, _vp],
    "hreg_icp_result": [_vp, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp],
}

# the fp32-MFMA twins of the level kernels: test checkers in libhregnet_checkers.so
# (include/hregnet_amd_checkers.h), loaded only when a checker is called
_CHECKER_SIGS = {
    "hreg_group_l1": [_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp],
    "hreg_group_l2": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_l3": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_split_l2": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    "hreg_group_split_l3": [_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp],
}
_CHECKER_TABLES = ("hreg_group_l1_table_floats", "hreg_group_l2_table_floats",
                   "hreg_group_l3_table_floats", "hreg_group_split_l2_table_floats",
                   "hreg_group_split_l3_table_floats")
CHECKER_EXPORTS = tuple(_CHECKER_SIGS) + _CHECKER_TABLES
CHECKER_PATH = os.path.join(_HERE, "libhregnet_checkers.so")

EXPORTS = tuple(_SIGS) + ("hreg_version", "hreg_spatial_index_bytes", "hreg_col_reduce_ws_bytes",
                          "hreg_gemm_tn_ws_bytes", "hreg_csr_ws_bytes", "hreg_ts_gemm_bn_ws_bytes",
                          "hreg_sim_feats_bwd_ws_bytes",
                          "hreg_nbr_head_table_floats", "hreg_group6_l2_table_floats",
                          "hreg_group6_l3_table_floats", "hreg_group_l1_6_table_floats",
                          "hreg_group_split6_l2_table_floats", "hreg_group_split6_l3_table_floats",
                          "hreg_coarse_head6_table_floats", "hreg_icp_ws_bytes",
                          "hreg_tok_attn_ws_bytes", "hreg_tok_block_ws_bytes")

_lib = None
_checkers = None


def load_checkers(require_gpu: bool = True):
    """The test-only checker library (fp32-MFMA level kernels); raises if it is not built."""
    global _checkers
    load(require_gpu)  # the product library first: one HIP runtime, one set of streams
    if _checkers is None:
        if not os.path.exists(CHECKER_PATH):
            raise RuntimeError(f"{CHECKER_PATH} not found: build it with "
                               "`python -m pcd_reg_hregnet_amd.build` (test checkers only)")
        L = ctypes.CDLL(CHECKER_PATH)
        for name, args in _CHECKER_SIGS.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = ctypes.c_int
        for name in _CHECKER_TABLES:
            getattr(L, name).restype = ctypes.c_int
            getattr(L, name).argtypes = []
        _checkers = L
    return _checkers


def load(require_gpu: bool = True):
    """Load the library (and check a GPU is visible unless require_gpu=False)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} not found: build it with `python -m pcd_reg_hregnet_amd.build` "
                "(hipcc --offload-arch=gfx950); there is no CPU fallback")
        L = ctypes.CDLL(LIB_PATH)
        for name, args in _SIGS.items():
            if os.environ.get("HREG_LIB") and not hasattr(L, name):
                # an A/B build of an older tree (HREG_LIB, timing only) may predate newer
                # entries: they raise when called; the product library must export them all
                continue
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = ctypes.c_int
        L.hreg_version.restype = ctypes.c_char_p
        L.hreg_version.argtypes = []
        L.hreg_spatial_index_bytes.restype = ctypes.c_size_t
        L.hreg_spatial_index_bytes.argtypes = [ctypes.c_int, ctypes.c_int]
        L.hreg_col_reduce_ws_bytes.restype = ctypes.c_size_t
        L.hreg_col_reduce_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int]
        L.hreg_gemm_tn_ws_bytes.restype = ctypes.c_size_t
        L.hreg_gemm_tn_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int]
        L.hreg_csr_ws_bytes.restype = ctypes.c_size_t
        L.hreg_csr_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int]
        L.hreg_sim_feats_bwd_ws_bytes.restype = ctypes.c_size_t
        L.hreg_sim_feats_bwd_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int]
        L.hreg_icp_ws_bytes.restype = ctypes.c_size_t
        L.hreg_icp_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int]
        L.hreg_ts_gemm_bn_ws_bytes.restype = ctypes.c_size_t
        L.hreg_ts_gemm_bn_ws_bytes.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int]
        L.hreg_tok_attn_ws_bytes.restype = ctypes.c_size_t
        L.hreg_tok_attn_ws_bytes.argtypes = [ctypes.POINTER(TokAttn), ctypes.c_int]
        L.hreg_tok_block_ws_bytes.restype = ctypes.c_size_t
        L.hreg_tok_block_ws_bytes.argtypes = [ctypes.POINTER(TokBlock)]
        for name in ("hreg_nbr_head_table_floats", "hreg_group6_l2_table_floats", "hreg_group6_l3_table_floats",
                     "hreg_group_l1_6_table_floats", "hreg_group_split6_l2_table_floats",
                     "hreg_group_split6_l3_table_floats", "hreg_coarse_head6_table_floats"):
            getattr(L, name).restype = ctypes.c_int
            getattr(L, name).argtypes = []
        _lib = L
    if require_gpu and not torch.cuda.is_available():
        raise RuntimeError("pcd_reg_hregnet_amd: no GPU visible; the HIP path has no CPU fallback")
    return _lib


def ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def stream_handle() -> int:
    return torch.cuda.current_stream().cuda_stream


# timing probe (tools/train_probe.sh only): the entries named in HREG_SWITCHES=PROBE_TWICE=a+b
# run twice per call, so a run's extra wall time is that kernel family's cost under the step's
# stream overlap (results change -- accumulating entries add twice -- so no test sets it, and
# bench.py refuses to report a measurement with it set)
_TWICE = frozenset(filter(None, switches.text("PROBE_TWICE").split("+")))


def call(name: str, *args) -> None:
    L = load_checkers() if name in _CHECKER_SIGS else load()
    conv = []
    for a in args:
        if isinstance(a, torch.Tensor):
            conv.append(a.data_ptr())
        else:
            conv.append(a)
    rc = getattr(L, name)(*conv)
    if rc == HREG_OK and name in _TWICE:
        rc = getattr(L, name)(*conv)
    if rc != HREG_OK:
        raise RuntimeError(f"{name} failed: {_ERRORS.get(rc, rc)} (code {rc})")


def device_status(clear: bool = True) -> int:
    """HREG_STATUS_* bits raised by kernels since the last clear (synchronous)."""
    L = load()
    v = ctypes.c_int(0)
    rc = L.hreg_device_status(ctypes.byref(v), 1 if clear else 0)
    if rc != HREG_OK:
        raise RuntimeError(f"hreg_device_status failed: {_ERRORS.get(rc, rc)} (code {rc})")
    return v.value


def gemm(g: Gemm) -> None:
    L = load()
    rc = L.hreg_gemm(ctypes.byref(g), stream_handle())
    if rc != HREG_OK:
        raise RuntimeError(f"hreg_gemm failed: {_ERRORS.get(rc, rc)} (code {rc})")


def gemm_grouped(gs) -> None:
    """hreg_gemm_grouped: independent GEMMs (a list of Gemm, no addends) in one launch."""
    L = load()
    arr = (Gemm * len(gs))(*gs)
    rc = L.hreg_gemm_grouped(arr, len(gs), stream_handle())
    if rc != HREG_OK:
        raise RuntimeError(f"hreg_gemm_grouped failed: {_ERRORS.get(rc, rc)} (code {rc})")


def gemm6(g: Gemm) -> None:
    """hreg_gemm6: the same GEMM with bf16x6 products on the bf16 matrix cores."""
    L = load()
    rc = L.hreg_gemm6(ctypes.byref(g), stream_handle())
    if rc != HREG_OK:
        raise RuntimeError(f"hreg_gemm6 failed: {_ERRORS.get(rc, rc)} (code {rc})")
