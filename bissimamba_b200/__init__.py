"""bissimamba_b200 -- B200-native k-mamba scanND / convND hot path.

The product is the C-ABI shared library ``libkmamba_b200.so`` (declared in
``include/scan_nd.h`` and ``include/convnd.h``).  This module only binds it
with ctypes, mirroring the reference's C interface (``ScanNDParams``,
``scannd()``, ``om_scannd_forward/backward``, ``ConvNDParams``, ``convnd()``)
so Python callers and the tests use the same entry points a C caller links.

There is no CPU fallback: if the library is missing, ``lib()`` raises.
"""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libkmamba_b200.so")

_f = C.POINTER(C.c_float)
_l = C.POINTER(C.c_long)


class ScanNDParams(C.Structure):
    """Same field order and types as the reference include/scan_nd.h:40-69."""
    _fields_ = [
        ("max_ndims", C.c_long), ("max_state", C.c_long), ("use_fast_exp", C.c_int),
        ("dims", _l), ("ndims", C.c_long), ("D", C.c_long), ("M", C.c_long),
        ("x", C.c_void_p), ("A", C.c_void_p), ("B", C.c_void_p), ("C", C.c_void_p),
        ("delta", C.c_void_p), ("h", C.c_void_p), ("y", C.c_void_p),
        ("theta", C.c_void_p), ("lambda_", C.c_void_p),
        ("default_lambda", C.c_float), ("use_a_log_clamp", C.c_int), ("a_log_min", C.c_float),
        ("dA", C.c_void_p), ("dB", C.c_void_p), ("dC", C.c_void_p), ("ddelta", C.c_void_p),
        ("dlambda", C.c_void_p), ("dtheta", C.c_void_p),
    ]


class ConvNDParams(C.Structure):
    """Same layout as the reference include/convnd.h:10-23."""
    _fields_ = [
        ("input", C.c_void_p), ("kernel", C.c_void_p), ("bias", C.c_void_p),
        ("output", C.c_void_p), ("dy", C.c_void_p), ("dinput", C.c_void_p),
        ("dkernel", C.c_void_p), ("dbias", C.c_void_p), ("dims", _l),
        ("ndims", C.c_long), ("D", C.c_long), ("K", C.c_long),
    ]


class KMBlockScanParams(C.Structure):
    """include/kmamba_block.h"""
    _fields_ = [("ndims", C.c_long), ("dims", _l), ("L", C.c_long), ("N", C.c_long), ("R", C.c_long),
                ("u", C.c_void_p), ("dt", C.c_void_p), ("lambda_", C.c_void_p), ("B", C.c_void_p),
                ("C", C.c_void_p), ("A_log", C.c_void_p), ("theta", C.c_void_p),
                ("default_lambda", C.c_float), ("use_fast_exp", C.c_int),
                ("h", C.c_void_p), ("Bu", C.c_void_p), ("y", C.c_void_p), ("inputs_bf16", C.c_int)]


class KMBlockScanGrads(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in ("dB", "dC", "du", "ddt", "dlambda", "dA_log", "dtheta")]


class KMBlockConfig(C.Structure):
    _fields_ = [("dim", C.c_long), ("N", C.c_long), ("R", C.c_long), ("ndims", C.c_long), ("dims", _l),
                ("L", C.c_long), ("dt_min", C.c_float), ("dt_max", C.c_float), ("default_lambda", C.c_float),
                ("use_fast_exp", C.c_int), ("bf16_storage", C.c_int)]


BLOCK_FIELDS = ("W_in", "W_out", "A_log", "W_B", "W_C", "delta_proj", "lambda_proj", "b_B", "b_C", "theta")


class KMBlockWeights(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in BLOCK_FIELDS]


class KMBlockGrads(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in BLOCK_FIELDS]


def block_config(dims, dim, N, R, dt_min=1e-3, dt_max=0.1, default_lambda=0.5, use_fast_exp=0, bf16=False):
    c = KMBlockConfig()
    darr = dims_array(dims)
    c._dims_keep = darr
    c.dim, c.N, c.R = int(dim), int(N), int(R)
    c.ndims = len(dims)
    c.dims = C.cast(darr, _l)
    L = 1
    for d in dims:
        L *= int(d)
    c.L = L
    c.dt_min, c.dt_max, c.default_lambda, c.use_fast_exp = dt_min, dt_max, default_lambda, use_fast_exp
    c.bf16_storage = int(bf16)
    return c


MAX_NDIMS = 32


class KMambaConfig(C.Structure):
    """Same layout as the reference include/kmamba.h:238-278."""
    _fields_ = [("max_ndims", C.c_long), ("max_state", C.c_long), ("use_fast_exp", C.c_int),
                ("vocab_size", C.c_size_t), ("dim", C.c_size_t), ("state_size", C.c_size_t),
                ("seq_len", C.c_size_t), ("n_layers", C.c_size_t), ("mimo_rank", C.c_size_t),
                ("dt_scale", C.c_float), ("dt_min", C.c_float), ("dt_max", C.c_float),
                ("default_lambda", C.c_float), ("use_a_log_clamp", C.c_int), ("a_log_min", C.c_float),
                ("spatial_ndims", C.c_long), ("spatial_dims", C.c_long * MAX_NDIMS),
                ("use_convnd", C.c_int), ("use_convnd_bias", C.c_int), ("convnd_K", C.c_long),
                ("convnd_ndims", C.c_long), ("pad_left", C.c_long * MAX_NDIMS), ("pad_right", C.c_long * MAX_NDIMS),
                ("d_conv", C.c_uint32), ("expand_factor", C.c_float), ("model_name", C.c_char * 64),
                ("vocab_data", C.c_void_p), ("gpu_device", C.c_int), ("weight_tying", C.c_int)]


class MBOptimConfig(C.Structure):
    _fields_ = [(k, C.c_float) for k in ("lr", "mu", "beta2", "eps", "clip_norm", "weight_decay")]


DTYPE_F32, DTYPE_BF16 = 0, 1


class KMBDeltaParams(C.Structure):
    """include/kmamba_delta.h"""
    _fields_ = [("batch", C.c_long), ("T", C.c_long), ("Hk", C.c_long), ("Hv", C.c_long), ("dk", C.c_long),
                ("dv", C.c_long), ("dtype", C.c_int), ("scale", C.c_float), ("cu_seqlens", C.c_void_p),
                ("n_seq", C.c_long), ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("g", C.c_void_p),
                ("beta", C.c_void_p), ("o", C.c_void_p), ("h0", C.c_void_p), ("hT", C.c_void_p),
                ("ld_q", C.c_long), ("ld_k", C.c_long), ("ld_v", C.c_long), ("ld_o", C.c_long)]


class KMBDeltaGrads(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("do_", "dhT", "dq", "dk", "dv", "dg", "dbeta", "dh0")] + \
               [(n, C.c_long) for n in ("ld_do", "ld_dq", "ld_dk", "ld_dv")]


class KMBNormParams(C.Structure):
    """include/kmamba_norm.h"""
    _fields_ = [("rows", C.c_long), ("D", C.c_long), ("dtype", C.c_int), ("eps", C.c_float)] + \
               [(n, C.c_void_p) for n in ("x", "residual", "total", "y", "w", "b", "mean", "rstd")] + \
               [(n, C.c_long) for n in ("ld_x", "ld_residual", "ld_total", "ld_y")]


class KMBNormGrads(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("dy", "dtotal", "dx", "dw", "db")] + \
               [(n, C.c_long) for n in ("ld_dy", "ld_dtotal", "ld_dx")] + [("accumulate", C.c_int)]


class KMBGradTensor(C.Structure):
    """include/kmamba_clip.h"""
    _fields_ = [("in_", C.c_void_p), ("out", C.c_void_p), ("n", C.c_longlong), ("dtype", C.c_int)]


CONVND_FORWARD, CONVND_BACKWARD, CONVND_COMPLETE = 1, 2, 3

# every symbol the public headers declare (checked by the CPU tests)
EXPORTS = [
    "scannd_validate", "scannd", "scannd_ref_with_plan", "om_scannd_forward", "om_scannd_backward",
    "scannd_batched", "scannd_backward_batched", "scannd_forward_async", "scannd_backward_async",
    "scannd_backward_ex", "kmb_last_backward_path",
    "convnd_kernel_volume", "convnd_forward_wavefront", "convnd_backward_wavefront", "convnd",
    "om_convnd_forward", "om_convnd_backward", "convnd_status", "convnd_batched_async",
    "convnd_backward_noalloc", "convnd_backward_noalloc_error",
    "wavefront_nd_validate_dims", "wavefront_nd_total_points", "wavefront_nd_max_level",
    "wavefront_nd_row_major_offset", "wavefront_nd_level_size", "wavefront_nd_for_level",
    "wavefront_nd_for_each_level", "km_wavefront_plan_create", "km_wavefront_plan_free",
    "km_wavefront_plan_matches_dims", "km_wavefront_plan_level_size", "km_wavefront_plan_level_offsets",
    "km_wavefront_plan_iter_forward", "km_wavefront_plan_iter_reverse",
    "kmb_last_error", "kmb_clear_error", "kmb_device_status", "kmb_last_forward_path", "kmb_set_force_generic",
    "kmb_set_scan_exp2", "kmb_get_scan_exp2", "kmb_init_tensor", "kmb_set_sm_reserve",
    "kmamba_distributed_split_batch", "kmamba_distributed_split_layers", "kmamba_distributed_init_nccl",
    "kmamba_distributed_fini_nccl", "kmamba_allreduce_gradients_nccl", "kmamba_broadcast_params_nccl",
    "kmb_dist_unique_id", "kmb_dist_init", "kmb_dist_exchange_id", "kmb_dist_world_size", "kmb_dist_rank",
    "kmb_dist_allreduce_async", "kmb_dist_allgather_async", "kmb_dist_broadcast_async", "kmb_dist_scannd_backward",
    "kmb_dist_convnd_backward", "kmb_dist_model_train_step",
    "kser_writer_create", "kser_writer_add_vocab", "kser_writer_add_tensor", "kser_writer_finalize", "kser_writer_free",
    "kser_reader_open", "kser_reader_config", "kser_reader_is_valid", "kser_reader_load_vocab", "kser_reader_load_tensor",
    "kser_reader_count_tensors", "kser_reader_get_tensor_info", "kser_reader_close", "kser_file_info", "kser_quantize",
    "kser_dequantize", "kser_dtype_size", "kser_sha256", "kmamba_save_ser", "kmamba_load_ser", "kmb_load_ser_ex",
    "kmamba_ser_info", "kmamba_save_checkpoint_ser", "kmamba_load_checkpoint_ser",
    "kmb_blockscan_forward", "kmb_blockscan_set_strips", "kmb_blockscan_last_forward_path", "kmb_blockscan_set_backward_strips",
    "kmb_blockscan_last_backward_path", "kmb_blockscan_backward", "kmb_blockscan_backward_ex", "kmb_block_activation_floats",
    "kmb_block_forward", "kmb_block_backward", "kmb_block_set_tensor_cores", "kmb_block_last_projection_path", "kmb_block_last_dx_path", "cuda_block_forward", "cuda_block_backward",
    "kmamba_config_set_defaults", "kmamba_optim_config_set_defaults", "kmamba_create", "kmamba_free",
    "kmamba_init", "kmamba_enable_training", "kmamba_forward", "kmamba_train_batch", "kmamba_train_step",
    "kmamba_get_config", "kmamba_step_count", "kmamba_update_lr", "kmamba_get_tensor", "kmamba_set_tensor",
    "kmb_model_forward_backward", "kmb_model_optimizer_step", "kmb_model_grad_arena", "kmb_model_param_arena", "kmb_model_tensor_offset",
    "kmb_delta_workspace_floats", "kmb_delta_forward", "kmb_delta_backward", "kmb_delta_step",
    "kmb_layernorm_forward", "kmb_layernorm_workspace_floats", "kmb_layernorm_backward",
    "kmb_grad_clip_workspace_floats", "kmb_grad_clip", "kmb_model_clip_gradients",
    "kmb_gemm_f32", "kmb_gemm_bf16", "kmb_gemm_set_f32_kind", "kmb_gemm_get_f32_kind", "kmb_gemm_set_f32_flush", "kmb_gemm_last_path",
]

_lib = None


def lib():
    """Load libkmamba_b200.so (build it first with ``bissimamba_b200.build``)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: run `python -m bissimamba_b200.build` "
                               "(there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        P = C.POINTER(ScanNDParams)
        Q = C.POINTER(ConvNDParams)
        for n in ("scannd_validate", "scannd", "om_scannd_forward", "om_scannd_backward"):
            getattr(L, n).argtypes = [P]
            getattr(L, n).restype = C.c_int
        L.scannd_batched.argtypes = [P, C.c_long]
        L.scannd_backward_batched.argtypes = [P, C.c_long, C.c_void_p]
        L.scannd_forward_async.argtypes = [P, C.c_long, C.c_void_p]
        L.scannd_backward_async.argtypes = [P, C.c_long, C.c_void_p, C.c_void_p]
        L.scannd_backward_ex.argtypes = [P, C.c_long, C.c_void_p, C.c_int, C.c_void_p]
        L.scannd_ref_with_plan.argtypes = [P, C.c_void_p]
        L.convnd.argtypes = [Q, C.c_int]
        L.convnd.restype = None
        L.convnd_batched_async.argtypes = [Q, C.c_long, C.c_int, C.c_void_p]
        L.om_convnd_forward.argtypes = [Q]
        L.convnd_backward_noalloc.argtypes = [Q, C.c_long, C.c_void_p]
        L.convnd_backward_noalloc_error.restype = C.c_char_p
        L.om_convnd_backward.argtypes = [Q]
        L.convnd_forward_wavefront.argtypes = [Q, C.c_void_p]
        L.convnd_forward_wavefront.restype = None
        L.convnd_backward_wavefront.argtypes = [Q, C.c_void_p]
        L.convnd_backward_wavefront.restype = None
        L.convnd_kernel_volume.argtypes = [C.c_long, C.c_long]
        L.convnd_kernel_volume.restype = C.c_long
        L.kmb_last_error.restype = C.c_char_p
        KC = C.POINTER(KMambaConfig)
        L.kmamba_config_set_defaults.argtypes = [KC]
        L.kmamba_config_set_defaults.restype = None
        L.kmamba_optim_config_set_defaults.argtypes = [C.POINTER(MBOptimConfig)]
        L.kmamba_optim_config_set_defaults.restype = None
        L.kmamba_create.argtypes = [KC]
        L.kmamba_create.restype = C.c_void_p
        L.kmamba_free.argtypes = [C.c_void_p]
        L.kmamba_free.restype = None
        L.kmamba_init.argtypes = [C.c_void_p, C.c_uint32]
        L.kmb_init_tensor.argtypes = [C.c_void_p, C.c_uint32, C.c_char_p, C.c_void_p, C.c_long]
        L.kmb_init_tensor.restype = C.c_long
        vp, sz = C.c_void_p, C.c_size_t
        L.kmamba_distributed_split_batch.argtypes = [vp, sz, sz]
        L.kmamba_distributed_split_batch.restype = None
        L.kmamba_distributed_split_layers.argtypes = [vp, sz, sz]
        L.kmamba_distributed_split_layers.restype = None
        L.kmamba_distributed_init_nccl.argtypes = [C.c_int, C.c_int]
        L.kmamba_distributed_init_nccl.restype = vp
        L.kmamba_distributed_fini_nccl.argtypes = [vp]
        L.kmamba_distributed_fini_nccl.restype = None
        L.kmamba_allreduce_gradients_nccl.argtypes = [vp, vp, sz]
        L.kmamba_broadcast_params_nccl.argtypes = [vp, vp, sz]
        L.kmb_dist_unique_id.argtypes = [vp]
        L.kmb_dist_init.argtypes = [vp, C.c_int, C.c_int, C.c_int]
        L.kmb_dist_init.restype = vp
        L.kmb_dist_exchange_id.argtypes = [vp, C.c_int, C.c_int, C.c_char_p, C.c_int]
        L.kmb_dist_world_size.argtypes = [vp]
        L.kmb_dist_rank.argtypes = [vp]
        L.kmb_dist_allreduce_async.argtypes = [vp, vp, sz, C.c_float, vp]
        L.kmb_dist_allgather_async.argtypes = [vp, vp, vp, sz, vp]
        L.kmb_dist_broadcast_async.argtypes = [vp, vp, sz, C.c_int, vp]
        L.kmb_dist_scannd_backward.argtypes = [vp, vp, C.c_long, vp, C.c_int, vp]
        L.kmb_dist_convnd_backward.argtypes = [vp, vp, C.c_long, vp]
        L.kmb_dist_model_train_step.argtypes = [vp, vp, vp, sz, sz, vp]
        L.kmb_dist_model_train_step.restype = C.c_float
        for fn in ("kser_writer_create", "kser_reader_open", "kser_reader_config", "kser_reader_load_tensor",
                   "kser_reader_get_tensor_info", "kmamba_load_ser", "kmb_load_ser_ex"):
            getattr(L, fn).restype = vp
        L.kser_writer_create.argtypes = [C.c_char_p, vp]
        L.kser_writer_add_vocab.argtypes = [vp, C.c_uint32, C.c_char_p, C.c_uint16]
        L.kser_writer_add_tensor.argtypes = [vp, C.c_char_p, vp, vp, C.c_int, C.c_int]
        L.kser_writer_finalize.argtypes = [vp]
        L.kser_writer_free.argtypes = [vp]
        L.kser_writer_free.restype = None
        L.kser_reader_open.argtypes = [C.c_char_p]
        L.kser_reader_config.argtypes = [vp]
        L.kser_reader_is_valid.argtypes = [vp]
        L.kser_reader_load_tensor.argtypes = [vp, C.c_char_p]
        L.kser_reader_count_tensors.argtypes = [vp]
        L.kser_reader_count_tensors.restype = C.c_uint64
        L.kser_reader_get_tensor_info.argtypes = [vp, C.c_uint64]
        L.kser_reader_close.argtypes = [vp]
        L.kser_reader_close.restype = None
        L.kser_quantize.argtypes = [vp, vp, C.c_uint64, C.c_int]
        L.kser_dequantize.argtypes = [vp, vp, C.c_uint64, C.c_int]
        L.kser_sha256.argtypes = [vp, sz, vp]
        L.kser_sha256.restype = None
        L.kmamba_save_ser.argtypes = [vp, C.c_char_p, C.c_int]
        L.kmamba_load_ser.argtypes = [C.c_char_p, C.c_int]
        L.kmb_load_ser_ex.argtypes = [C.c_char_p, C.c_int, vp]
        L.kmamba_enable_training.argtypes = [C.c_void_p, C.POINTER(MBOptimConfig), C.c_float, C.c_float]
        L.kmamba_forward.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        L.kmamba_train_batch.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t]
        L.kmamba_train_batch.restype = C.c_float
        L.kmamba_train_step.argtypes = [C.c_void_p, C.c_void_p]
        L.kmamba_train_step.restype = C.c_float
        L.kmamba_get_tensor.argtypes = [C.c_void_p, C.c_char_p]
        L.kmamba_get_tensor.restype = _f
        L.kmamba_set_tensor.argtypes = [C.c_void_p, C.c_char_p, C.c_void_p]
        L.kmamba_step_count.argtypes = [C.c_void_p]
        L.kmamba_step_count.restype = C.c_size_t
        L.kmamba_update_lr.argtypes = [C.c_void_p, C.c_float, C.c_float]
        L.kmamba_update_lr.restype = None
        ll = C.c_longlong
        L.kmb_gemm_f32.argtypes = [C.c_int, C.c_int, ll, ll, ll, vp, ll, vp, ll, vp, ll, C.c_int, vp]
        L.kmb_gemm_bf16.argtypes = [C.c_int, ll, ll, ll, vp, ll, vp, ll, vp, ll, C.c_int, vp]
        L.kmb_gemm_set_f32_kind.argtypes = [C.c_int]
        L.kmb_gemm_set_f32_flush.argtypes = [C.c_int]
        L.kmamba_get_config.argtypes = [C.c_void_p]
        L.kmamba_get_config.restype = KC
        L.kmb_model_forward_backward.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
        L.kmb_model_forward_backward.restype = C.c_float
        L.kmb_model_optimizer_step.argtypes = [C.c_void_p, C.c_void_p]
        L.kmb_model_grad_arena.argtypes = [C.c_void_p, C.POINTER(C.c_size_t)]
        L.kmb_model_grad_arena.restype = C.c_void_p
        L.kmb_model_tensor_offset.argtypes = [C.c_void_p, C.c_char_p, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]
        L.kmb_model_param_arena.argtypes = [C.c_void_p, C.POINTER(C.c_size_t)]
        L.kmb_model_param_arena.restype = C.c_void_p
        L.kmb_block_activation_floats.argtypes = [C.POINTER(KMBlockConfig), C.c_long]
        L.kmb_block_activation_floats.restype = C.c_size_t
        L.kmb_block_forward.argtypes = [C.POINTER(KMBlockConfig), C.POINTER(KMBlockWeights), C.c_void_p,
                                        C.c_void_p, C.c_long, C.c_void_p, C.c_void_p]
        L.kmb_block_backward.argtypes = [C.POINTER(KMBlockConfig), C.POINTER(KMBlockWeights), C.c_void_p,
                                         C.c_void_p, C.c_void_p, C.POINTER(KMBlockGrads), C.c_long, C.c_void_p,
                                         C.c_void_p]
        L.kmb_blockscan_forward.argtypes = [C.POINTER(KMBlockScanParams), C.c_long, C.c_void_p]
        L.kmb_blockscan_backward.argtypes = [C.POINTER(KMBlockScanParams), C.c_long, C.c_void_p,
                                             C.POINTER(KMBlockScanGrads), C.c_void_p]
        L.kmb_blockscan_backward_ex.argtypes = [C.POINTER(KMBlockScanParams), C.c_long, C.c_void_p,
                                                C.POINTER(KMBlockScanGrads), C.c_int, C.c_void_p]
        L.kmb_blockscan_set_backward_strips.argtypes = [C.c_int]
        L.kmb_blockscan_set_backward_strips.restype = None
        L.kmb_set_force_generic.argtypes = [C.c_int]
        L.kmb_set_force_generic.restype = None
        L.kmb_set_scan_exp2.argtypes = [C.c_int]
        L.kmb_set_scan_exp2.restype = None
        L.kmb_set_sm_reserve.argtypes = [C.c_int]
        L.kmb_set_sm_reserve.restype = None
        L.km_wavefront_plan_create.argtypes = [_l, C.c_long, C.c_long]
        L.km_wavefront_plan_create.restype = C.c_void_p
        L.km_wavefront_plan_free.argtypes = [C.c_void_p]
        L.km_wavefront_plan_level_size.argtypes = [C.c_void_p, C.c_long]
        L.km_wavefront_plan_level_size.restype = C.c_long
        L.km_wavefront_plan_level_offsets.argtypes = [C.c_void_p, C.c_long]
        L.km_wavefront_plan_level_offsets.restype = _l
        L.wavefront_nd_level_size.argtypes = [_l, C.c_long, C.c_long]
        L.wavefront_nd_level_size.restype = C.c_long
        L.wavefront_nd_total_points.argtypes = [_l, C.c_long]
        L.wavefront_nd_total_points.restype = C.c_long
        L.wavefront_nd_max_level.argtypes = [_l, C.c_long]
        L.wavefront_nd_max_level.restype = C.c_long
        DP, NP = C.POINTER(KMBDeltaParams), C.POINTER(KMBNormParams)
        L.kmb_delta_workspace_floats.argtypes = [DP, C.c_int]
        L.kmb_delta_workspace_floats.restype = sz
        L.kmb_delta_forward.argtypes = [DP, vp, C.c_int, vp]
        L.kmb_delta_backward.argtypes = [DP, C.POINTER(KMBDeltaGrads), vp, vp]
        L.kmb_delta_step.argtypes = [DP, vp, C.c_long, vp, vp]
        L.kmb_layernorm_forward.argtypes = [NP, vp]
        L.kmb_layernorm_workspace_floats.argtypes = [NP]
        L.kmb_layernorm_workspace_floats.restype = sz
        L.kmb_layernorm_backward.argtypes = [NP, C.POINTER(KMBNormGrads), vp, vp]
        L.kmb_grad_clip_workspace_floats.argtypes = [C.c_long]
        L.kmb_grad_clip_workspace_floats.restype = sz
        L.kmb_grad_clip.argtypes = [vp, C.c_long, C.c_float, vp, vp, vp]
        L.kmb_model_clip_gradients.argtypes = [vp, C.c_float, vp, vp, vp]
        _lib = L
    return _lib


def last_error() -> str:
    return lib().kmb_last_error().decode()


def _ptr(t):
    """Data pointer of a tensor / numpy array / None."""
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


def dims_array(dims):
    arr = (C.c_long * len(dims))(*[int(d) for d in dims])
    return arr


def scan_params(dims, D, M, x, A, B, Cm, delta, h, y, theta=None, lam=None, default_lambda=0.5,
                use_fast_exp=0, use_a_log_clamp=0, a_log_min=-1e-5, grads=None):
    """Build a ScanNDParams (single-item layout; batched calls use the same
    struct with contiguous [batch, ...] buffers).  Keeps the dims array alive
    on the returned object."""
    p = ScanNDParams()
    darr = dims_array(dims)
    p._dims_keep = darr
    p.max_ndims = 32
    p.max_state = 0
    p.use_fast_exp = int(use_fast_exp)
    p.dims = C.cast(darr, _l)
    p.ndims = len(dims)
    p.D, p.M = int(D), int(M)
    p.x, p.A, p.B, p.C, p.delta = _ptr(x), _ptr(A), _ptr(B), _ptr(Cm), _ptr(delta)
    p.h, p.y = _ptr(h), _ptr(y)
    p.theta, p.lambda_ = _ptr(theta), _ptr(lam)
    p.default_lambda = float(default_lambda)
    p.use_a_log_clamp = int(use_a_log_clamp)
    p.a_log_min = float(a_log_min)
    g = grads or {}
    for k in ("dA", "dB", "dC", "ddelta", "dlambda", "dtheta"):
        setattr(p, k, _ptr(g.get(k)))
    return p


def conv_params(dims, D, K, inp=None, kernel=None, bias=None, out=None, dy=None, dinput=None,
                dkernel=None, dbias=None):
    p = ConvNDParams()
    darr = dims_array(dims)
    p._dims_keep = darr
    p.input, p.kernel, p.bias, p.output = _ptr(inp), _ptr(kernel), _ptr(bias), _ptr(out)
    p.dy, p.dinput, p.dkernel, p.dbias = _ptr(dy), _ptr(dinput), _ptr(dkernel), _ptr(dbias)
    p.dims = C.cast(darr, _l)
    p.ndims = len(dims)
    p.D, p.K = int(D), int(K)
    return p


def check(rc: int, what: str = "call"):
    if rc != 0:
        raise RuntimeError(f"{what} failed: {last_error()}")


def blockscan_params(dims, N, R, u, dt, lam, B, Cm, A_log, theta, h, Bu, y, default_lambda=0.5, use_fast_exp=0):
    p = KMBlockScanParams()
    darr = dims_array(dims)
    p._dims_keep = darr
    p.ndims = len(dims)
    p.dims = C.cast(darr, _l)
    L = 1
    for d in dims:
        L *= int(d)
    p.L, p.N, p.R = L, int(N), int(R)
    p.u, p.dt, p.lambda_, p.B, p.C = _ptr(u), _ptr(dt), _ptr(lam), _ptr(B), _ptr(Cm)
    p.A_log, p.theta = _ptr(A_log), _ptr(theta)
    p.default_lambda = float(default_lambda)
    p.use_fast_exp = int(use_fast_exp)
    p.h, p.Bu, p.y = _ptr(h), _ptr(Bu), _ptr(y)
    return p


def model_config(dims, vocab, dim, N, R, n_layers):
    """KMambaConfig with the reference defaults and the given shape."""
    c = KMambaConfig()
    lib().kmamba_config_set_defaults(C.byref(c))
    L = 1
    for d in dims:
        L *= int(d)
    c.vocab_size, c.dim, c.state_size, c.seq_len = vocab, dim, N, L
    c.n_layers, c.mimo_rank = n_layers, R
    c.spatial_ndims = len(dims)
    for i, d in enumerate(dims):
        c.spatial_dims[i] = int(d)
    return c


def _dtype_of(t):
    """KMB_DTYPE_* of a tensor (float32 or bfloat16)."""
    name = str(t.dtype)
    if name.endswith("bfloat16"):
        return DTYPE_BF16
    if name.endswith("float32"):
        return DTYPE_F32
    raise TypeError(f"float32 or bfloat16 expected, got {name}")


def _rows_ld(t, inner, what):
    """Elements between two tokens (or rows) of t, whose last `inner` axes must be contiguous and whose leading axes
    must be walked by one stride."""
    st, sh = t.stride(), t.shape
    if t.numel() == 0:
        return 0
    want = 1
    for i in range(1, inner + 1):
        if sh[-i] != 1 and st[-i] != want:
            raise ValueError(f"{what}: the last {inner} axes must be contiguous")
        want *= sh[-i]
    lead = [(n, s) for n, s in zip(sh[:-inner], st[:-inner]) if n != 1]
    if not lead:
        return want
    for (n, s), (n1, s1) in zip(lead, lead[1:]):
        if s != n1 * s1:
            raise ValueError(f"{what}: rows must follow each other at one stride")
    if lead[-1][1] < want:
        raise ValueError(f"{what}: rows overlap")
    return lead[-1][1]


def _f32(t, what, shape=None):
    if t is None:
        return
    if _dtype_of(t) != DTYPE_F32 or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous float32 tensor is expected")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: shape {tuple(shape)} expected, got {tuple(t.shape)}")


def _typed(t, like, shape, what):
    if t is None:
        return
    if t.dtype != like.dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {like.dtype} {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}")


def _space(t, what, floats):
    """A workspace or result that the library writes: contiguous float32, at least so long."""
    if t.element_size() != 4 or not t.is_floating_point() or not t.is_contiguous() or t.numel() < floats:
        raise ValueError(f"{what}: a contiguous float32 tensor of at least {floats} entries is expected")


def _one_device(like, **tensors):
    for what, t in tensors.items():
        if t is not None and t.device != like.device:
            raise ValueError(f"{what}: on {t.device}, expected on {like.device}")


def _on_device(p, *tensors):
    """The kernels read device memory: a call takes only CUDA tensors of its parameters' device."""
    if p._device < 0:
        raise ValueError("CUDA tensors are expected")
    for t in tensors:
        if t is not None and t.get_device() != p._device:
            raise ValueError(f"a tensor is on {t.device}, its call's parameters on cuda:{p._device}")


def delta_params(q, k, v, g, beta, o, scale=1.0, h0=None, hT=None, cu_seqlens=None):
    """KMBDeltaParams of device tensors: q, k [batch, T, Hk, dk], v, o [batch, T, Hv, dv] (slices of a wider token row
    are fine), g, beta [batch, T, Hv] or None, states [sequences, Hv, dk, dv] or None, cu_seqlens int32
    [sequences + 1] with batch 1.  The struct holds its tensors, the outputs among them: an autograd function that kept it
    on its context would keep itself alive."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    _typed(k, q, q.shape, "k")
    _typed(v, q, (B, T, Hv, dv), "v")
    _typed(o, q, v.shape, "o")
    for t, n in ((g, "g"), (beta, "beta")):
        _f32(t, n, (B, T, Hv))
    if cu_seqlens is not None and (not str(cu_seqlens.dtype).endswith("int32") or not cu_seqlens.is_contiguous()):
        raise ValueError("cu_seqlens: a contiguous int32 tensor is expected")
    n = B if cu_seqlens is None else cu_seqlens.numel() - 1
    for t, name in ((h0, "h0"), (hT, "hT")):
        _f32(t, name, (n, Hv, dk, dv))
    _one_device(q, k=k, v=v, g=g, beta=beta, o=o, h0=h0, hT=hT, cu_seqlens=cu_seqlens)
    p = KMBDeltaParams()
    p.batch, p.T, p.Hk, p.Hv, p.dk, p.dv = B, T, Hk, Hv, dk, dv
    p.dtype, p.scale = _dtype_of(q), float(scale)
    p.cu_seqlens, p.n_seq = _ptr(cu_seqlens), n if cu_seqlens is not None else 0
    p.q, p.k, p.v, p.g, p.beta, p.o = _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(o)
    p.h0, p.hT = _ptr(h0), _ptr(hT)
    p.ld_q, p.ld_k, p.ld_v, p.ld_o = (_rows_ld(t, 2, w) for t, w in ((q, "q"), (k, "k"), (v, "v"), (o, "o")))
    p._keep = (q, k, v, g, beta, o, h0, hT, cu_seqlens)
    import torch   # loaded already: the tensors are its own
    p._state, p._device, p._index_type = (Hv, dk, dv), q.get_device(), torch.int32
    return p


def delta_workspace_floats(p, train=False):
    return lib().kmb_delta_workspace_floats(C.byref(p), int(bool(train)))


def delta_grads(p, do, dq, dk, dv, dg=None, dbeta=None, dh0=None, dhT=None):
    """KMBDeltaGrads for a KMBDeltaParams of delta_params."""
    q, k, v = p._keep[:3]
    for t, like, n in ((do, v, "do"), (dq, q, "dq"), (dk, k, "dk"), (dv, v, "dv")):
        _typed(t, q, like.shape, n)
    for t, n in ((dg, "dg"), (dbeta, "dbeta")):
        _f32(t, n, v.shape[:3])
    seqs = p.n_seq if p.cu_seqlens else p.batch
    for t, n in ((dh0, "dh0"), (dhT, "dhT")):
        _f32(t, n, (seqs, p.Hv, p.dk, p.dv))
    _one_device(q, do=do, dq=dq, dk=dk, dv=dv, dg=dg, dbeta=dbeta, dh0=dh0, dhT=dhT)
    g = KMBDeltaGrads()
    g.do_, g.dhT, g.dq, g.dk, g.dv = _ptr(do), _ptr(dhT), _ptr(dq), _ptr(dk), _ptr(dv)
    g.dg, g.dbeta, g.dh0 = _ptr(dg), _ptr(dbeta), _ptr(dh0)
    g.ld_do, g.ld_dq, g.ld_dk, g.ld_dv = (_rows_ld(t, 2, n) for t, n in
                                          ((do, "do"), (dq, "dq"), (dk, "dk"), (dv, "dv")))
    g._keep = (do, dq, dk, dv, dg, dbeta, dh0, dhT)
    return g


def delta_forward(p, ws, keep=False, stream=None):
    """Chunked gated delta rule; keep=True leaves in ws (a training workspace) what delta_backward reads."""
    _space(ws, "delta workspace", delta_workspace_floats(p, keep))
    _on_device(p, ws)
    if (_lib or lib()).kmb_delta_forward(p, ws.data_ptr(), 1 if keep else 0, stream):
        check(-1, "kmb_delta_forward")


def delta_backward(p, grads, ws, stream=None):
    _space(ws, "delta workspace", delta_workspace_floats(p, True))
    _on_device(p, ws)
    if (_lib or lib()).kmb_delta_backward(p, grads, ws.data_ptr(), stream):
        check(-1, "kmb_delta_backward")


def delta_step(p, pool, slots=None, stream=None):
    """Recurrent form: the T tokens of each row against its state in pool [entries, Hv, dk, dv], updated in place."""
    shape = pool.shape
    if (len(shape) != 4 or shape != (shape[0],) + p._state or pool.element_size() != 4 or not pool.is_floating_point()
            or not pool.is_contiguous()):
        raise ValueError("pool: a contiguous float32 [entries, Hv, dk, dv] tensor is expected")
    if slots is not None and (slots.dtype is not p._index_type or slots.numel() != p.batch or not slots.is_contiguous()):
        raise ValueError("slots: a contiguous int32 tensor with one entry per row is expected")
    _on_device(p, pool, slots)
    if (_lib or lib()).kmb_delta_step(p, pool.data_ptr(), shape[0], None if slots is None else slots.data_ptr(), stream):
        check(-1, "kmb_delta_step")


def norm_params(x, w, b, y, eps=1e-5, residual=None, total=None, stats=None):
    """KMBNormParams of device tensors: x, residual, total, y [..., D]; w, b float32 [D] or None; stats float32
    [2, rows] (mean, rstd) or None."""
    D = x.shape[-1]
    rows = x.numel() // D if D else 0
    for t, n in ((y, "y"), (residual, "residual"), (total, "total")):
        _typed(t, x, x.shape, n)
    for t, n in ((w, "w"), (b, "b")):
        _f32(t, n, (D,))
    _f32(stats, "stats", (2, rows))
    _one_device(x, w=w, b=b, y=y, residual=residual, total=total, stats=stats)
    p = KMBNormParams()
    p.rows, p.D, p.dtype, p.eps = rows, D, _dtype_of(x), float(eps)
    p.x, p.residual, p.total, p.y, p.w, p.b = _ptr(x), _ptr(residual), _ptr(total), _ptr(y), _ptr(w), _ptr(b)
    if stats is not None:
        p.mean, p.rstd = stats.data_ptr(), stats.data_ptr() + 4 * rows
    p.ld_x, p.ld_residual, p.ld_total, p.ld_y = (0 if t is None else _rows_ld(t, 1, n) for t, n in
                                                 ((x, "x"), (residual, "residual"), (total, "total"), (y, "y")))
    p._keep = (x, w, b, y, residual, total, stats)
    p._device = x.get_device()
    return p


def norm_grads(p, dy, dx=None, dw=None, db=None, dtotal=None, accumulate=False):
    """KMBNormGrads for a KMBNormParams of norm_params."""
    x = p._keep[0]
    for t, n in ((dy, "dy"), (dx, "dx"), (dtotal, "dtotal")):
        _typed(t, x, x.shape, n)
    for t, n in ((dw, "dw"), (db, "db")):
        _f32(t, n, (p.D,))
    _one_device(x, dy=dy, dx=dx, dw=dw, db=db, dtotal=dtotal)
    g = KMBNormGrads()
    g.dy, g.dtotal, g.dx, g.dw, g.db = _ptr(dy), _ptr(dtotal), _ptr(dx), _ptr(dw), _ptr(db)
    g.ld_dy, g.ld_dtotal, g.ld_dx = (0 if t is None else _rows_ld(t, 1, n) for t, n in
                                     ((dy, "dy"), (dtotal, "dtotal"), (dx, "dx")))
    g.accumulate = int(bool(accumulate))
    g._keep = (dy, dx, dw, db, dtotal)
    return g


def norm_workspace_floats(p):
    return lib().kmb_layernorm_workspace_floats(C.byref(p))


def norm_forward(p, stream=None):
    _on_device(p)
    if (_lib or lib()).kmb_layernorm_forward(p, stream):
        check(-1, "kmb_layernorm_forward")


def norm_backward(p, grads, ws=None, stream=None):
    if ws is not None:
        _space(ws, "norm workspace", norm_workspace_floats(p) if grads.dw or grads.db else 0)
    _on_device(p, ws)
    if (_lib or lib()).kmb_layernorm_backward(p, grads, _ptr(ws), stream):
        check(-1, "kmb_layernorm_backward")


def grad_list(grads, outs=None):
    """KMBGradTensor array of contiguous gradient tensors; outs: where the clipped ones go (default: in place)."""
    outs = grads if outs is None else outs
    if len(outs) != len(grads):
        raise ValueError(f"grad_list: {len(grads)} gradients, {len(outs)} outputs")
    arr = (KMBGradTensor * len(grads))()
    for e, t, o in zip(arr, grads, outs):
        if not t.is_contiguous():
            raise ValueError("grad_list: contiguous tensors are expected")
        if o is not None and (o.dtype != t.dtype or o.numel() != t.numel() or not o.is_contiguous()):
            raise ValueError("grad_list: an output does not match its gradient")
        _one_device(grads[0], gradient=t, output=o)
        e.in_, e.out, e.n, e.dtype = t.data_ptr(), _ptr(o), t.numel(), _dtype_of(t)
    arr._keep = (list(grads), list(outs))
    arr._device = grads[0].get_device() if len(grads) else None
    arr._space = grad_clip_workspace_floats(arr)
    return arr


def grad_clip_workspace_floats(lst):
    return lib().kmb_grad_clip_workspace_floats(len(lst))


def grad_clip(lst, max_norm, result, ws, stream=None):
    """Global norm of a grad_list and clipping by it; result: float32 [2], norm and coefficient."""
    if result is not None:
        _space(result, "result", 2)
    _space(ws, "clip workspace", lst._space)
    if len(lst):
        _on_device(lst, ws, result)
    elif ws.get_device() < 0:
        raise ValueError("CUDA tensors are expected")
    if (_lib or lib()).kmb_grad_clip(lst, len(lst), max_norm, _ptr(result), ws.data_ptr(), stream):
        check(-1, "kmb_grad_clip")


class DeviceArray:
    """Minimal __cuda_array_interface__ view of a library-owned device buffer
    (float32), so torch.as_tensor can read it without copying."""

    def __init__(self, ptr, n):
        self.__cuda_array_interface__ = {"shape": (int(n),), "typestr": "<f4", "data": (int(ptr), False),
                                         "version": 3}
