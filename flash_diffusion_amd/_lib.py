"""ctypes binding of libfdmi.so (include/fdmi.h).  Fails loudly when the library is missing --
there is deliberately no fallback path."""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("FDMI_LIB", os.path.join(_HERE, "libfdmi.so"))
_lib = None

i32, i64, f32, vp = C.c_int32, C.c_int64, C.c_float, C.c_void_p


class GemmDesc(C.Structure):
    _fields_ = [
        ("M", i32), ("N", i32), ("K", i32),
        ("A", vp), ("lda", i64), ("W", vp), ("ldw", i64),
        ("mode", i32),
        ("Hin", i32), ("Win", i32), ("Cin", i32), ("Hout", i32), ("Wout", i32), ("KH", i32), ("KW", i32),
        ("stride", i32), ("pad", i32), ("ups", i32), ("dgrad", i32),
        ("bias", vp),
        ("rowvec", vp), ("rowvec_ld", i64), ("rows_per_batch", i32),
        ("residual", vp), ("ldr", i64),
        ("act", i32),
        ("preact", vp), ("ldp", i64),
        ("C", vp), ("ldc", i64), ("out_f32", i32),
        ("alpha", f32),
        ("splitk", i32), ("ws", vp),
        ("accum_atomic", i32), ("force_tile", i32), ("use_glds", i32),
        ("A2", vp), ("lda2", i64), ("K1", i32),
        ("rowvec_mul", i32),
    ]


class WgradProblem(C.Structure):
    """fdmi_wgrad_problem (include/fdmi.h)"""
    _fields_ = [("X", C.c_void_p), ("ldx", C.c_int64), ("Y", C.c_void_p), ("ldy", C.c_int64), ("M", C.c_int64),
                ("N1", C.c_int32), ("N2", C.c_int32), ("C", C.c_void_p), ("ldc", C.c_int64)]


class Fp8Desc(C.Structure):
    """fdmi_fp8_desc (include/fdmi.h)"""
    _fields_ = [("M", i32), ("N", i32), ("K", i32), ("x", vp), ("ldxr", i64), ("x_f32", i32), ("X", vp), ("sx", vp), ("W", vp), ("sw", vp),
                ("W2", vp), ("sw2", vp), ("bias", vp), ("residual", vp), ("ldr", i64), ("C", vp), ("ldc", i64), ("out_f32", i32),
                ("act", i32), ("H", vp), ("sh", vp)]


class UNetCfg(C.Structure):
    _fields_ = [("in_channels", i32), ("out_channels", i32), ("n_levels", i32), ("block_out", i32 * 4),
                ("down_attn", i32 * 4), ("up_attn", i32 * 4), ("layers_per_block", i32), ("tlayers", i32 * 4),
                ("heads", i32 * 4), ("cross_dim", i32), ("groups", i32), ("eps", f32), ("class_embed_dim", i32),
                ("flip_sin_to_cos", i32), ("freq_shift", f32), ("precision", i32)]


class NetCfg(C.Structure):
    _fields_ = [("kind", i32), ("in_channels", i32), ("out_channels", i32), ("n_levels", i32), ("block_out", i32 * 4),
                ("layers_per_block", i32), ("groups", i32), ("eps", f32), ("precision", i32), ("lpips_shift", f32 * 3),
                ("lpips_scale", f32 * 3), ("adapter_downscale", i32), ("adapter_xl", i32)]


class DitCfg(C.Structure):
    _fields_ = [("kind", i32), ("in_channels", i32), ("out_channels", i32), ("patch_size", i32), ("num_layers", i32),
                ("heads", i32), ("head_dim", i32), ("cross_dim", i32), ("caption_channels", i32), ("tdim", i32),
                ("vec_dim", i32), ("n_vec", i32), ("attention_bias", i32), ("norm_eps", f32), ("precision", i32)]


_SIGS = {
    "fdmi_dit_create": (vp, [C.POINTER(DitCfg)]),
    "fdmi_dit_workspace_bytes": (i64, [vp, i32, i32, i32, i32, i32, i32]),
    "fdmi_dit_forward": (i32, [vp, i32, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, vp, i64, i32, vp]),
    "fdmi_dit_backward": (i32, [vp, i32, vp, vp, vp]),
    "fdmi_unet_declare_lora": (i32, [vp, C.c_char_p, i32]),
    "fdmi_dit_teacher_loop_scratch_bytes": (i64, [vp, i32, i32, i32]),
    "fdmi_dit_teacher_loop": (i32, [vp, i32, vp, vp, i32, vp, vp, vp, vp, vp, i32, i32, i32, i32, vp, i64, vp, i64, vp]),
    "fdmi_unet_create": (vp, [C.POINTER(UNetCfg)]),
    "fdmi_unet_destroy": (None, [vp]),
    "fdmi_unet_num_params": (i64, [vp]),
    "fdmi_unet_param_name": (i32, [vp, i64, C.c_char_p, i64, C.POINTER(i64)]),
    "fdmi_unet_set_param": (i32, [vp, C.c_char_p, vp, i64, vp]),
    "fdmi_unet_set_lora": (i32, [vp, C.c_char_p, vp, vp, vp, vp, i32]),
    "fdmi_unet_ready": (i32, [vp]),
    "fdmi_unet_workspace_bytes": (i64, [vp, i32, i32, i32, i32, i32]),
    "fdmi_unet_forward": (i32, [vp, i32, vp, vp, vp, vp, vp, i32, i32, i32, i32, vp, i64, i32, vp]),
    "fdmi_unet_backward": (i32, [vp, i32, vp, vp, vp]),
    "fdmi_unet_last_flops": (C.c_double, [vp]),
    "fdmi_unet_last_gn_epilogue": (i32, [vp, C.POINTER(i32)]),
    "fdmi_unet_last_hbm_bytes": (C.c_double, [vp, i32]),
    "fdmi_unet_set_down_residuals": (i32, [vp, vp, i32, f32]),
    "fdmi_net_create": (vp, [C.POINTER(NetCfg)]),
    "fdmi_net_workspace_bytes": (i64, [vp, i32, i32, i32, i32]),
    "fdmi_net_forward": (i32, [vp, i32, vp, vp, vp, i32, i32, i32, vp, i64, i32, vp]),
    "fdmi_net_backward": (i32, [vp, i32, vp, vp, vp]),
    "fdmi_adapter_out_shape": (i32, [vp, i32, i32, i32, C.POINTER(i32), C.POINTER(i32), C.POINTER(i32)]),
    "fdmi_adapter_forward": (i32, [vp, i32, vp, vp, i32, i32, i32, i32, vp, i64, vp]),
    "fdmi_teacher_loop_scratch_bytes": (i64, [vp, i32, i32, i32]),
    "fdmi_teacher_loop": (i32, [vp, i32, vp, vp, i32, vp, vp, vp, i32, i32, i32, i32, vp, i64, vp, i64, vp]),
    "fdmi_version": (i32, []),
    "fdmi_comm_unique_id": (i32, [vp]),
    "fdmi_allreduce_init": (i32, [i32, i32, vp]),
    "fdmi_allreduce": (i32, [vp, i64, i32, vp]),
    "fdmi_allreduce_world": (i32, []),
    "fdmi_allreduce_destroy": (i32, []),
    "fdmi_tune_set": (i32, [i32, i32]),
    "fdmi_tune_value": (i32, [i32]),
    "fdmi_prof_enable": (i32, [i32]),
    "fdmi_prof_collect": (i32, [i32, vp, vp, vp]),
    "fdmi_prof_collect2": (i32, [i32, vp, vp, vp, vp]),
    "fdmi_prof_dump": (i32, [C.c_char_p]),
    "fdmi_gemm": (i32, [C.POINTER(GemmDesc), vp]),
    "fdmi_gemm_plan": (i32, [C.POINTER(GemmDesc), vp, vp, vp, vp]),
    "fdmi_gemm_a2_ok": (i32, [C.POINTER(GemmDesc)]),
    "fdmi_wgrad_tn": (i32, [vp, i64, vp, i64, i64, i32, i32, vp, i64, vp]),
    "fdmi_wgrad_tn_group": (i32, [vp, i32, vp]),
    "fdmi_gemm_gn_ok": (i32, [C.POINTER(GemmDesc), i32, i32]),
    "fdmi_gemm_gn": (i32, [C.POINTER(GemmDesc), vp, i32, i32, vp]),
    "fdmi_groupnorm_apply": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, vp]),
    "fdmi_groupnorm_fwd": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, vp]),
    "fdmi_groupnorm_bwd": (i32, [vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, i32, vp]),
    "fdmi_groupnorm_cat_fwd": (i32, [vp, vp, i32, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, vp]),
    "fdmi_groupnorm_cat_bwd": (i32, [vp, vp, i32, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, i32, vp]),
    "fdmi_layernorm_fwd": (i32, [vp, vp, vp, vp, i64, i32, f32, vp]),
    "fdmi_layernorm_bwd": (i32, [vp, vp, vp, vp, i64, i32, f32, i32, vp]),
    "fdmi_layernorm_mod_fwd": (i32, [vp, vp, vp, i64, i32, vp, vp, i64, i32, f32, vp]),
    "fdmi_layernorm_mod_bwd": (i32, [vp, vp, vp, i64, i32, vp, i64, i32, f32, i32, vp]),
    "fdmi_gate_residual": (i32, [vp, vp, i64, vp, vp, i64, i32, i32, vp]),
    "fdmi_gelu_tanh": (i32, [vp, vp, i64, vp]),
    "fdmi_gelu_tanh_bwd": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_batch_colsum": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, vp]),
    "fdmi_attn_tr_elems": (i64, [i32, i32, i32, i32]),
    "fdmi_attn_bwd_ws_bytes": (i64, [i32, i32, i32, i32, i32]),
    "fdmi_attn_fwd": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, vp, vp, i32, i32, i32, i32, i32, f32, vp]),
    "fdmi_attn_bwd": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, vp, i64, vp, vp, i64, vp, i64, vp, i64, vp,
                            i32, i32, i32, i32, i32, f32, vp]),
    "fdmi_nchw_to_nhwc": (i32, [vp, vp, i32, i32, i32, i32, vp]),
    "fdmi_nhwc_to_nchw": (i32, [vp, i64, vp, i32, i32, i32, i32, vp]),
    "fdmi_timestep_embed": (i32, [vp, vp, i32, i32, i32, f32, vp]),
    "fdmi_geglu_bwd": (i32, [vp, vp, vp, i64, i32, vp]),
    "fdmi_pool2x2_sum": (i32, [vp, vp, i32, i32, i32, i32, i32, vp]),
    "fdmi_cast_transpose": (i32, [vp, vp, vp, i32, i32, vp]),
    "fdmi_transpose2d": (i32, [vp, i64, vp, i64, i64, i32, vp]),
    "fdmi_adamw": (i32, [vp, vp, vp, vp, i64, f32, f32, f32, f32, f32, i32, f32, vp]),
    "fdmi_add_noise": (i32, [vp, vp, vp, vp, vp, i32, i64, vp]),
    "fdmi_axpby4": (i32, [vp, f32, vp, f32, vp, f32, vp, f32, vp, i64, vp]),
    "fdmi_im2col": (i32, [vp, vp, i32, i32, i32, i32, i32, i32, i32, i32, i32, i32, vp]),
    "fdmi_silu": (i32, [vp, vp, i64, vp]),
    "fdmi_silu_bwd": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_colsum": (i32, [vp, vp, vp, vp, vp, i64, i32, i32, i32, f32, vp]),
    "fdmi_transpose2d_pad": (i32, [vp, i64, vp, i64, i64, i32, i64, vp]),
    "fdmi_pad_cols": (i32, [vp, i32, vp, i32, i64, vp]),
    "fdmi_f32_to_bf16": (i32, [vp, vp, i64, vp]),
    "fdmi_distill_loss": (i32, [vp, vp, i64, i32, vp, vp]),
    "fdmi_distill_grad": (i32, [vp, vp, i64, i32, f32, vp, vp]),
    "fdmi_dmd_loss": (i32, [vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i64, vp]),
    # 8-bit block-scaled products (csrc/fp8.hip) and the embedding lookup (csrc/embed.hip)
    "fdmi_quant_fp8": (i32, [vp, i32, i64, vp, f32, vp, vp, i64, i32, vp]),
    "fdmi_pack_fp8": (i32, [vp, i32, i64, i32, i32, vp, vp, vp, vp, vp]),
    "fdmi_gemm_fp8": (i32, [C.POINTER(Fp8Desc), vp]),
    "fdmi_fp8_scratch_bytes": (i64, [i64, i32]),
    "fdmi_embed_fwd": (i32, [vp, i32, i64, i32, i64, vp, i32, i64, f32, vp, i64, i64, vp, i32, vp]),
    "fdmi_embed_bwd_ws_bytes": (i64, [i64, i32]),
    "fdmi_embed_bwd": (i32, [vp, i32, i64, vp, i32, i64, i64, i32, f32, i32, vp, i64, vp, vp]),
    # fp32 validation mode (csrc/ref32.hip)
    "fdmi_gemm_f32": (i32, [C.POINTER(GemmDesc), vp]),
    "fdmi_wgrad_tn_f32": (i32, [vp, i64, vp, i64, i64, i32, i32, vp, i64, vp]),
    "fdmi_attn_scratch_elems_f32": (i64, [i32, i32, i32, i32, i32]),
    "fdmi_attn_fwd_f32": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, i32, f32, vp, i64, vp]),
    "fdmi_attn_causal_fwd_f32": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, f32, vp, i64, vp]),
    "fdmi_attn_bias_fwd_f32": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, i32, f32, vp, vp, vp, i64, vp]),
    "fdmi_rmsnorm": (i32, [vp, vp, vp, i64, i32, f32, vp]),
    "fdmi_rmsnorm_f32": (i32, [vp, vp, vp, i64, i32, f32, vp]),
    "fdmi_mul": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_mul_f32": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_attn_bwd_f32": (i32, [vp, i64, vp, i64, vp, i64, vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, i32, f32, vp,
                                i64, vp]),
    "fdmi_groupnorm_fwd_f32": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, vp]),
    "fdmi_groupnorm_bwd_f32": (i32, [vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, vp]),
    "fdmi_layernorm_fwd_f32": (i32, [vp, vp, vp, vp, vp, i64, i32, vp, vp, i64, i32, f32, vp]),
    "fdmi_layernorm_bwd_f32": (i32, [vp, vp, vp, vp, i64, i32, vp, i64, i32, f32, i32, vp]),
    "fdmi_nchw_to_nhwc_f32": (i32, [vp, vp, i32, i32, i32, i32, vp]),
    "fdmi_nhwc_to_nchw_f32": (i32, [vp, i64, vp, i32, i32, i32, i32, vp]),
    "fdmi_silu_f32": (i32, [vp, vp, i64, vp]),
    "fdmi_silu_bwd_f32": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_gelu_tanh_f32": (i32, [vp, vp, i64, vp]),
    "fdmi_gelu_tanh_bwd_f32": (i32, [vp, vp, vp, i64, vp]),
    "fdmi_gate_residual_f32": (i32, [vp, vp, i64, vp, vp, i64, i32, i32, vp]),
    "fdmi_batch_colsum_f32": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, vp]),
    "fdmi_im2col_f32": (i32, [vp, vp, i32, i32, i32, i32, i32, i32, i32, i32, i32, i32, vp]),
    "fdmi_colsum_f32": (i32, [vp, vp, vp, vp, vp, i64, i32, i32, i32, vp]),
    "fdmi_timestep_embed_f32": (i32, [vp, vp, i32, i32, i32, f32, vp]),
    "fdmi_pad_cols_f32": (i32, [vp, i32, vp, i32, i64, vp]),
}
# extended lazily by unet.py for the plan API
EXTRA_SIGS = {}


def declared_symbols():
    return sorted(list(_SIGS) + list(EXTRA_SIGS) + ["fdmi_last_error"])


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                "(make -C flash_diffusion_amd/csrc). There is no fallback path.")
        l = C.CDLL(LIB_PATH)
        l.fdmi_last_error.restype = C.c_char_p
        l.fdmi_last_error.argtypes = []
        for name, (res, args) in list(_SIGS.items()) + list(EXTRA_SIGS.items()):
            fn = getattr(l, name)
            fn.restype = res
            fn.argtypes = args
        for kv in filter(None, os.environ.get("FDMI_TUNE", "").split(",")):   # developer knobs, e.g. FDMI_TUNE=12=1
            k, v = kv.split("=")
            l.fdmi_tune_set(int(k), int(v))
        _lib = l
    return _lib


def source_hash():
    """sha256 (first 16 hex digits) over the kernel sources of this build (csrc/*.hip, *.h, include/fdmi.h): ties measured
    artefacts under profiles/ (PMC traffic) to the build they describe"""
    import glob
    import hashlib
    h = hashlib.sha256()
    for f in sorted(glob.glob(os.path.join(_HERE, "csrc", "*.hip")) + glob.glob(os.path.join(_HERE, "csrc", "*.h")) +
                    [os.path.join(os.path.dirname(_HERE), "include", "fdmi.h")]):
        with open(f, "rb") as fh:
            h.update(os.path.basename(f).encode() + b"\0" + fh.read())
    return h.hexdigest()[:16]


# the sources that define each MFMA kernel family (bench.py's bucket names): PMC traffic measured for a family stays valid for
# as long as THESE files are unchanged -- an edit to another kernel's file no longer voids it
_KERNEL_SOURCES = {"gemm4_kernel": ("gemm4.hip", "gemm_tile.h", "gemm.h", "common.h"),
                   "gemm3_kernel": ("gemm3.hip", "gemm_tile.h", "gemm.h", "common.h"),
                   "gemm_kernel": ("gemm.hip", "gemm.h", "common.h"),
                   "attn_": ("attn.hip", "ops.h", "common.h"),
                   "wgrad_tn_kernel": ("wgrad.hip", "gemm_tile.h", "gemm.h", "common.h")}


def kernel_source_hash(bucket: str):
    """sha256 (first 16 hex digits) over the source files of one kernel family ("gemm4_kernel<256x320,row>" -> gemm4.hip +
    the headers it includes); None for an unknown family"""
    import hashlib
    for prefix, files in _KERNEL_SOURCES.items():
        if bucket.startswith(prefix):
            h = hashlib.sha256()
            for f in files:
                with open(os.path.join(_HERE, "csrc", f), "rb") as fh:
                    h.update(f.encode() + b"\0" + fh.read())
            return h.hexdigest()[:16]
    return None


def check(rc):
    if rc != 0:
        raise RuntimeError("fdmi: " + lib().fdmi_last_error().decode())


def stream_ptr():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    """device pointer of a torch tensor (or None)"""
    return None if t is None else C.c_void_p(t.data_ptr())
