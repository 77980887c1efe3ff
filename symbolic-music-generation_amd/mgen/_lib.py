"""ctypes binding of libmgen_hip.so (the C-ABI declared in include/mgen.h).

The library holds the hand-written gfx950 kernels. There is no fallback: if it is missing or a call fails the
caller gets an exception.
"""
import ctypes
import os
from ctypes import c_void_p as P, c_int as I, c_long as L, c_float as F, c_ulonglong as U64

_HERE = os.path.dirname(os.path.abspath(__file__))
# MGEN_LIB names another build of the same library (A/B measurements of kernel variants on one machine)
LIB_PATH = os.environ.get("MGEN_LIB") or os.path.join(_HERE, "libmgen_hip.so")

# name -> argument types (every function returns int, 0 = ok), in the order of include/mgen.h
SIGNATURES = {
    "mgen_gemm_bf16": [P, P, P, P, I, I, I, L, L, L, L, I, I, I, F, P],
    "mgen_gemm_bf16_seg": [P, P, P, P, P, P, I, I, I, I, L, L, L, L, L, L, I, I, P],
    "mgen_gemm_bf16_slabs": [P, P, P, I, I, I, L, L, I, I, I, P],
    "mgen_slab_resid_rmsnorm": [P, I, L, P, P, P, P, L, I, F, I, P],
    "mgen_rmsnorm_fwd": [P, P, P, P, L, I, F, I, P],
    "mgen_resid_rmsnorm_fwd": [P, P, L, P, P, P, P, L, I, F, P],
    "mgen_rmsnorm_bwd": [P, P, P, P, P, P, P, L, I, I, I, P],
    "mgen_rope_table": [P, P, I, I, P],
    "mgen_qknorm_rope_fwd": [P, L, P, P, L, L, P, P, P, P, I, L, I, I, I, F, I, P],
    "mgen_qknorm_rope_bwd": [P, L, P, P, L, L, P, L, P, P, P, P, P, P, I, L, I, I, I, F, I, P],
    "mgen_qknorm_rope_il_fwd": [P, L, P, P, L, L, P, P, P, P, I, L, I, I, I, F, I, P],
    "mgen_qknorm_rope_il_bwd": [P, L, P, P, L, L, P, L, P, P, P, P, P, P, I, L, I, I, I, F, I, P],
    "mgen_rope4d_table": [P, P, P, L, I, P],
    "mgen_qkvnorm_rope4d_fwd": [P, L, P, P, P, L, L, L, P, P, P, L, I, I, I, I, F, I, P],
    "mgen_qkvnorm_rope4d_bwd": [P, L, P, P, P, L, L, L, P, L, P, P, P, P, P, L, I, I, I, I, F, I, P],
    "mgen_fill_rows": [P, P, L, I, P],
    "mgen_cos4d_count": [P, L, P, P, P],
    "mgen_cos4d_fwd_bwd": [P, P, P, F, P, P, P, L, I, P],
    "mgen_cos4d_components": [P, P, L, P, P],
    "mgen_pos4d_next": [P, L, P, L, P, L, I, P],
    "mgen_attn_fwd": [P, P, P, P, P, L, L, L, L, I, I, I, I, I, F, P],
    "mgen_attn_bwd": [P, P, P, P, P, P, P, P, P, P, L, L, L, L, L, L, L, L, I, I, I, I, I, F, P],
    "mgen_attn_fwd_dropout": [P, P, P, P, P, L, L, L, L, I, I, I, I, I, F, F, U64, P],
    "mgen_attn_bwd_dropout": [P, P, P, P, P, P, P, P, P, P, L, L, L, L, L, L, L, L, I, I, I, I, I, F, F, U64, P],
    "mgen_dropout": [P, P, L, I, F, U64, P],
    "mgen_dropout_add": [P, P, L, I, F, U64, P],
    "mgen_dropout_resid": [P, P, P, L, F, U64, P],
    "mgen_swiglu_fwd": [P, P, L, I, I, P],
    "mgen_swiglu_bwd": [P, P, P, L, I, P],
    "mgen_swiglu_bwd_ld": [P, L, P, L, P, L, L, I, P],
    "mgen_gemm_bf16_swiglu": [P, P, P, P, I, I, I, L, L, L, L, P],
    "mgen_comm_unique_id": [P],
    "mgen_comm_rccl_version": [P],
    "mgen_comm_init": [P, P, I, I, I],
    "mgen_comm_allreduce_bucket": [P, P, L, I, P],
    "mgen_comm_wait": [P, P, P, P],
    "mgen_comm_abort": [P],
    "mgen_comm_destroy": [P],
    "mgen_embedding_fwd": [P, P, P, L, I, L, P, P],
    "mgen_embedding_bwd": [P, P, P, L, I, L, P],
    "mgen_gemm_bf16_bias": [P, P, P, P, P, I, I, I, L, L, L, L, I, I, I, P],
    "mgen_layernorm_fwd": [P, P, P, P, P, P, L, I, F, I, P],
    "mgen_layernorm_bwd": [P, P, P, P, P, P, P, P, P, L, I, I, I, P],
    "mgen_gelu_new_fwd": [P, P, L, P],
    "mgen_gelu_new_bwd": [P, P, P, L, P],
    "mgen_colsum_bf16": [P, L, P, L, I, P],
    "mgen_embed_pos_fwd": [P, P, P, P, P, L, I, I, L, I, P, P],
    "mgen_split_bf16": [P, P, P, L, P],
    "mgen_swiglu_f32_fwd": [P, P, L, I, P],
    "mgen_swiglu_f32_bwd": [P, P, P, L, I, P],
    "mgen_attn_f32_fwd": [P, P, P, P, P, L, L, L, L, I, I, I, I, I, F, P],
    "mgen_attn_f32_bwd": [P, P, P, P, P, P, P, P, P, P, L, L, L, L, L, L, L, L, I, I, I, I, I, F, P],
    "mgen_gelu_new_f32_fwd": [P, P, L, P],
    "mgen_gelu_new_f32_bwd": [P, P, P, L, P],
    "mgen_bias_add_f32": [P, L, P, L, I, P],
    "mgen_colsum_f32": [P, L, P, L, I, P],
    "mgen_collate_tokens": [P, P, P, P, P, P, I, I, L, I, P],
    "mgen_collate_pos4d": [P, L, P, P, P, P, P, I, I, P],
    "mgen_notes_to_events": [P, L, F, P, P, P],
    "mgen_cast": [P, P, L, I, P],
    "mgen_transpose_bf16": [P, P, I, I, L, L, I, L, L, P],
    "mgen_gemm_bf16_wgrad_group": [I, P, P, P, P, P, I, P, P, P, P],
    "mgen_ce_count": [P, L, I, L, P, P, L, P, P],
    "mgen_check_right_padding": [P, I, I, P, P],
    "mgen_ce_fwd_bwd": [P, P, L, L, I, L, I, L, P, F, P, P, I, I, P],
    "mgen_ce_finalize": [P, L, P, P, P],
    "mgen_lmhead_ce_fwd_bwd": [P, L, P, L, P, L, I, I, I, L, L, P, L, P, P, L, P, I, P, P],
    "mgen_grad_norm_clip": [P, L, F, P, P, P],
    "mgen_grad_norm_clip_static": [P, L, F, P, P],
    "mgen_adamw_step": [P, P, P, P, P, L, P, F, F, F, F, F, L, P],
    "mgen_scale_f32": [P, L, F, P, P],
    "mgen_axpy_f32": [P, P, L, F, P, P],
    "mgen_scale_bf16": [P, L, F, P, P],
    "mgen_kv_append": [P, P, L, L, P, P, P, I, I, I, I, I, P],
    "mgen_attn_decode": [P, L, P, P, P, P, L, P, I, I, I, I, I, I, F, P],
    "mgen_gemm_bf16_skinny": [P, P, P, I, I, I, L, L, L, I, L, I, P],
    "mgen_decode_layer": [P] * 22 + [I] * 8 + [F, I, P],
    "mgen_decode_qkv_prep": [P, L, P, L, P, P, P, P, P, P, I, I, I, I, I, F, I, P],
    "mgen_attn_decode_prep": [P, L, P, P, P, P, F, I, P, P, P, P, L, P, I, I, I, I, I, I, F, P],
    "mgen_kv_append_mx": [P, P, L, L, P, P, P, P, P, I, I, I, I, I, I, P],
    "mgen_kv_read_mx": [P, P, P, P, P, P, P, L, L, I, I, I, I, I, I, P],
    "mgen_attn_decode_mx_splits": [I, I, I, I, I],
    "mgen_attn_decode_mx": [P, L, P, P, P, P, P, P, L, P, I, I, I, I, I, I, I, F, P],
    "mgen_attn_decode_prep_mx": [P, L, P, P, P, I, P, F, I, P, P, P, P, P, P, L, P, I, I, I, I, I, I, I, F, P],
    "mgen_decode_layer_mx": [P] * 18 + [I] + [P] * 6 + [I] * 9 + [F, I, P],
    "mgen_sample_rows": [P, L, I, I, I, I, F, I, F, P, L, U64, U64, I, P, P, L, P],
    "mgen_sample": [P, L, I, I, I, I, F, I, F, P, L, U64, U64, P, P, L, P],
    "mgen_sample_step": [P, L, I, I, I, I, F, I, F, P, L, U64, U64, I, P, P, L, P, P, L, L, P],
    "mgen_decode_advance": [P, P, I, P, P],
    "mgen_philox_exponential": [P, L, I, I, U64, U64, P],
}

_lib = None


class MgenError(RuntimeError):
    pass


def _check_source_id(l):
    """The in-tree library must have been built from the sources beside it: a library left behind by a failed or
    interrupted build would otherwise run in place of the kernels one is looking at. Skipped for a library named by
    MGEN_LIB (another build on purpose) and when the sources are not there (an installed package)."""
    csrc = os.path.join(_HERE, "..", "csrc")
    if os.environ.get("MGEN_LIB") or not os.path.isdir(csrc):
        return
    from ._srcid import source_id
    if not hasattr(l, "mgen_source_id"):
        raise MgenError(f"{LIB_PATH} predates its sources (no mgen_source_id): run `make -C symbolic-music-generation_amd/csrc`")
    l.mgen_source_id.restype = ctypes.c_char_p
    l.mgen_source_id.argtypes = []
    built, here = l.mgen_source_id().decode(), source_id(csrc)
    if built != here:
        raise MgenError(
            f"{LIB_PATH} was built from other sources (library {built}, {os.path.normpath(csrc)} {here}): "
            "run `make -C symbolic-music-generation_amd/csrc`")


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise MgenError(
                f"{LIB_PATH} not found: build it with `make -C symbolic-music-generation_amd/csrc` "
                "(the HIP kernel library is required; there is no CPU fallback)")
        l = ctypes.CDLL(LIB_PATH)
        for name, args in SIGNATURES.items():
            fn = getattr(l, name)
            fn.argtypes = args
            fn.restype = ctypes.c_int
        l.mgen_last_error.restype = ctypes.c_char_p
        l.mgen_last_error.argtypes = []
        l.mgen_version.restype = ctypes.c_int
        _check_source_id(l)
        l.mgen_sumsq_partial_count.restype = ctypes.c_int
        l.mgen_gemm_slab_count.argtypes = [I, I]
        l.mgen_gemm_slab_count.restype = ctypes.c_int
        l.mgen_lmhead_ce_workspace_bytes.argtypes = [L, I, L]
        l.mgen_lmhead_ce_workspace_bytes.restype = ctypes.c_long
        l.mgen_decode_layer_fits.argtypes = [I] * 6
        l.mgen_decode_layer_fits.restype = ctypes.c_int
        l.mgen_gemm_skinny_fits.argtypes = [I, I, I, L, L, L, I]
        l.mgen_gemm_skinny_fits.restype = ctypes.c_int
        l.mgen_gemm_skinny_slabs.argtypes = [I, I, I]
        l.mgen_gemm_skinny_slabs.restype = ctypes.c_int
        l.mgen_attn_decode_workspace.argtypes = [I, I, I, I]
        l.mgen_attn_decode_workspace.restype = ctypes.c_long
        l.mgen_device_info.argtypes = [I, ctypes.c_char_p, I]
        l.mgen_device_info.restype = ctypes.c_int
        _lib = l
    return _lib


def call(name, *args):
    l = lib()
    rc = getattr(l, name)(*args)
    if rc != 0:
        raise MgenError(f"{name} failed ({rc}): {l.mgen_last_error().decode()}")
