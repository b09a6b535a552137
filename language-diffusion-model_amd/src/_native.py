"""ctypes binding of ``libldm_hip.so`` (the C ABI declared in ``include/ldm_hip.h``).

There is no CPU fallback: if the library is missing, or a tensor handed to an
op is not on a ROCm device, the call raises.
"""

from __future__ import annotations

import ctypes as C
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("LDM_LIB") or os.path.join(os.path.dirname(_HERE), "lib", "libldm_hip.so")

F32, BF16 = 0, 1
ABI_VERSION = 23   # what ldm_abi_version() of a matching library returns
DTYPE_CODE = {torch.float32: F32, torch.bfloat16: BF16}

_vp, _i64, _i32, _f32, _u64, _f64 = C.c_void_p, C.c_int64, C.c_int, C.c_float, C.c_uint64, C.c_double


class BStride(C.Structure):
    _fields_ = [("outer", C.c_int64), ("inner", C.c_int64)]


class AdamWTensor(C.Structure):     # ldm_adamw_tensor
    _fields_ = [("p", C.c_void_p), ("g", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p),
                ("shadow", C.c_void_p), ("n", C.c_int64), ("shadow_kind", C.c_int32)]


# name -> (restype, argtypes); kept in sync with include/ldm_hip.h
SIGNATURES = {
    "ldm_abi_version": (_i32, []),
    "ldm_error_string": (C.c_char_p, [_i32]),
    "ldm_mask_fwd": (_i32, [_vp, _vp, _i32, _f32, _vp, _f32, _i64, _i64, _i64, _i64, _i64, _i64, _u64, _u64,
                            _vp, _vp, _vp]),
    "ldm_embed_fwd": (_i32, [_vp, _vp, _i64, _i64, _i64, _vp, _i32, _vp]),
    "ldm_embed_bwd": (_i32, [_vp, _vp, _i32, _i64, _i64, _i64, _i64, _vp, _vp]),
    "ldm_rmsnorm_fwd": (_i32, [_vp, _vp, _i64, _i64, _f32, _i32, _vp, _vp, _vp]),
    "ldm_rmsnorm_bwd_ws_floats": (_i64, [_i64, _i64]),
    "ldm_rmsnorm_bwd": (_i32, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _vp, _vp, _vp, _vp]),
    "ldm_rmsnorm_bwd_dropgrad": (_i32, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _vp, _vp, _f32, _u64, _vp, _vp, _vp]),
    "ldm_rmsnorm_fwd_f32_bf16": (_i32, [_vp, _vp, _i64, _i64, _f32, _vp, _vp, _vp]),
    "ldm_rmsnorm_bwd_f32_bf16": (_i32, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp]),
    "ldm_rmsnorm_bwd_noalloc_max_d": (_i64, []),
    "ldm_rmsnorm_bwd_noalloc": (_i32, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _vp, _vp, _vp]),
    "ldm_rope_qk": (_i32, [_vp, _i32, _i64, _i64, _i64, _i64, _i64, _vp, _vp, _f32, _i32, _vp]),
    "ldm_swiglu_fwd": (_i32, [_vp, _i64, _i64, _i32, _vp, _vp]),
    "ldm_swiglu_bwd": (_i32, [_vp, _vp, _i64, _i64, _i32, _vp, _vp]),
    "ldm_gemm": (_i32, [_i32, _i32, _i32, _i32, _i64, _i64, _i64, _f32, _vp, _i64, _vp, _i64, _vp, _i64,
                        _vp, _vp, _i64, _vp]),
    "ldm_gemm_acc": (_i32, [_i32, _i32, _i32, _i64, _i64, _i64, _f32, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    "ldm_gemm_batched": (_i32, [_i32, _i32, _i32, _i32, _i64, _i64, _i64, _f32, _vp, _i64, BStride, _vp, _i64,
                                BStride, _vp, _i64, BStride, _i64, _i64, _vp]),
    "ldm_colsum_ws_floats": (_i64, [_i64, _i64]),
    "ldm_colsum": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _vp]),
    "ldm_cast_f32_to_bf16": (_i32, [_vp, _vp, _i64, _vp]),
    "ldm_transpose_bf16": (_i32, [_vp, _i64, _vp, _i64, _i64, _i64, _vp]),
    "ldm_attn_saved_bytes": (_i64, [_i32, _i64, _i64, _i64, _i64]),
    "ldm_attn_bwd_ws_bytes": (_i64, [_i32, _i64, _i64, _i64, _i64]),
    "ldm_attn_fwd": (_i32, [_i32, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _i64, _vp, _vp]),
    "ldm_attn_bwd": (_i32, [_i32, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _vp]),
    "ldm_attn_bwd_unrope": (_i32, [_i32, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp,
                                   _f32, _vp]),
    "ldm_gemm_swiglu_fwd": (_i32, [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp]),
    "ldm_gemm_qkv_rope": (_i32, [_i64, _i64, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _f32, _vp, _i64,
                                 _vp]),
    "ldm_dropout_add": (_i32, [_vp, _vp, _vp, _i64, _i64, _i32, _f32, _u64, _vp]),
    "ldm_gemm_dropout_residual": (_i32, [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _f32, _u64, _vp]),
    "ldm_attn_fwd_dropout": (_i32, [_i32, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _i64, _vp, _vp, _f32, _u64, _vp]),
    "ldm_attn_fwd_addmask": (_i32, [_i32, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _i64, _vp,
                                    _vp, _f32, _u64, _vp]),
    "ldm_attn_bwd_dropout": (_i32, [_i32, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp,
                                    _f32, _f32, _u64, _vp]),
    "ldm_rmsnorm_fp8": (_i32, [_vp, _i32, _i64, _vp, _i32, _i64, _vp, _i64, _i64, _f32, _vp, _vp, _i64, _vp, _i64, _vp]),
    "ldm_quant_fp8": (_i32, [_vp, _i32, _i64, _i64, _i64, _i32, _vp, _i64, _vp, _i64, _vp]),
    "ldm_quant_fp8_block": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp]),
    "ldm_gemm_fp8": (_i32, [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp]),
    "ldm_gemm_fp8_f32": (_i32, [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp]),
    "ldm_ce_fwd": (_i32, [_vp, _i32, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _i32, _vp, _vp,
                          _vp, _vp, _vp]),
    "ldm_ce_bwd": (_i32, [_vp, _i32, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _i32, _vp, _vp,
                          _vp, _vp, _i64, _vp]),
    "ldm_ce_compact_rows": (_i32, [_i64, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp]),
    "ldm_sample_tokens": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _i64, _i32, _f32, _u64, _u64, _vp, _vp, _vp]),
    "ldm_sample_filtered": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _i64, _f64, _i64, _f64, _f64, _vp, _vp]),
    "ldm_remask_eligible": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp]),
    "ldm_remask_apply": (_i32, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp]),
    "ldm_ce_bwd_compact": (_i32, [_vp, _i32, _i64, _i64, _i64, _i64, _vp, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp,
                                  _i64, _vp]),
    "ldm_ce_fwd_grad": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _i32, _f32, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ldm_scale_rows_dev": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _vp]),
    "ldm_adamw_step": (_i32, [C.POINTER(AdamWTensor), _i64, _i64, _f32, _f32, _f32, _f32, _f32, _f32, _vp]),
    "ldm_adamw_step_gated": (_i32, [C.POINTER(AdamWTensor), _i64, _i64, _f32, _f32, _f32, _f32, _f32, _f32, _vp, _vp,
                                    _vp]),
    "ldm_adamw_gate_commit": (_i32, [_vp, _vp, _vp]),
    "ldm_comm_unique_id": (_i32, [_vp]),
    "ldm_comm_init_rank": (_i32, [C.POINTER(_vp), _i32, _vp, _i32]),
    "ldm_comm_size": (_i32, [_vp, C.POINTER(_i32)]),
    "ldm_comm_destroy": (_i32, [_vp]),
    "ldm_comm_last_error": (C.c_char_p, []),
    "ldm_allreduce_bucket": (_i32, [_vp, _vp, _i64, _i32, _vp, _vp]),
    "ldm_allreduce_join": (_i32, [_vp, _vp]),
    "ldm_collate_pad": (_i32, [_vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp]),
    "ldm_synth_tokens": (_i32, [_i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _u64, _u64, _vp, _vp, _vp]),
    "ldm_gemm_swiglu_bwd": (_i32, [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    "ldm_gather_rows": (_i32, [_vp, _i32, _i64, _vp, _vp, _i64, _i64, _vp, _vp]),
    "ldm_scatter_rows": (_i32, [_vp, _i32, _i64, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp]),
    "ldm_gemm_rows_dyn": (_i32, [_i32, _i32, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp,
                                 _vp]),
    "ldm_gemm_acc_kdyn": (_i32, [_i32, _i32, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp]),
    "ldm_gemm_acc_rowsum": (_i32, [_i32, _i32, _i64, _i64, _i64, _f32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp]),
    "ldm_colsum_rows_dyn": (_i32, [_vp, _i32, _i64, _i64, _i64, _vp, _vp, _vp, _vp]),
    "ldm_softmax_rows_f32": (_i32, [_vp, _vp, _i64, _i64, _i64, _i64, _vp]),
    "ldm_softmax_bwd_rows_f32": (_i32, [_vp, _vp, _i64, _i64, _vp]),
}

_lib = None


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                "(or `make -C language-diffusion-model_amd`). There is no fallback path.")
        handle = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        got = handle.ldm_abi_version()
        if got != ABI_VERSION:
            raise RuntimeError(f"{LIB_PATH} has ABI version {got}, this package needs {ABI_VERSION}: rebuild it "
                               "(`make -C language-diffusion-model_amd`)")
        _lib = handle
    return _lib


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().ldm_error_string(rc).decode()
        if rc == -6:
            msg += ": " + lib().ldm_comm_last_error().decode()
        raise RuntimeError(f"{what} failed with code {rc}: {msg}")


def stream() -> int:
    # (the raw handle: building torch's Stream object costs 2.7 us a call)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def require_device(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "this operator runs only on a ROCm device (HIP kernels, no CPU fallback); "
                f"got a tensor on {t.device}")


def dtype_code(dt: torch.dtype) -> int:
    try:
        return DTYPE_CODE[dt]
    except KeyError:
        raise TypeError(f"unsupported compute dtype {dt}; use torch.float32 or torch.bfloat16") from None
