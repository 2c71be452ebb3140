"""ctypes binding of the C-ABI library (include/instascene_rasterizer.h,
include/instascene_ops.h).  The library is the product: if it is missing or a
symbol cannot be resolved this module raises — there is no CPU or PyTorch
fallback anywhere in ``instascene_amd``.
"""
from __future__ import annotations

import ctypes
import os
import subprocess
from ctypes import c_char_p, c_float, c_int, c_int32, c_int64, c_size_t, c_uint, c_uint8, c_void_p

_HERE = os.path.dirname(os.path.abspath(__file__))
# ISR_LIB_PATH: an A/B build of the library (tools/build_variant.sh); default = the in-tree build
LIB_PATH = os.environ.get("ISR_LIB_PATH") or os.path.join(_HERE, "libinstascene_hip.so")
_lib = None

MODE_EXACT, MODE_FAST = 0, 1
MODE_PREBINNED = 0x100
MODE_FEATURE_ONLY = 0x200
GRAD_EXTRA, GRAD_GEOMETRY = 1, 2

# every exported symbol and its signature (tests/test_abi.py static_asserts each one against include/*.h with g++)
_P = c_void_p
SIGNATURES = {
    "isr_last_error": (c_char_p, []),
    "isr_version": (c_int, []),
    "isr_set_debug": (c_int, [c_int, c_int]),
    "isr_profile_enable": (None, [c_int]),
    "isr_forward_set_counters": (None, [_P]),
    "isr_backward_set_counters": (None, [_P]),
    "isr_profile_summary": (c_size_t, [_P, c_size_t]),
    "isr_geom_bytes": (c_size_t, [c_int]),
    "isr_image_bytes": (c_size_t, [c_int, c_int]),
    "isr_binning_bytes": (c_size_t, [c_int64, c_int, c_int]),
    "isr_backward_scratch_bytes": (c_size_t, [c_int64, c_int, c_uint]),
    "isr_forward_prepare": (c_int, [c_int, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, c_float, _P, _P, _P, _P, _P,
                                    c_float, c_float, c_int, _P, _P, _P, _P, _P]),
    "isr_read_num_rendered": (c_int, [_P, _P, _P]),
    "isr_forward_bin": (c_int, [c_int, c_int, c_int, _P, _P, c_int64, _P, _P]),
    "isr_forward_bin_event": (c_int, [c_int, c_int, c_int, _P, _P, c_int64, _P, _P, _P]),
    "isr_forward_render": (c_int, [c_int, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, _P, c_int64, _P, _P, _P, _P,
                                   _P, c_int64, _P, _P]),
    "isr_forward_render_scaled": (c_int, [c_int, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, _P, _P, c_int64, _P, _P, _P, _P,
                                          _P, c_int64, _P, _P]),
    "isr_row_scales": (c_int, [c_int, c_int, c_float, c_float, _P, _P, _P]),
    "isr_backward": (c_int, [c_int, c_int, c_int, c_int64, c_int, c_int, c_int, c_int, c_uint,
                             _P, _P, _P, _P, _P, c_float, _P, _P, _P, _P, _P, _P, c_float, c_float, _P,
                             _P, _P, _P, _P, _P, _P,
                             _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
                             _P, c_size_t, _P]),
    "isr_backward_sampled_scratch_bytes": (c_size_t, [c_int64, c_int, c_int, c_int, c_int]),
    "isr_sample_extra": (c_int, [c_int, c_int, c_int, c_int, _P, _P, _P, _P]),
    "isr_backward_sampled": (c_int, [c_int, c_int64, c_int, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, _P, _P, c_int, _P,
                                     c_size_t, _P]),
    "isr_feature_rows_step": (c_int, [c_int, c_int, c_int, c_int64, c_int, _P, _P, _P, _P, _P, _P, c_float, c_float, _P, _P, ctypes.c_double,
                                      ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_longlong, _P, _P, _P, _P,
                                      _P]),
    "isr_feature_rows_step_scaled": (c_int, [c_int, c_int, c_int, c_int64, c_int, _P, _P, _P, _P, _P, _P, c_float, c_float, _P, _P,
                                             ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_longlong,
                                             _P, _P, _P, _P, _P, _P]),
    "isr_seg_step_tail": (c_int, [c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_int64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
                                  c_float, c_float, c_float, c_float, _P, _P, _P, _P, _P, ctypes.c_double, ctypes.c_double,
                                  ctypes.c_double, ctypes.c_double, ctypes.c_longlong, c_float, c_float, _P, c_int, _P, c_size_t, _P, _P,
                                  _P, _P, _P, c_size_t, _P, _P, _P, _P, _P]),
    "isr_rgb_step_tail": (c_int, [c_int, c_int, c_int, c_int, c_int, c_int, c_int64, _P, _P, _P, _P, _P, _P, _P, c_float, c_float,
                                  c_float, c_float, _P, _P, _P, _P, _P, _P, c_float, _P, _P, _P, _P, c_float, c_float, _P, _P, _P, _P,
                                  _P, _P, _P, _P, ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_longlong, _P, _P, _P, _P,
                                  _P, _P, _P, c_size_t, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, c_size_t, _P,
                                  _P]),
    "isr_mark_visible": (c_int, [c_int, _P, _P, _P, _P, _P]),
    "isr_debug_state": (c_int, [c_int, c_int, c_int, c_int64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "isr_debug_check_hit_masks": (c_int, [c_int, c_int, c_int, c_int64, _P, _P, _P, _P, _P]),
    # include/instascene_ops.h
    "iso_knn_scratch_bytes": (c_size_t, [c_int]),
    "iso_dist2_3nn": (c_int, [c_int, _P, _P, _P, c_size_t, _P]),
    "iso_contrastive_scratch_bytes": (c_size_t, [c_int, c_int, c_int]),
    "iso_contrastive_forward": (c_int, [c_int, c_int, c_int, _P, _P, c_int, _P, c_int, c_int, c_float, _P, _P, c_size_t, _P]),
    "iso_contrastive_backward": (c_int, [c_int, c_int, c_int, c_int, _P, _P, _P, c_size_t, _P]),
    "iso_contrastive_forward_batch": (c_int, [c_int, c_int, c_int, c_int, _P, _P, c_int, _P, c_int, c_int, c_float, _P, _P, _P,
                                              _P, c_size_t, _P]),
    "iso_contrastive_backward_batch": (c_int, [c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, c_size_t, _P]),
    "iso_rownorm": (c_int, [ctypes.c_longlong, c_int, c_float, c_int, _P, _P, _P, _P]),
    "iso_render_post_forward": (c_int, [c_int, c_int, c_float] + [_P] * 11 + [_P]),
    "iso_render_post_backward": (c_int, [c_int, c_int, c_float] + [_P] * 14 + [_P]),
    "iso_ssim_scratch_bytes": (c_size_t, [c_int, c_int, c_int]),
    "iso_ssim_forward": (c_int, [c_int, c_int, c_int, _P, _P, _P, _P, _P, c_size_t, _P]),
    "iso_ssim_backward": (c_int, [c_int, c_int, c_int, _P, _P, _P, _P, _P, _P]),
    "iso_photometric_forward": (c_int, [c_int, c_int, c_int, _P, _P, _P, _P, _P, _P, c_size_t, _P]),
    "iso_photometric_backward": (c_int, [c_int, c_int, c_int, _P, _P, _P, _P, _P, _P, _P]),
    "iso_train_loss_scratch_bytes": (c_size_t, [c_int, c_int, c_int]),
    "iso_train_loss_forward": (c_int, [c_int, c_int, c_int, _P, _P, c_float, _P, _P, c_float, _P, c_float, _P, _P, _P, c_size_t, _P]),
    "iso_train_loss_backward": (c_int, [c_int, c_int, c_int, _P, _P, _P, c_float, _P, _P, c_float, c_float, _P, _P, _P, _P, _P, _P]),
    "iso_densify_stats": (c_int, [c_int, c_int, _P, _P, _P, _P, _P, _P, _P]),
    "iso_gaussian_adam_step": (c_int, [c_int, c_int, _P, _P, _P, _P, ctypes.c_double, ctypes.c_double, ctypes.c_double,
                                       ctypes.c_longlong, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "iso_gather_rownorm": (c_int, [c_int, c_int, ctypes.c_longlong, c_float, _P, _P, _P, _P]),
    "iso_sample_step": (c_int, [ctypes.c_ulonglong, ctypes.c_ulonglong, c_int, ctypes.c_longlong, _P, _P, _P, ctypes.c_longlong, _P,
                                _P, _P, _P, _P, _P, _P, _P]),
    "iso_rows_compact": (c_int, [c_int, c_int, ctypes.c_longlong, _P, _P, _P, _P, _P, c_int, _P]),
    "iso_adam_rownorm2": (c_int, [ctypes.c_longlong, c_int, ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_double,
                                  ctypes.c_longlong, c_float,
                                  c_float, _P, _P, _P, _P, _P, _P, _P]),
    "iso_peer_sum": (c_int, [c_int, _P, ctypes.c_longlong, ctypes.c_longlong, _P, _P]),
    "iso_ipc_alloc": (c_int, [c_size_t, _P, _P]),
    "iso_ipc_open": (c_int, [_P, _P]),
    "iso_ipc_close": (c_int, [_P, c_int]),
    "iso_enable_peer_access": (c_int, [c_int]),
    "iso_flag_set": (c_int, [_P, c_uint, _P]),
    "iso_flag_wait": (c_int, [c_int, _P, c_int, c_uint, _P, c_int, _P]),
    "iso_rows_pack": (c_int, [c_int, c_int, _P, _P, _P, _P, _P, _P]),
    "iso_rows_scatter_add": (c_int, [c_int, c_int, ctypes.c_longlong, _P, _P, _P, _P, c_int, _P]),
    "iso_rms_norm_forward": (c_int, [c_int, ctypes.c_longlong, c_int, _P, ctypes.c_longlong, _P, ctypes.c_longlong, _P, c_int, c_float, _P,
                                     _P, _P, _P]),
    "iso_rms_norm_quant": (c_int, [c_int, c_int, ctypes.c_longlong, c_int, c_int, _P, ctypes.c_longlong, _P, ctypes.c_longlong, _P, c_int,
                                   c_float, _P, _P, _P, _P]),
    "iso_rms_norm_scratch_bytes": (c_size_t, [c_int, ctypes.c_longlong, c_int]),
    "iso_rms_norm_backward": (c_int, [c_int, ctypes.c_longlong, c_int, _P, ctypes.c_longlong, _P, ctypes.c_longlong, _P, c_int, _P, _P, ctypes.c_longlong, _P,
                                      ctypes.c_longlong, _P, _P, _P, c_size_t, _P]),
    "iso_rows8_write": (c_int, [c_int, c_int, ctypes.c_longlong, c_int, c_int, ctypes.c_longlong, _P, ctypes.c_longlong, ctypes.c_longlong,
                                _P, c_int, _P, _P, _P, _P]),
    "iso_rows8_read": (c_int, [c_int, c_int, ctypes.c_longlong, c_int, c_int, ctypes.c_longlong, _P, _P, ctypes.c_longlong, _P, c_int, c_int,
                               c_float, _P, _P]),
    "iso_grad_norm_scratch_bytes": (c_size_t, [c_int, _P]),
    "iso_grad_norm": (c_int, [c_int, _P, _P, _P, c_int, c_float, c_int, _P, _P, c_size_t, _P]),
    "iso_gaussian_grad_norm": (c_int, [c_int, c_int, _P, _P, _P, _P, _P, _P, c_float, _P, _P, c_size_t, _P]),
    "iso_adam_rownorm2_clipped": (c_int, [ctypes.c_longlong, c_int, ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_double,
                                          ctypes.c_longlong, c_float, c_float, _P, _P, _P, _P, _P, _P, _P, _P]),
    "iso_gaussian_adam_step_clipped": (c_int, [c_int, c_int, _P, _P, _P, _P, ctypes.c_double, ctypes.c_double, ctypes.c_double,
                                               ctypes.c_longlong, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "iso_rownorm2": (c_int, [ctypes.c_longlong, c_int, c_float, c_float, c_int, _P, _P, _P, _P, _P, _P]),
}


def build(force: bool = False) -> str:
    """Compile the HIP library for gfx950 with hipcc (cross-compiles without a GPU)."""
    src_dir = os.path.join(_HERE, "csrc")
    args = ["make", "-C", src_dir, "-s", "-j", str(min(6, os.cpu_count() or 1))]
    if force:
        args.append("-B")
    subprocess.check_call(args)
    return LIB_PATH


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"instascene_amd: {LIB_PATH} is missing. Build it with `python -c 'import __graft_entry__ as g; "
                "g.build()'` (hipcc, --offload-arch=gfx950). There is no CPU fallback.")
        # torch first: it brings its own copy of the HIP runtime (same SONAME), and a process must end up with ONE runtime.
        # Loaded the other way round, the library binds /opt/rocm's copy and torch's kernels and ours no longer share
        # streams and devices ("no ROCm-capable device is detected" from the second runtime).
        import torch  # noqa: F401
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)        # AttributeError if the symbol is not exported: fail loudly
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


class IsrError(RuntimeError):
    """Mirrors the reference's RuntimeError raised from C++ (AT_ERROR / std::runtime_error)."""


def check(rc: int, what: str):
    if rc != 0:
        msg = lib().isr_last_error()
        raise IsrError(f"{what} failed (code {rc}): {msg.decode() if msg else ''}")
