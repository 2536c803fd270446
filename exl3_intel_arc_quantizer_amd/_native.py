"""ctypes binding of ``libexl3_hip.so`` and the extension facade.

``QuantizeExtension`` mirrors the functions of the reference's pybind module
``quantize_xpu_ext`` (csrc/quantize_xpu/quantize_xpu.cpp:302-357) with the
same names, argument order, defaults and error behaviour (``RuntimeError``
for rejected tensors, as its ``TORCH_CHECK``s raise), but takes torch-ROCm
device tensors (``cuda:i``) and calls the C-ABI declared in
``include/exl3_encoder.h``. Work is enqueued on the tensor's current torch
stream; nothing here synchronises.

There is no CPU fallback: loading fails loudly when the library is missing.
"""

from __future__ import annotations

import ctypes
from pathlib import Path
from typing import Optional

from .build import LIB_PATH

_LIB = None

_c_int, _c_i64, _c_vp = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
_c_float, _c_double = ctypes.c_float, ctypes.c_double

# name -> (restype, argtypes)
_SIGNATURES = {
    "exl3_last_error": (ctypes.c_char_p, []),
    "exl3_version": (ctypes.c_char_p, []),
    "exl3_set_traceback_policy": (_c_int, [_c_int]),
    "exl3_decode_codebook": (_c_int, [_c_int, _c_vp, _c_vp]),
    "exl3_scratch_row_bytes": (_c_i64, [_c_int]),
    "exl3_scratch_edges_bytes": (_c_i64, [_c_int, _c_int, _c_i64]),
    "exl3_cost_row_slot": (_c_i64, [_c_int, _c_i64]),
    "exl3_quantize_tiles": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_int,
                                     _c_int, _c_int, _c_int, _c_i64, _c_vp]),
    "exl3_quantize_tiles_tb": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64,
                                        _c_int, _c_int, _c_int, _c_int, _c_i64, _c_int, _c_vp]),
    "exl3_quantize_tiles_noalloc": (_c_int, [_c_vp, _c_vp, _c_vp, _c_i64, _c_int, _c_int, _c_int,
                                             _c_int, _c_vp]),
    "exl3_forward_pass": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_int, _c_int, _c_int,
                                   _c_int, _c_int, _c_int, _c_vp]),
    "exl3_backward_pass": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_int, _c_int,
                                    _c_int, _c_int, _c_int, _c_int, _c_vp]),
    "exl3_prepare_tiles": (_c_int, [_c_vp, _c_vp, _c_i64, _c_int, _c_int, _c_vp, _c_vp]),
    "exl3_finalize_tiles": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp,
                                     _c_i64, _c_int, _c_int, _c_int, _c_vp]),
    "exl3_pack_trellis": (_c_int, [_c_vp, _c_vp, _c_i64, _c_int, _c_vp]),
    "exl3_unpack_trellis": (_c_int, [_c_vp, _c_vp, _c_i64, _c_int, _c_vp]),
    "exl3_probe_hfma": (_c_int, [_c_vp, _c_vp, _c_vp, _c_i64, _c_int, _c_vp]),
    # include/exl3_layer.h
    "exl3_hadamard128": (_c_int, [_c_vp, _c_vp, _c_i64, _c_i64, _c_int, _c_vp]),
    "exl3_hadamard128_scaled": (_c_int, [_c_vp, _c_vp, _c_i64, _c_i64, _c_int, _c_vp, _c_vp,
                                         _c_vp]),
    "exl3_row_energy": (_c_int, [_c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_vp]),
    "exl3_rotate": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_vp]),
    "exl3_unrotate": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_vp]),
    "exl3_decode_weight": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_int, _c_int,
                                    _c_vp]),
    "exl3_block_rms_from_slices": (_c_int, [_c_vp, _c_vp, _c_i64, _c_i64, _c_i64, _c_vp]),
    "exl3_input_scales": (_c_int, [_c_vp, _c_vp, _c_vp, _c_vp, _c_i64, _c_i64, _c_i64, _c_vp]),
    "exl3_output_scales": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_i64, _c_vp, _c_int,
                                    _c_int, _c_vp, _c_i64, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp]),
    "exl3_block_rms": (_c_int, [_c_vp, _c_vp, _c_i64, _c_i64, _c_int, _c_int, _c_vp, _c_i64,
                                _c_vp]),
    "exl3_block_rms_workspace": (_c_i64, [_c_i64, _c_i64, _c_int, _c_int]),
    "exl3_cholesky_diag_block": (_c_int, [_c_vp, _c_i64, _c_int, _c_i64, _c_vp, _c_vp]),
    "exl3_gram": (_c_int, [_c_vp, _c_int, _c_i64, _c_i64, _c_i64, _c_float, _c_vp, _c_vp, _c_i64,
                           _c_vp]),
    "exl3_gram_chunked": (_c_int, [_c_vp, _c_int, _c_i64, _c_i64, _c_i64, _c_float, _c_i64, _c_vp,
                                   _c_vp, _c_i64, _c_vp]),
    "exl3_gram_workspace": (_c_i64, [_c_i64, _c_i64]),
    "exl3_damp_diagonal": (_c_int, [_c_vp, _c_i64, _c_i64, _c_double, _c_float, _c_vp, _c_vp]),
    "exl3_cholesky_block_order": (_c_int, []),
    "exl3_cholesky": (_c_int, [_c_vp, _c_i64, _c_vp, _c_vp, _c_vp]),
    "exl3_cholesky_inverse_elems": (_c_i64, [_c_i64]),
    "exl3_block_fold": (_c_int, [_c_vp, _c_vp, _c_vp, _c_i64, _c_vp]),
    "exl3_ldlq_gather": (_c_int, [_c_vp, _c_int, _c_i64, _c_vp, _c_vp]),
    "exl3_ldlq_scatter": (_c_int, [_c_vp, _c_int, _c_i64, _c_vp, _c_vp, _c_vp]),
    "exl3_linear_workspace": (_c_i64, [_c_i64, _c_i64, _c_i64, _c_int]),
    "exl3_linear": (_c_int, [_c_vp, _c_i64, _c_i64, _c_int, _c_vp, _c_vp, _c_vp, _c_int, _c_i64,
                             _c_i64, _c_int, _c_int, _c_vp, _c_vp, _c_i64, _c_vp]),
    # the attention cache of include/exl3_layer.h
    "exl3_rotary": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_i64, _c_int,
                             _c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_i64, _c_int, _c_i64,
                             _c_int, _c_int, _c_vp, _c_int, _c_vp, _c_int, _c_int, _c_float,
                             _c_int, _c_vp]),
    "exl3_rotary_axes": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_i64, _c_int,
                                  _c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_i64, _c_int, _c_i64,
                                  _c_int, _c_int, _c_vp, _c_int, _c_vp, _c_int, _c_vp, _c_int,
                                  _c_int, _c_float, _c_int, _c_vp]),
    "exl3_plan_step": (_c_int, [_c_vp, _c_vp, _c_int, _c_vp, _c_int, _c_vp, _c_int, _c_vp, _c_int,
                                _c_i64, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp, _c_vp]),
    "exl3_cache_append": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_int, _c_vp, _c_i64, _c_i64,
                                   _c_vp, _c_i64, _c_i64, _c_i64, _c_int, _c_vp, _c_vp, _c_int,
                                   _c_vp, _c_int, _c_int, _c_float, _c_vp, _c_i64, _c_int, _c_int,
                                   _c_int, _c_vp]),
    "exl3_cache_append_axes": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_int, _c_vp, _c_i64,
                                        _c_i64, _c_vp, _c_i64, _c_i64, _c_i64, _c_int, _c_vp,
                                        _c_vp, _c_int, _c_vp, _c_int, _c_vp, _c_int, _c_int,
                                        _c_float, _c_vp, _c_i64, _c_int, _c_int, _c_int, _c_vp]),
    "exl3_cache_read": (_c_int, [_c_vp, _c_i64, _c_int, _c_int, _c_int, _c_vp, _c_i64, _c_int,
                                 _c_vp, _c_vp, _c_vp]),
    "exl3_cache_attention_workspace": (_c_i64, [_c_i64, _c_int, _c_int, _c_int, _c_int, _c_i64]),
    "exl3_cache_attention_trees_workspace": (_c_i64, [_c_i64, _c_int, _c_int, _c_int, _c_int, _c_i64]),
    "exl3_cache_attention": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_int, _c_int, _c_vp,
                                      _c_i64, _c_int, _c_int, _c_int, _c_vp, _c_int, _c_vp, _c_vp,
                                      _c_int, _c_float, _c_i64, _c_i64, _c_vp, _c_i64, _c_vp]),
    "exl3_cache_attention_trees": (_c_int, [_c_vp, _c_i64, _c_i64, _c_vp, _c_i64, _c_int, _c_int,
                                            _c_vp, _c_i64, _c_int, _c_int, _c_int, _c_vp, _c_int,
                                            _c_vp, _c_vp, _c_int, _c_vp, _c_int, _c_float, _c_i64,
                                            _c_i64, _c_vp, _c_i64, _c_vp]),
    "exl3_plan_tree": (_c_int, [_c_vp, _c_vp, _c_vp, _c_int, _c_i64, _c_int, _c_vp, _c_vp, _c_vp]),
    "exl3_accept_drafts": (_c_int, [_c_vp, _c_vp, _c_int, _c_vp, _c_vp, _c_vp, _c_vp, _c_int,
                                    _c_i64, _c_vp, _c_vp, _c_vp, _c_vp]),
    "exl3_accept_trees": (_c_int, [_c_vp, _c_vp, _c_int, _c_vp, _c_vp, _c_vp, _c_vp, _c_int,
                                   _c_i64, _c_int, _c_vp, _c_vp, _c_vp, _c_vp]),
    "exl3_cache_keep": (_c_int, [_c_vp, _c_i64, _c_int, _c_int, _c_int, _c_vp, _c_vp, _c_vp, _c_int,
                                 _c_i64, _c_vp]),
    "exl3_release_pages": (_c_int, [_c_vp, _c_vp, _c_int, _c_vp, _c_int, _c_int, _c_vp, _c_int,
                                    _c_vp, _c_vp, _c_vp]),
}


def exported_symbols() -> list:
    """C-ABI entry points declared in include/exl3_encoder.h and
    include/exl3_layer.h."""
    return sorted(_SIGNATURES)


def load_library(path: Optional[Path] = None):
    """Load the native library (no build, no fallback)."""
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    lib_path = Path(path) if path is not None else LIB_PATH
    if not lib_path.exists():
        raise RuntimeError(
            f"native encoder library {lib_path} is missing; build it with "
            "`python -m exl3_intel_arc_quantizer_amd.build` (hipcc, gfx950)")
    lib = ctypes.CDLL(str(lib_path))
    for name, (restype, argtypes) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    if path is None:
        _LIB = lib
    return lib



TRACEBACK_POLICIES = {"auto": 0, "rows": 1, "stream": 2}


def _policy_code(policy: Optional[str]) -> int:
    """C-ABI code of a traceback policy name; None = the process default (-1)."""
    if policy is None:
        return -1
    if policy not in TRACEBACK_POLICIES:
        raise ValueError(f"policy must be one of {sorted(TRACEBACK_POLICIES)}, got {policy!r}")
    return TRACEBACK_POLICIES[policy]


def set_traceback_policy(policy: str) -> str:
    """Choose the default traceback kernel for later calls in this process
    that do not name one: "auto" (by batch size), "rows" (per-row tree
    loads) or "stream" (whole rows streamed through LDS); results are
    identical. Returns the previous default. ``quantize_tiles(...,
    traceback_policy=...)`` chooses per call without changing it."""
    if policy is None:
        raise ValueError("set_traceback_policy needs a policy name")
    prev = load_library().exl3_set_traceback_policy(_policy_code(policy))
    return {v: k for k, v in TRACEBACK_POLICIES.items()}[prev]

def last_error() -> str:
    return load_library().exl3_last_error().decode()


def _check(status: int, what: str) -> None:
    if status != 0:
        raise RuntimeError(f"{what}: {last_error()}")


# ------------------------------------------------------------- validation

_TORCH = None


def _torch():
    """torch, imported on first use and then held: a small call's checks ask for it
    up to ten times, and the import statement alone takes 0.1 us."""
    global _TORCH
    if _TORCH is None:
        import torch
        _TORCH = torch
    return _TORCH


def _check_device_tensor(t, name: str, dtype, ndim: int) -> int:
    """TORCH_CHECK equivalents of check_xpu_tensor (quantize_xpu.cpp:73-83)."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be a GPU (cuda) tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} has wrong dtype")
    if t.dim() != ndim:
        raise RuntimeError(f"{name} must be {ndim}-D, got {t.dim()}-D")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _check_buffer(t, name: str, dtype, shape, dev: int) -> None:
    """A device tensor of exactly ``shape`` on device ``dev``: every buffer a
    kernel indexes by the launch's sizes is checked before the launch."""
    if _check_device_tensor(t, name, dtype, len(shape)) != dev:
        raise RuntimeError(f"{name} must be on the same GPU device")
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _resolve_cb(mcg: bool, mul1: bool) -> int:
    """quantize_xpu.cpp:85-91."""
    if mcg and mul1:
        raise RuntimeError("mcg and mul1 cannot both be true (ambiguous codebook)")
    return 2 if mul1 else (1 if mcg else 0)


def _validate_common(K: int, cb: int, L: int, sg_size: int) -> None:
    """quantize_xpu.cpp:93-101. sg_size is accepted for API parity; wave64
    hardware has no sub-group width choice."""
    if not 1 <= K <= 8:
        raise RuntimeError(f"K must be in 1..8, got {K}")
    if L not in (256, 160):
        raise RuntimeError(f"tile length L must be 256 or 160, got {L}")
    if L == 160 and cb != 2:
        raise RuntimeError("tile length L=160 is only supported with mul1 (cb=2)")
    if sg_size not in (16, 32):
        raise RuntimeError(f"sg_size must be 16 or 32, got {sg_size}")


def _stream(device_index: int) -> int:
    torch = _torch()
    return torch.cuda.current_stream(device_index).cuda_stream


def row_bytes(K: int) -> int:
    """Bytes of one scratch row at bitrate K."""
    return int(load_library().exl3_scratch_row_bytes(K))


def tile_rows(K: int, L: int = 256) -> int:
    """Scratch rows per tile (stored cost rows or ring rows, plus a header)."""
    lib = load_library()
    return int(lib.exl3_scratch_edges_bytes(K, L, 1) // lib.exl3_scratch_row_bytes(K))


def edges_shape(B: int, K: int, L: int = 256) -> tuple:
    """Shape of a uint8 ``temp_edges`` scratch tensor for B tiles."""
    return (B, tile_rows(K, L), row_bytes(K))


class QuantizeExtension:
    """Drop-in for the reference's ``quantize_xpu_ext`` module object."""

    def __init__(self, lib=None):
        self.lib = lib or load_library()

    # quantize_xpu.cpp:105-110
    def decode_codebook(self, cb: int, out_lut) -> None:
        torch = _torch()
        if not 0 <= cb <= 2:
            raise RuntimeError("cb must be 0, 1, or 2")
        dev = _check_device_tensor(out_lut, "out_lut", torch.float16, 1)
        if out_lut.size(0) != 65536:
            raise RuntimeError("out_lut must have length 65536")
        with torch.cuda.device(dev):
            _check(self.lib.exl3_decode_codebook(cb, out_lut.data_ptr(), _stream(dev)),
                   "decode_codebook")

    def _scratch_checks(self, temp_costs, temp_edges, K: int, L: int, dev: int) -> int:
        torch = _torch()
        if _check_device_tensor(temp_costs, "temp_costs", torch.float16, 3) != dev:
            raise RuntimeError("temp_costs must be on the same GPU device as input_tiles")
        if _check_device_tensor(temp_edges, "temp_edges", torch.uint8, 3) != dev:
            raise RuntimeError("temp_edges must be on the same GPU device as input_tiles")
        edges = 65536 >> K
        batch_cap = temp_costs.size(0)
        if batch_cap < 1:
            raise RuntimeError("temp_costs batch dimension B must be >= 1")
        if temp_costs.size(1) != 2 or temp_costs.size(2) != edges:
            raise RuntimeError("temp_costs must have shape (B, 2, 65536 >> K)")
        _, rows, rb = edges_shape(batch_cap, K, L)
        if (temp_edges.size(0) < batch_cap or temp_edges.size(1) != rows
                or temp_edges.size(2) != rb):
            raise RuntimeError(
                f"temp_edges must have shape (B, {rows}, {rb}) for K={K}, L={L} "
                "(cost-row scratch layout)")
        return batch_cap

    # quantize_xpu.cpp:112-167
    def quantize_tiles(self, input_tiles, output_tiles, output_indices, temp_costs, temp_edges,
                       K: int, mcg: bool, mul1: bool, sg_size: int = 32,
                       force_global_costs: bool = False, wave_cap_override: int = 0,
                       traceback_policy: Optional[str] = None) -> None:
        """The reference's arguments, plus ``traceback_policy`` (no counterpart
        there): the traceback kernel for this call only, "auto", "rows",
        "stream", or None for the process default."""
        torch = _torch()
        cb = _resolve_cb(mcg, mul1)
        tb = _policy_code(traceback_policy)
        dev = _check_device_tensor(input_tiles, "input_tiles", torch.float32, 2)
        if _check_device_tensor(output_tiles, "output_tiles", torch.float32, 2) != dev:
            raise RuntimeError("output_tiles must be on the same GPU device as input_tiles")
        if _check_device_tensor(output_indices, "output_indices", torch.int16, 2) != dev:
            raise RuntimeError("output_indices must be on the same GPU device as input_tiles")
        n, L = input_tiles.shape
        if n <= 0:
            raise RuntimeError(f"num_tiles must be positive, got {n}")
        _validate_common(K, cb, L, sg_size)
        batch_cap = self._scratch_checks(temp_costs, temp_edges, K, L, dev)
        if tuple(output_tiles.shape) != (n, L):
            raise RuntimeError("output_tiles shape must match input_tiles")
        if tuple(output_indices.shape) != (n, L):
            raise RuntimeError("output_indices shape must match input_tiles")
        with torch.cuda.device(dev):
            _check(self.lib.exl3_quantize_tiles_tb(
                input_tiles.data_ptr(), output_tiles.data_ptr(), output_indices.data_ptr(),
                temp_costs.data_ptr(), temp_edges.data_ptr(), batch_cap, n, K, cb, L,
                int(bool(force_global_costs)), int(wave_cap_override), tb, _stream(dev)),
                "quantize_tiles")

    # quantize_xpu.cpp:169-215
    def quantize_tiles_forward_pass(self, input_tiles, temp_costs, temp_edges, pre_states,
                                    K: int, mcg: bool, mul1: bool, roll: int, cost_slot: int = 0,
                                    sg_size: int = 32, force_global_costs: bool = False) -> None:
        torch = _torch()
        cb = _resolve_cb(mcg, mul1)
        dev = _check_device_tensor(input_tiles, "input_tiles", torch.float32, 2)
        if _check_device_tensor(pre_states, "pre_states", torch.int32, 1) != dev:
            raise RuntimeError("pre_states must be an int32 GPU tensor")
        n, L = input_tiles.shape
        _validate_common(K, cb, L, sg_size)
        batch_cap = self._scratch_checks(temp_costs, temp_edges, K, L, dev)
        if not 0 < n <= batch_cap:
            raise RuntimeError("num_tiles must be in 1..B")
        if pre_states.size(0) < n:
            raise RuntimeError("pre_states length must be >= num_tiles")
        if cost_slot not in (0, 1):
            raise RuntimeError("cost_slot must be 0 or 1")
        with torch.cuda.device(dev):
            _check(self.lib.exl3_forward_pass(
                input_tiles.data_ptr(), temp_costs.data_ptr(), temp_edges.data_ptr(),
                pre_states.data_ptr(), n, K, cb, L, int(roll), int(cost_slot),
                int(bool(force_global_costs)), _stream(dev)), "quantize_tiles_forward_pass")

    # quantize_xpu.cpp:217-259
    def quantize_tiles_backward_pass(self, temp_costs, temp_edges, output_tiles, output_indices,
                                     end_states, num_tiles: int, K: int, mcg: bool, mul1: bool,
                                     roll: int, cost_slot: int, write_output: bool,
                                     sg_size: int = 32) -> None:
        torch = _torch()
        cb = _resolve_cb(mcg, mul1)
        dev = _check_device_tensor(temp_costs, "temp_costs", torch.float16, 3)
        if _check_device_tensor(output_tiles, "output_tiles", torch.float32, 2) != dev:
            raise RuntimeError("output_tiles must be on the same GPU device")
        if _check_device_tensor(output_indices, "output_indices", torch.int16, 2) != dev:
            raise RuntimeError("output_indices must be on the same GPU device")
        if _check_device_tensor(end_states, "end_states", torch.int32, 1) != dev:
            raise RuntimeError("end_states must be an int32 GPU tensor")
        # The tile length is the one (256 or 160) whose scratch row count the
        # temp_edges tensor has; the two counts differ at every K.
        _validate_common(K, cb, 256, sg_size)
        if temp_edges.dim() != 3:
            raise RuntimeError("temp_edges must be 3-D (B, rows, row_bytes)")
        matches = [n for n in (256, 160) if tile_rows(K, n) == temp_edges.size(1)]
        if not matches:
            raise RuntimeError(f"temp_edges has {temp_edges.size(1)} rows, which fits neither "
                               f"L=256 ({tile_rows(K, 256)}) nor L=160 ({tile_rows(K, 160)}) "
                               f"at K={K}")
        L = matches[0]
        _validate_common(K, cb, L, sg_size)
        batch_cap = self._scratch_checks(temp_costs, temp_edges, K, L, dev)
        if not 0 < num_tiles <= batch_cap:
            raise RuntimeError("num_tiles must be in 1..B")
        if end_states.size(0) < num_tiles:
            raise RuntimeError("end_states length must be >= num_tiles")
        if write_output and (output_tiles.size(0) < num_tiles or output_tiles.size(1) != L
                             or output_indices.size(0) < num_tiles
                             or output_indices.size(1) != L):
            raise RuntimeError("output tensors must have shape (>= num_tiles, L)")
        with torch.cuda.device(dev):
            _check(self.lib.exl3_backward_pass(
                temp_costs.data_ptr(), temp_edges.data_ptr(), output_tiles.data_ptr(),
                output_indices.data_ptr(), end_states.data_ptr(), int(num_tiles), K, cb, L,
                int(roll), int(cost_slot), int(bool(write_output)), _stream(dev)),
                "quantize_tiles_backward_pass")

    # quantize_xpu.cpp:261-300, quantize_kernels.sycl:756-841
    def quantize_tiles_usm_host(self, input_tiles, temp_costs, output_tiles_cpu,
                                output_indices_cpu, lut_cpu, K: int, mcg: bool, mul1: bool,
                                sg_size: int = 32) -> list:
        """The reference's host-visible-edges variant: states and codebook
        values land in CPU tensors, and [search_s, trace_s] is returned. On
        MI355X the search and the traceback both run on the GPU (split
        forward/backward passes over an internal device scratch of
        temp_costs' batch size); the results are copied to the CPU tensors.
        ``lut_cpu`` is validated as in the reference and otherwise unused:
        the GPU decodes states in registers."""
        torch = _torch()
        cb = _resolve_cb(mcg, mul1)
        dev = _check_device_tensor(input_tiles, "input_tiles", torch.float32, 2)
        if _check_device_tensor(temp_costs, "temp_costs", torch.float16, 3) != dev:
            raise RuntimeError("temp_costs must be on the same GPU device")
        if not (output_tiles_cpu.device.type == "cpu" and output_tiles_cpu.is_contiguous()
                and output_tiles_cpu.dtype == torch.float32):
            raise RuntimeError("output_tiles_cpu must be a contiguous float32 CPU tensor")
        if not (output_indices_cpu.device.type == "cpu" and output_indices_cpu.is_contiguous()
                and output_indices_cpu.dtype == torch.int16):
            raise RuntimeError("output_indices_cpu must be a contiguous int16 CPU tensor")
        if not (lut_cpu.device.type == "cpu" and lut_cpu.is_contiguous()
                and lut_cpu.dtype == torch.float32 and lut_cpu.numel() == 65536):
            raise RuntimeError("lut_cpu must be a 65536-element float32 CPU tensor")
        n, L = input_tiles.shape
        _validate_common(K, cb, L, sg_size)
        if tuple(output_tiles_cpu.shape) != (n, L) or tuple(output_indices_cpu.shape) != (n, L):
            raise RuntimeError("output tensors must have shape (num_tiles, L)")
        B = temp_costs.size(0)
        if B < 1 or temp_costs.size(1) != 2 or temp_costs.size(2) != (65536 >> K):
            raise RuntimeError("temp_costs must have shape (B, 2, 65536 >> K)")
        search_s = trace_s = 0.0
        with torch.cuda.device(dev):
            edges = torch.empty(edges_shape(B, K, L), dtype=torch.uint8, device=f"cuda:{dev}")
            out_w = torch.empty((n, L), dtype=torch.float32, device=f"cuda:{dev}")
            out_i = torch.empty((n, L), dtype=torch.int16, device=f"cuda:{dev}")
            ends = torch.empty(B, dtype=torch.int32, device=f"cuda:{dev}")
            free = torch.full((B,), -1, dtype=torch.int32, device=f"cuda:{dev}")
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(5)]
            for off in range(0, n, B):
                c = min(B, n - off)
                x = input_tiles[off:off + c]
                ev[0].record()
                self.quantize_tiles_forward_pass(x, temp_costs, edges, free, K, mcg, mul1,
                                                 L // 2, 0, sg_size)
                ev[1].record()
                self.quantize_tiles_backward_pass(temp_costs, edges, out_w[off:off + c],
                                                  out_i[off:off + c], ends, c, K, mcg, mul1,
                                                  L // 2, 0, False, sg_size)
                ev[2].record()
                self.quantize_tiles_forward_pass(x, temp_costs, edges, ends, K, mcg, mul1, 0, 1,
                                                 sg_size)
                ev[3].record()
                self.quantize_tiles_backward_pass(temp_costs, edges, out_w[off:off + c],
                                                  out_i[off:off + c], ends, c, K, mcg, mul1, 0, 1,
                                                  True, sg_size)
                ev[4].record()
                ev[4].synchronize()
                search_s += (ev[0].elapsed_time(ev[1]) + ev[2].elapsed_time(ev[3])) / 1e3
                trace_s += (ev[1].elapsed_time(ev[2]) + ev[3].elapsed_time(ev[4])) / 1e3
            output_tiles_cpu.copy_(out_w.cpu())
            output_indices_cpu.copy_(out_i.cpu())
        return [search_s, trace_s]

    # -------------------------------------------------- device-side helpers

    def prepare_tiles(self, raw, out, permute: bool, nan_count=None) -> None:
        """fp16-round (and optionally permute) ``raw`` into ``out``; a given
        ``nan_count`` (device int32, one element) gains one per NaN value."""
        torch = _torch()
        dev = _check_device_tensor(raw, "raw", torch.float32, 2)
        n, L = raw.shape
        _check_buffer(out, "out", torch.float32, (n, L), dev)
        counter = None
        if nan_count is not None:
            if (not isinstance(nan_count, torch.Tensor) or nan_count.dtype != torch.int32
                    or nan_count.device != raw.device or nan_count.numel() < 1):
                raise RuntimeError("nan_count must be an int32 tensor on the tiles' device")
            counter = nan_count.data_ptr()
        with torch.cuda.device(dev):
            _check(self.lib.exl3_prepare_tiles(raw.data_ptr(), out.data_ptr(), n, L,
                                               int(bool(permute)), counter, _stream(dev)),
                   "prepare_tiles")

    def finalize_tiles(self, x, raw, out_w, out_idx, packed, path_cost, distortion, recon_orig,
                       K: int, permuted: bool) -> None:
        torch = _torch()
        dev = _check_device_tensor(x, "x", torch.float32, 2)
        n, L = x.shape
        for t, name, dt, shape in ((out_w, "out_w", torch.float32, (n, L)),
                                   (out_idx, "out_idx", torch.int16, (n, L)),
                                   (path_cost, "path_cost", torch.float32, (n,)),
                                   (distortion, "distortion", torch.float32, (n,)),
                                   (recon_orig, "recon_orig", torch.int16, (n, L))):
            _check_buffer(t, name, dt, shape, dev)
        if packed is not None:
            _check_buffer(packed, "packed", torch.int16, (n, 16 * K), dev)
        if permuted:
            _check_buffer(raw, "raw", torch.float32, (n, L), dev)
        with torch.cuda.device(dev):
            _check(self.lib.exl3_finalize_tiles(
                x.data_ptr(), raw.data_ptr() if permuted else None, out_w.data_ptr(),
                out_idx.data_ptr(), packed.data_ptr() if packed is not None else None,
                path_cost.data_ptr(), distortion.data_ptr(), recon_orig.data_ptr(), n, K, L,
                int(bool(permuted)), _stream(dev)), "finalize_tiles")

    def pack_trellis(self, states, packed, K: int) -> None:
        torch = _torch()
        dev = _check_device_tensor(states, "states", torch.int16, 2)
        n = states.size(0)
        if states.size(1) != 256 or not 1 <= K <= 8:
            raise RuntimeError("pack_trellis expects (n, 256) states and K in 1..8")
        _check_buffer(packed, "packed", torch.int16, (n, 16 * K), dev)
        with torch.cuda.device(dev):
            _check(self.lib.exl3_pack_trellis(states.data_ptr(), packed.data_ptr(), n, K,
                                              _stream(dev)), "pack_trellis")

    def unpack_trellis(self, packed, states, K: int) -> None:
        """Packed (n, 16*K) int16 tiles back to (n, 256) int16 states."""
        torch = _torch()
        dev = _check_device_tensor(packed, "packed", torch.int16, 2)
        n = packed.size(0)
        if not 1 <= K <= 8 or packed.size(1) != 16 * K:
            raise RuntimeError("unpack_trellis expects (n, 16*K) words and K in 1..8")
        _check_buffer(states, "states", torch.int16, (n, 256), dev)
        with torch.cuda.device(dev):
            _check(self.lib.exl3_unpack_trellis(packed.data_ptr(), states.data_ptr(), n, K,
                                                _stream(dev)), "unpack_trellis")

    def probe_hfma(self, dh, cost, out, mode: int) -> None:
        """exl3_quant/xpu_probe.py ``probe_hfma`` (mode 0: fused, 1: two roundings)."""
        torch = _torch()
        dev = _check_device_tensor(dh, "dh", torch.float16, 1)
        _check_buffer(cost, "cost", torch.float16, tuple(dh.shape), dev)
        _check_buffer(out, "out", torch.float16, tuple(dh.shape), dev)
        with torch.cuda.device(dev):
            _check(self.lib.exl3_probe_hfma(dh.data_ptr(), cost.data_ptr(), out.data_ptr(),
                                            dh.numel(), int(mode), _stream(dev)), "probe_hfma")


# ------------------------------------------------- layer pipeline kernels

def _matrix(t, name: str) -> int:
    """A contiguous 2-D float32 GPU tensor; returns its device index."""
    return _check_device_tensor(t, name, _torch().float32, 2)


def hadamard128(x, out, side: int) -> None:
    """``out = H @ x`` per 128-row block (side 0) or ``x @ H`` per 128-column
    block (side 1), H the orthonormal Sylvester matrix of order 128
    (hadamard.py:73-96); ``out`` may be ``x``."""
    dev = _matrix(x, "x")
    _check_buffer(out, "out", x.dtype, tuple(x.shape), dev)
    rows, cols = x.shape
    torch = _torch()
    with torch.cuda.device(dev):
        _check(load_library().exl3_hadamard128(x.data_ptr(), out.data_ptr(), rows, cols,
                                               int(side), _stream(dev)), "hadamard128")


def hadamard128_scaled(x, out, side: int, divisor=None, slice_sumsq=None) -> None:
    """``out = (x / divisor[col]) @ H`` per 128-column block (side 1) or
    ``out = H @ (x / divisor[row])`` per 128-row block (side 0); with side 1
    ``slice_sumsq`` (rows x cols / 32 float32) receives the sums of squares
    of every 32-element slice of the output rows. ``out`` may be ``x``."""
    torch = _torch()
    dev = _matrix(x, "x")
    _check_buffer(out, "out", x.dtype, tuple(x.shape), dev)
    rows, cols = x.shape
    if divisor is not None:
        want = cols if side == 1 else rows
        if (not isinstance(divisor, torch.Tensor) or divisor.dtype != torch.float32
                or not divisor.is_contiguous() or divisor.device != x.device
                or divisor.numel() != want):
            raise RuntimeError(f"divisor must be a contiguous float32 tensor of {want} elements "
                               f"on {x.device}")
    if slice_sumsq is not None:
        if side != 1 or cols % 32:
            raise RuntimeError("slice sums of squares need side 1 and columns divisible by 32")
        _check_buffer(slice_sumsq, "slice_sumsq", torch.float32, (rows, cols // 32), dev)
    with torch.cuda.device(dev):
        _check(load_library().exl3_hadamard128_scaled(
            x.data_ptr(), out.data_ptr(), rows, cols, int(side),
            divisor.data_ptr() if divisor is not None else None,
            slice_sumsq.data_ptr() if slice_sumsq is not None else None, _stream(dev)),
            "hadamard128_scaled")


def _scale_vector(t, name: str, numel: int, like) -> None:
    torch = _torch()
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or not t.is_contiguous()
            or t.device != like.device or t.numel() != numel):
        raise RuntimeError(f"{name} must be a contiguous float32 tensor of {numel} elements on "
                           f"{like.device}")


def row_energy(x, sv, sums) -> None:
    """Sums of squares of the 128-element segments of the rows of ``(x / sv)
    H``, (rows, cols / 128) (exl3_row_energy)."""
    torch = _torch()
    dev = _matrix(x, "x")
    rows, cols = x.shape
    _scale_vector(sv, "sv", cols, x)
    _check_buffer(sums, "sums", torch.float32, (rows, cols // 128), dev)
    with torch.cuda.device(dev):
        _check(load_library().exl3_row_energy(x.data_ptr(), sv.data_ptr(), sums.data_ptr(), rows,
                                              cols, _stream(dev)), "row_energy")


def rotate(x, sv, su, out) -> None:
    """``out = H (((x / sv) H) / su)`` with blockwise order-128 transforms
    (exl3_rotate); ``out`` must not be ``x``."""
    torch = _torch()
    dev = _matrix(x, "x")
    _check_buffer(out, "out", x.dtype, tuple(x.shape), dev)
    rows, cols = x.shape
    _scale_vector(sv, "sv", cols, x)
    _scale_vector(su, "su", rows, x)
    with torch.cuda.device(dev):
        _check(load_library().exl3_rotate(x.data_ptr(), sv.data_ptr(), su.data_ptr(),
                                          out.data_ptr(), rows, cols, _stream(dev)), "rotate")


def unrotate(x, su, sv, out) -> None:
    """``out = (H x * su) H * sv`` with blockwise order-128 transforms
    (exl3_unrotate); ``out`` must not be ``x``."""
    dev = _matrix(x, "x")
    _check_buffer(out, "out", x.dtype, tuple(x.shape), dev)
    rows, cols = x.shape
    _scale_vector(su, "su", rows, x)
    _scale_vector(sv, "sv", cols, x)
    torch = _torch()
    with torch.cuda.device(dev):
        _check(load_library().exl3_unrotate(x.data_ptr(), su.data_ptr(), sv.data_ptr(),
                                            out.data_ptr(), rows, cols, _stream(dev)), "unrotate")


def decode_weight(words, su, sv, out, K: int, cb: int) -> None:
    """The (16 tk, 16 tn) weight of packed ``words`` ((tk * tn, 16 K) int16,
    4-byte aligned) into ``out`` (exl3_decode_weight)."""
    torch = _torch()
    dev = _check_device_tensor(words, "words", torch.int16, 2)
    _check_device_tensor(out, "out", torch.float32, 2)
    rows, cols = out.shape
    if words.shape[0] * 256 != rows * cols or words.shape[1] != 16 * K:
        raise RuntimeError(f"words {tuple(words.shape)} do not hold a {rows} x {cols} weight at "
                           f"K={K}")
    _check_buffer(out, "out", torch.float32, (rows, cols), dev)
    _scale_vector(su, "su", rows, out)
    _scale_vector(sv, "sv", cols, out)
    with torch.cuda.device(dev):
        _check(load_library().exl3_decode_weight(words.data_ptr(), su.data_ptr(), sv.data_ptr(),
                                                 out.data_ptr(), rows, cols, int(K), int(cb),
                                                 _stream(dev)), "decode_weight")


def block_rms_from_slices(slice_sumsq, out, n: int) -> None:
    """``out[o] = sqrt(sum_s slice_sumsq[o, s] / n)``, the slices added in
    order (the second pass of block_rms)."""
    torch = _torch()
    dev = _matrix(slice_sumsq, "slice_sumsq")
    outputs, slices = slice_sumsq.shape
    if (not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or not out.is_contiguous()
            or out.device != slice_sumsq.device or out.numel() != outputs):
        raise RuntimeError(f"out must be a contiguous float32 tensor of {outputs} elements")
    with torch.cuda.device(dev):
        _check(load_library().exl3_block_rms_from_slices(slice_sumsq.data_ptr(), out.data_ptr(),
                                                         outputs, int(n), slices, _stream(dev)),
               "block_rms_from_slices")


def input_scales(slice_sumsq, su, scales, su_out, n: int) -> None:
    """regularize's input-channel scales and su from the slice sums of
    squares of (rows, n) (exl3_input_scales)."""
    torch = _torch()
    dev = _matrix(slice_sumsq, "slice_sumsq")
    rows, slices = slice_sumsq.shape
    for t, name in ((su, "su"), (scales, "scales"), (su_out, "su_out")):
        _scale_vector(t, name, rows, slice_sumsq)
    with torch.cuda.device(dev):
        _check(load_library().exl3_input_scales(slice_sumsq.data_ptr(), su.data_ptr(),
                                                scales.data_ptr(), su_out.data_ptr(), rows,
                                                int(n), slices, _stream(dev)), "input_scales")


def output_scales(x, sv, decide: int, forced: bool, scales, divisor, sv_out, flags,
                  diag=None) -> None:
    """regularize's output-channel scales (exl3_output_scales). ``diag`` is a
    1-D float32 tensor on x's device, of any positive stride."""
    torch = _torch()
    dev = _matrix(x, "x")
    rows, cols = x.shape
    for t, name in ((sv, "sv"), (scales, "scales"), (divisor, "divisor"), (sv_out, "sv_out")):
        _scale_vector(t, name, cols, x)
    _check_buffer(flags, "flags", torch.float64, (3,), dev)
    if diag is not None and (diag.dtype != torch.float32 or diag.dim() != 1
                             or diag.device != x.device or diag.numel() < 1
                             or diag.stride(0) < 1):
        raise RuntimeError(f"diag must be a 1-D float32 tensor on {x.device}, not expanded")
    lib = load_library()
    with torch.cuda.device(dev):
        need = int(lib.exl3_block_rms_workspace(rows, cols, 0, 32))
        ws = torch.empty(max(need, 1), dtype=torch.float32, device=x.device)
        _check(lib.exl3_output_scales(
            x.data_ptr(), rows, cols, diag.data_ptr() if diag is not None else None,
            diag.stride(0) if diag is not None else 1,
            diag.numel() if diag is not None else 0, sv.data_ptr(), int(decide),
            int(bool(forced)), ws.data_ptr(), ws.numel(), scales.data_ptr(), divisor.data_ptr(),
            sv_out.data_ptr(), flags.data_ptr(), _stream(dev)), "output_scales")


def block_rms(x, out, dim: int, blocksize: int = 32) -> None:
    """regularize.py:41-56 into ``out`` (``x.shape[1 - dim]`` elements,
    any shape)."""
    dev = _matrix(x, "x")
    rows, cols = x.shape
    n_out = cols if dim == 0 else rows
    torch = _torch()
    if (not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or not out.is_contiguous()
            or out.device != x.device or out.numel() != n_out):
        raise RuntimeError(f"out must be a contiguous float32 tensor of {n_out} elements on "
                           f"{x.device}")
    lib = load_library()
    need = int(lib.exl3_block_rms_workspace(rows, cols, int(dim), int(blocksize)))
    if need < 0:
        raise RuntimeError(f"block_rms: invalid dim {dim} or blocksize {blocksize}")
    with torch.cuda.device(dev):
        ws = torch.empty(max(need, 1), dtype=torch.float32, device=x.device)
        _check(lib.exl3_block_rms(x.data_ptr(), out.data_ptr(), rows, cols, int(dim),
                                  int(blocksize), ws.data_ptr(), ws.numel(), _stream(dev)),
               "block_rms")


def gram_takes(x) -> bool:
    """Whether ``gram`` takes the 2-D tensor ``x`` (exl3_gram's shape, stride
    and alignment rules)."""
    torch = _torch()
    return (x.device.type == "cuda" and x.dim() == 2
            and x.dtype in (torch.bfloat16, torch.float16) and x.shape[0] >= 1
            and 8 <= x.shape[1] <= 1 << 20 and x.shape[1] % 8 == 0 and x.stride(1) == 1
            and x.shape[1] <= x.stride(0) <= 1 << 24 and x.stride(0) % 8 == 0
            and x.data_ptr() % 16 == 0)


def gram(x, scale: float, chunk_tokens: int = 8192):
    """``scale * x.T @ x`` in float32 for bf16 / fp16 activations, no float32
    sum over more than ``chunk_tokens`` tokens (exl3_gram_chunked)."""
    torch = _torch()
    if not gram_takes(x):
        raise RuntimeError(f"gram does not take {x.dtype} {tuple(x.shape)} with strides "
                           f"{x.stride()}")
    tokens, d = x.shape
    dev = x.device.index if x.device.index is not None else torch.cuda.current_device()
    lib = load_library()
    with torch.cuda.device(dev):
        need = int(lib.exl3_gram_workspace(tokens, d))
        h = torch.empty((d, d), dtype=torch.float32, device=x.device)
        ws = torch.empty(max(need, 1), dtype=torch.float32, device=x.device)
        _check(lib.exl3_gram_chunked(x.data_ptr(), int(x.dtype == torch.bfloat16), tokens,
                                     x.stride(0), d, float(scale), min(chunk_tokens, tokens),
                                     h.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev)),
               "gram")
    return h


def damp_diagonal(h, damping: float, floor: float):
    """Damps and floors the diagonal of the square matrix ``h`` in place
    (exl3_damp_diagonal); returns its mean before, as a device scalar."""
    torch = _torch()
    dev = _matrix(h, "h")
    d = h.shape[0]
    if h.shape[1] != d:
        raise RuntimeError(f"h must be square, got {tuple(h.shape)}")
    with torch.cuda.device(dev):
        mean = torch.empty((), dtype=torch.float32, device=h.device)
        _check(load_library().exl3_damp_diagonal(h.data_ptr(), d, d, float(damping), float(floor),
                                                 mean.data_ptr(), _stream(dev)), "damp_diagonal")
    return mean


def cholesky_block_order() -> int:
    return int(load_library().exl3_cholesky_block_order())


def cholesky_diag_block(a, j0: int, nb: int, info) -> None:
    """Factor the diagonal block ``a[j0:j0+nb, j0:j0+nb]`` of the square
    matrix ``a`` in place; a failed pivot k records ``j0 + k + 1`` in
    ``info`` (one int32 on the same device) unless it is already set."""
    torch = _torch()
    dev = _matrix(a, "a")
    n = a.shape[0]
    if a.shape[1] != n:
        raise RuntimeError(f"a must be square, got {tuple(a.shape)}")
    if not (0 <= j0 and 1 <= nb <= cholesky_block_order() and j0 + nb <= n):
        raise RuntimeError(f"block [{j0}, {j0 + nb}) does not fit a {n} x {n} matrix")
    if (not isinstance(info, torch.Tensor) or info.dtype != torch.int32
            or info.device != a.device or info.numel() < 1):
        raise RuntimeError("info must be an int32 tensor on a's device")
    with torch.cuda.device(dev):
        _check(load_library().exl3_cholesky_diag_block(a.data_ptr() + 4 * (j0 * n + j0), n, nb,
                                                       j0, info.data_ptr(), _stream(dev)),
               "cholesky_diag_block")


def cholesky(a, info):
    """Factor the square float32 matrix ``a`` in place (exl3_cholesky; its
    lower triangle is read, what lies above the diagonal is left as it is
    outside the diagonal blocks). Returns the inverses of the factor's 16 x
    16 diagonal tiles, (ceil(n / 16), 16, 16)."""
    torch = _torch()
    dev = _matrix(a, "a")
    n = a.shape[0]
    if a.shape[1] != n or n < 1:
        raise RuntimeError(f"a must be square, got {tuple(a.shape)}")
    if (not isinstance(info, torch.Tensor) or info.dtype != torch.int32
            or info.device != a.device or info.numel() < 1):
        raise RuntimeError("info must be an int32 tensor on a's device")
    lib = load_library()
    with torch.cuda.device(dev):
        inverses = torch.empty(int(lib.exl3_cholesky_inverse_elems(n)), dtype=torch.float32,
                               device=a.device)
        _check(lib.exl3_cholesky(a.data_ptr(), n, inverses.data_ptr(), info.data_ptr(),
                                 _stream(dev)), "cholesky")
    return inverses.view(-1, 16, 16)


def block_fold(l, inverses, out) -> None:
    """``out`` = the factor of a 16-wide block LDL from the Cholesky factor
    ``l`` and the inverses of its diagonal tiles (exl3_block_fold)."""
    torch = _torch()
    dev = _matrix(l, "l")
    n = l.shape[0]
    _check_buffer(l, "l", torch.float32, (n, n), dev)
    _check_buffer(out, "out", torch.float32, (n, n), dev)
    _check_buffer(inverses, "inverses", torch.float32, (n // 16, 16, 16), dev)
    with torch.cuda.device(dev):
        _check(load_library().exl3_block_fold(l.data_ptr(), inverses.data_ptr(), out.data_ptr(),
                                              n, _stream(dev)), "block_fold")


LDLQ_BLOCK_FIELDS = ("w", "comp", "wq", "err", "states", "n", "tile0", "reserved")


def check_ldlq_rows(rows, tiles: int) -> None:
    """Host check of one encoder call's ``exl3_ldlq_block`` rows before they
    are uploaded: every block's n is a positive multiple of 16, the first
    block starts at batch tile 0, each next one where the previous ends, and
    together they cover exactly ``tiles`` tiles. The kernels trust the table
    for their addresses, so a table that breaks this is refused here."""
    import numpy as np
    r = np.asarray(rows, dtype=np.int64).reshape(-1, len(LDLQ_BLOCK_FIELDS))
    check_ldlq_table(r, [(0, r.shape[0], tiles)])


def check_ldlq_table(rows, calls) -> None:
    """``check_ldlq_rows`` for a whole traversal at once: ``rows`` holds the
    ``exl3_ldlq_block`` rows of every call back to back and ``calls`` lists
    each call's (first row, row count, tiles), in order and covering every
    row."""
    import numpy as np
    r = np.asarray(rows, dtype=np.int64).reshape(-1, len(LDLQ_BLOCK_FIELDS))
    c = np.asarray(calls, dtype=np.int64).reshape(-1, 3)
    first, count, tiles = c[:, 0], c[:, 1], c[:, 2]
    if (count < 1).any():
        raise ValueError("an LDLQ call needs at least one block")
    if (not np.array_equal(first, np.concatenate([[0], np.cumsum(count)[:-1]]))
            or int(count.sum()) != r.shape[0]):
        raise ValueError("the calls must list the table's rows back to back")
    n = r[:, LDLQ_BLOCK_FIELDS.index("n")]
    tile0 = r[:, LDLQ_BLOCK_FIELDS.index("tile0")]
    if (n <= 0).any() or (n % 16).any():
        raise ValueError(f"block widths must be positive multiples of 16, got {n.tolist()}")
    # Each row's start within its call: the widths of the call's earlier rows.
    widths = n // 16
    ends = np.cumsum(widths)
    base = np.concatenate([[0], ends])[first]
    starts = ends - widths - np.repeat(base, count)
    call_bad = (np.add.reduceat((tile0 != starts).astype(np.int64), first) > 0) | (
        ends[first + count - 1] - base != tiles)
    if call_bad.any():
        i = int(np.flatnonzero(call_bad)[0])
        rows_i = slice(int(first[i]), int(first[i] + count[i]))
        raise ValueError(f"blocks must tile the batch back to back from 0 to {int(tiles[i])}: "
                         f"tile0 {tile0[rows_i].tolist()}, widths {widths[rows_i].tolist()}")
    for field in ("w", "comp", "wq", "err", "states"):
        if (r[:, LDLQ_BLOCK_FIELDS.index(field)] == 0).any():
            raise ValueError(f"NULL {field} address in an LDLQ block row")


def _ldlq_table(table, tiles_like, name: str) -> tuple:
    torch = _torch()
    dev = _check_device_tensor(tiles_like, name, tiles_like.dtype, 2)
    if tiles_like.size(1) != 256:
        raise RuntimeError(f"{name} must be (tiles, 256), got {tuple(tiles_like.shape)}")
    if (not isinstance(table, torch.Tensor) or table.dtype != torch.int64 or table.dim() != 2
            or table.size(1) != len(LDLQ_BLOCK_FIELDS) or not table.is_contiguous()
            or table.device != tiles_like.device or table.size(0) < 1):
        raise RuntimeError("the block table must be a contiguous (blocks, 8) int64 tensor on "
                           f"{tiles_like.device}")
    return dev, table.size(0), tiles_like.size(0)


def ldlq_gather(table, x) -> None:
    """Tile formation of one LDLQ encoder call (exl3_ldlq_gather): ``table``
    is the call's (blocks, 8) int64 ``exl3_ldlq_block`` rows on the device,
    whose addresses the caller has checked; ``x`` receives (tiles, 256)
    float32 tiles in tensor-core order."""
    torch = _torch()
    dev, nb, tiles = _ldlq_table(table, x, "x")
    if x.dtype != torch.float32:
        raise RuntimeError("x must be float32")
    with torch.cuda.device(dev):
        _check(load_library().exl3_ldlq_gather(table.data_ptr(), nb, tiles, x.data_ptr(),
                                               _stream(dev)), "ldlq_gather")


def ldlq_scatter(table, recon, idx) -> None:
    """Write-back of one LDLQ encoder call (exl3_ldlq_scatter) from the
    encoder's (tiles, 256) float32 reconstruction and int16 states."""
    torch = _torch()
    dev, nb, tiles = _ldlq_table(table, recon, "recon")
    if recon.dtype != torch.float32:
        raise RuntimeError("recon must be float32")
    _check_buffer(idx, "idx", torch.int16, tuple(recon.shape), dev)
    with torch.cuda.device(dev):
        _check(load_library().exl3_ldlq_scatter(table.data_ptr(), nb, tiles, recon.data_ptr(),
                                                idx.data_ptr(), _stream(dev)), "ldlq_scatter")


_EXT: Optional[QuantizeExtension] = None


def extension() -> QuantizeExtension:
    global _EXT
    if _EXT is None:
        _EXT = QuantizeExtension()
    return _EXT


# ------------------------------------------------- the 4-bit attention cache

_TYPES = None


def _types() -> dict:
    """C codes of the element types that rows may have."""
    global _TYPES
    if _TYPES is None:
        torch = _torch()
        _TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return _TYPES


def _rows(t, name: str, like=None, heads=None, dim=None) -> tuple:
    """The shape and strides of a (tokens, heads, head_dim) GPU tensor whose
    last axis is contiguous."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 3:
        raise RuntimeError(f"{name} must be a 3-D GPU (cuda) tensor (tokens, heads, head_dim)")
    if t.dtype not in _types():
        raise RuntimeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    shape, strides = t.shape, t.stride()
    if strides[2] != 1 and shape[2] > 1:
        raise RuntimeError(f"the last axis of {name} must be contiguous")
    if like is not None and (t.dtype != like.dtype or shape[0] != like.shape[0]
                             or t.device != like.device):
        raise RuntimeError(f"{name} must have the device, type and tokens of the other rows")
    if (heads is not None and shape[1] != heads) or (dim is not None and shape[2] != dim):
        raise RuntimeError(f"{name} must have {heads if heads is not None else 'any'} heads of "
                           f"{dim} values, got {tuple(shape)}")
    return shape, strides


def _vector(t, name: str, dtypes: tuple, numel, device) -> None:
    torch = _torch()
    if (not isinstance(t, torch.Tensor) or t.dtype not in dtypes
            or (t.dim() != 1 if numel is None else t.shape != (numel,)) or not t.is_contiguous()
            or t.device != device):
        raise RuntimeError(f"{name} must be a contiguous vector of "
                           f"{'any length' if numel is None else numel}, "
                           f"{' or '.join(map(str, dtypes))}, on {device}")


def _positions(positions, axes, tokens: int, pairs: int, device) -> tuple:
    """The arguments of the tokens' positions: a vector, or one of each axis with
    the axis of every pair."""
    torch = _torch()
    if axes is None:
        _vector(positions, "positions", (torch.int32, torch.int64), tokens, device)
        return positions.data_ptr(), positions.dtype == torch.int64, None, 1
    _vector(axes, "axes", (torch.int32,), pairs, device)
    if (not isinstance(positions, torch.Tensor) or positions.dim() != 2
            or positions.dtype not in (torch.int32, torch.int64) or positions.shape[0] < 1
            or positions.shape[1] != tokens or not positions.is_contiguous()
            or positions.device != device):
        raise RuntimeError(f"positions must be a contiguous (axes, {tokens}) tensor, int32 or int64, "
                           f"on {device}")
    return (positions.data_ptr(), positions.dtype == torch.int64, axes.data_ptr(),
            positions.shape[0])


def _pages(pages) -> tuple:
    """(pages, page size, kv heads, head dim) of a cache."""
    torch = _torch()
    if (not isinstance(pages, torch.Tensor) or pages.device.type != "cuda" or pages.dim() != 4
            or pages.dtype != torch.uint8 or not pages.is_contiguous()):
        raise RuntimeError("pages must be a contiguous 4-D uint8 GPU (cuda) tensor "
                           "(pages, kv_heads, page_size / 32, 36 * head_dim)")
    n, heads, tiles, size = pages.shape
    if size not in (2304, 4608, 9216) or tiles not in (1, 2, 4, 8) or heads < 1:
        raise RuntimeError(f"pages of shape {tuple(pages.shape)} are no cache: head_dim 64, 128 "
                           "or 256 (36 * head_dim bytes a tile), page_size 32, 64, 128 or 256")
    return n, 32 * tiles, heads, size // 36


def _run(device, what: str, call, *args) -> None:
    """One C call on the current stream of ``device``. A small call is bound by
    the host: the stream is read without the Stream object that
    torch.cuda.current_stream makes (1.9 us), and the device switched only where
    it is not the current one."""
    torch = _torch()
    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _check(status, what)


def _written(*tensors) -> None:
    """Tell torch that a kernel wrote into the caller's tensors: a backward pass
    that saved one of them then refuses, as after torch's own in-place operations."""
    _torch().autograd.graph.increment_version(tensors)


class _Span:
    """Rows at an address, as numpy's overlap solver takes them (it reads none)."""

    def __init__(self, address: int, shape, strides):
        self.__array_interface__ = {"version": 3, "data": (address, False),
                                    "shape": tuple(shape[:2]),
                                    "strides": tuple(strides[:2]), "typestr": f"|V{shape[2]}"}


def shares_memory(a: tuple, b: tuple) -> bool:
    """Whether two (address, (tokens, heads, bytes of a row), (token stride, head
    stride) in bytes) have a byte in common. Rows of one projection lie between
    each other without sharing any, so the ranges alone do not say; what the
    solver gives up on counts as shared."""
    (at_a, shape_a, (token, head_a)), (at_b, shape_b, (token_b, head_b)) = a, b
    if not (all(shape_a) and all(shape_b)):
        return False
    # What a token's rows reach over: apart where ranges are, or (slices of one
    # tensor) where the first token's are within a stride of tokens.
    reach_a = (shape_a[1] - 1) * head_a + shape_a[2]
    reach_b = (shape_b[1] - 1) * head_b + shape_b[2]
    if (at_a + (shape_a[0] - 1) * token + reach_a <= at_b
            or at_b + (shape_b[0] - 1) * token_b + reach_b <= at_a):
        return False
    if token and token == token_b and reach_a <= (at_b - at_a) % token <= token - reach_b:
        return False
    import numpy as np
    try:
        return np.shares_memory(np.asarray(_Span(*a)), np.asarray(_Span(*b)), max_work=10 ** 6)
    except np.exceptions.TooHardError:
        return True


def rows_are_apart(shape, strides) -> bool:
    """Whether no two rows of (tokens, heads, row size) share memory, from the
    strides of tokens and heads: the shorter one passes a row, the longer all of
    the other axis."""
    reach = shape[2]
    if not all(shape):
        return True
    for stride, n in sorted(zip(strides, shape)):
        if n > 1:
            if stride < reach:
                return False
            reach += (n - 1) * stride
    return True


def _check_outputs(size: int, *rows) -> None:
    """Of (input, output), each an (address, shape, strides in elements of
    ``size`` bytes): the kernel's blocks run in any order, each reading and
    writing whole rows, so an output may be its input, and else shares no memory
    with any tensor of the call."""
    def span(address, shape, strides):
        return (address, (shape[0], shape[1], shape[2] * size),
                (strides[0] * size, strides[1] * size))

    written, read = [], []
    for given, out in rows:
        out = span(*out)
        if not rows_are_apart(*out[1:]):
            raise RuntimeError(f"rows of out[{len(written)}] share memory with each other")
        written.append(out)
        given = span(*given)
        (tokens, heads, _), (token, head), (to_token, to_head) = given[1], given[2], out[2]
        if (given[0] != out[0] or (token != to_token and tokens > 1)
                or (head != to_head and heads > 1)):
            read.append(given)
    for i, out in enumerate(written):
        if any(shares_memory(out, given) for given in read):
            raise RuntimeError(f"out[{i}] shares memory with q or k: outputs are the inputs "
                               "themselves, or apart from both")
    if len(written) == 2 and shares_memory(*written):
        raise RuntimeError("out[0] and out[1] share memory")


def rotary(q, k, positions, frequencies, layout: int, magnitude: float, inverse: bool,
           out=None, axes=None) -> tuple:
    """q and k turned by their positions (exl3_rotary_axes); k may be None."""
    torch = _torch()
    (tokens, heads, dim), sq = _rows(q, "q")
    device = q.device
    _vector(frequencies, "frequencies", (torch.float64,), None, device)
    pairs = frequencies.numel()
    if not 1 <= pairs <= dim // 2:
        raise RuntimeError(f"frequencies must hold 1 to {dim // 2} pairs, got {pairs}")
    places = _positions(positions, axes, tokens, pairs, device)
    dense = torch.contiguous_format
    q_out, k_out = out or (torch.empty_like(q, memory_format=dense), None)
    so = _rows(q_out, "out[0]", q, heads, dim)[1] if out else (heads * dim, dim)
    k_args = (None, 0, 0, None, 0, 0, 0)
    if k is not None:
        (_, k_heads, _), sk = _rows(k, "k", q, None, dim)
        if not out:
            k_out = torch.empty_like(k, memory_format=dense)
        sp = _rows(k_out, "out[1]", q, k_heads, dim)[1] if out else (k_heads * dim, dim)
        k_args = (k.data_ptr(), sk[0], sk[1], k_out.data_ptr(), sp[0], sp[1], k_heads)
    else:
        k_out = None
    if out:
        at, shape = k_args[0], (tokens, heads, dim)
        more = () if k is None else (((at, k.shape, sk), (k_args[3], k.shape, sp)),)
        _check_outputs(q.element_size(), ((q.data_ptr(), shape, sq), (q_out.data_ptr(), shape, so)),
                       *more)
    _run(device, "apply_rotary", load_library().exl3_rotary_axes, q.data_ptr(), sq[0], sq[1],
         q_out.data_ptr(), so[0], so[1], heads, *k_args, tokens, dim, _types()[q.dtype],
         *places, frequencies.data_ptr(), pairs, layout, magnitude, inverse)
    if out:
        _written(*(t for t in (q_out, k_out) if t is not None))
    return q_out, k_out


def plan_step(cached, new, tables, free_pages, taken, page_size: int, max_tokens: int) -> tuple:
    """Slots, positions, starts, lengths, taken and status (exl3_plan_step)."""
    torch = _torch()
    dev = tables.device if isinstance(tables, torch.Tensor) else None
    if (dev is None or dev.type != "cuda" or tables.dim() != 2 or tables.dtype != torch.int32
            or not tables.is_contiguous()):
        raise RuntimeError("tables must be a contiguous 2-D int32 GPU (cuda) tensor")
    requests, width = tables.shape
    _vector(cached, "cached", (torch.int32,), requests, dev)
    _vector(new, "new", (torch.int32,), requests, dev)
    _vector(free_pages, "free_pages", (torch.int32,), None, dev)
    _vector(taken, "taken", (torch.int32,), 1, dev)
    if not 0 <= max_tokens < 2 ** 31:
        raise RuntimeError(f"max_tokens must be in 0..2^31 - 1, got {max_tokens}")
    slots = tables.new_empty(max_tokens, dtype=torch.int64)
    positions, starts, lengths, taken_out, status = tables.new_empty(
        max_tokens + 2 * requests + 3).split_with_sizes([max_tokens, requests + 1, requests, 1, 1])
    _run(dev, "plan_step", load_library().exl3_plan_step, cached.data_ptr(), new.data_ptr(),
         requests, tables.data_ptr(), width, free_pages.data_ptr(), free_pages.numel(),
         taken.data_ptr(), page_size, max_tokens, slots.data_ptr(), positions.data_ptr(),
         starts.data_ptr(), lengths.data_ptr(), taken_out.data_ptr(), status.data_ptr())
    _written(tables)
    return slots, positions, starts, lengths, taken_out, status


def cache_append(pages, k, v, slots, q, positions, frequencies, layout: int, magnitude: float,
                 axes=None):
    """k and v into the cache, k (and q) turned first (exl3_cache_append_axes);
    returns the turned q."""
    torch = _torch()
    n, page_size, heads, dim = _pages(pages)
    device = pages.device
    # The kernel reads 16 bytes at a time; rows that start elsewhere are copied.
    k, v = _wide(k), _wide(v)
    (tokens, _, _), sk = _rows(k, "k", None, heads, dim)
    sv = _rows(v, "v", k, heads, dim)[1]
    if k.device != device:
        raise RuntimeError("k and v must be on the cache's device")
    _vector(slots, "slots", (torch.int64,), tokens, device)
    pairs, freq, at = 0, None, (None, 0, None, 1)
    q_out, q_args = None, (None, 0, 0, None, 0)
    if frequencies is not None:
        _vector(frequencies, "frequencies", (torch.float64,), None, device)
        pairs = frequencies.numel()
        if pairs % 8 or not 8 <= pairs <= dim // 2:
            raise RuntimeError(f"frequencies must hold a multiple of 8 pairs up to {dim // 2}, got "
                               f"{pairs}: turn with apply_rotary first")
        at, freq = _positions(positions, axes, tokens, pairs, device), frequencies.data_ptr()
        if q is not None:
            q = _wide(q)
            (_, q_heads, _), sq = _rows(q, "q", k, None, dim)
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            q_args = (q.data_ptr(), sq[0], sq[1], q_out.data_ptr(), q_heads)
    elif q is not None or positions is not None or axes is not None:
        raise RuntimeError("q, positions and axes are only taken with frequencies")
    _run(device, "append_tokens", load_library().exl3_cache_append_axes, *q_args,
         k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], tokens,
         _types()[k.dtype], slots.data_ptr(), *at, freq, pairs, layout, magnitude,
         pages.data_ptr(), n, page_size, heads, dim)
    _written(pages)
    return q_out


def _wide(t):
    """A 3-D tensor, or a copy of it, with every row 16-byte aligned; anything
    else as it is, for the checks to refuse."""
    torch = _torch()
    if isinstance(t, torch.Tensor) and t.dim() == 3:
        size, strides = t.element_size(), t.stride()
        if t.data_ptr() % 16 or strides[0] * size % 16 or strides[1] * size % 16:
            return t.clone(memory_format=torch.contiguous_format)
    return t


def cache_read(pages, slots, dtype) -> tuple:
    """Keys and values at ``slots`` (exl3_cache_read)."""
    torch = _torch()
    n, page_size, heads, dim = _pages(pages)
    _vector(slots, "slots", (torch.int64,), None, pages.device)
    if dtype not in _types():
        raise RuntimeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    tokens = slots.numel()
    k = slots.new_empty((tokens, heads, dim), dtype=dtype)
    v = torch.empty_like(k)
    _run(pages.device, "read_tokens", load_library().exl3_cache_read, pages.data_ptr(), n,
         page_size, heads, dim, slots.data_ptr(), tokens, _types()[dtype], k.data_ptr(),
         v.data_ptr())
    return k, v


def cache_attention(q, pages, tables, starts, lengths, scale, window, max_new, trees=None):
    """Attention over the cache (exl3_cache_attention_trees)."""
    torch = _torch()
    n, page_size, heads, dim = _pages(pages)
    dev = pages.device
    q = _wide(q)
    (tokens, q_heads, _), sq = _rows(q, "q", None, None, dim)
    if q.dtype == torch.float32 or q.device != dev:
        raise RuntimeError("q must be float16 or bfloat16, on the cache's device")
    if q_heads < 1 or q_heads % heads:
        raise RuntimeError(f"q must have a multiple of the cache's {heads} heads, got {q_heads}")
    if (not isinstance(tables, torch.Tensor) or tables.device != dev or tables.dim() != 2
            or tables.dtype != torch.int32 or not tables.is_contiguous()):
        raise RuntimeError(f"tables must be a contiguous 2-D int32 tensor on {dev}")
    requests, width = tables.shape
    _vector(starts, "starts", (torch.int32,), requests + 1, dev)
    _vector(lengths, "lengths", (torch.int32,), requests, dev)
    if window is not None and window < 1:
        raise RuntimeError(f"window must be positive, got {window}")
    if max_new is not None and max_new < 0:
        raise RuntimeError(f"max_new must not be negative, got {max_new}")
    masks, words = None, 0
    if trees is not None:
        if (not isinstance(trees, torch.Tensor) or trees.device != dev or trees.dim() != 2
                or trees.dtype != torch.int64 or not trees.is_contiguous()
                or trees.shape[0] < tokens or not 1 <= trees.shape[1] <= MAX_TREE_WORDS):
            raise RuntimeError(f"trees must be a contiguous int64 tensor of at least {tokens} rows of "
                               f"1 to {MAX_TREE_WORDS} words on {dev}")
        masks, words = trees.data_ptr(), trees.shape[1]
    lib = load_library()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    # Python's integers end nowhere, the C arguments at 64 bits.
    most = tokens if max_new is None else min(int(max_new), tokens)
    window = 2 ** 31 - 1 if window is None else min(int(window), 2 ** 31 - 1)
    asked = lib.exl3_cache_attention_workspace if masks is None else lib.exl3_cache_attention_trees_workspace
    size = asked(tokens, q_heads, heads, dim, requests, most)
    workspace = pages.new_empty(max(size, 0))
    _run(dev, "cache_attention", lib.exl3_cache_attention_trees, q.data_ptr(), sq[0], sq[1],
         out.data_ptr(), tokens, q_heads, _types()[q.dtype], pages.data_ptr(), n, page_size, heads,
         dim, tables.data_ptr(), width, starts.data_ptr(), lengths.data_ptr(), requests,
         masks, words, dim ** -0.5 if scale is None else float(scale), window, most, workspace.data_ptr(), size)
    return out


# ------------------------------------------------- drafted tokens

MAX_TREE_WORDS = 16


def _ranges(starts, lengths=None) -> int:
    """Requests of the starts of their tokens (and of their lengths)."""
    torch = _torch()
    if not isinstance(starts, torch.Tensor) or not starts.is_cuda or starts.dim() != 1:
        raise RuntimeError("starts must be a 1-D GPU (cuda) tensor")
    if starts.dtype != torch.int32 or not starts.is_contiguous():
        raise RuntimeError(f"starts must be a contiguous int32 vector, got {starts.dtype}")
    requests = starts.numel() - 1
    if lengths is not None:
        _vector(lengths, "lengths", (torch.int32,), requests, starts.device)
    return requests


def plan_tree(parents, starts, lengths, words: int) -> tuple:
    """Masks and positions of drafted tokens (exl3_plan_tree)."""
    torch = _torch()
    requests, device = _ranges(starts, lengths), starts.device
    _vector(parents, "parents", (torch.int32,), None, device)
    tokens = parents.numel()
    masks = parents.new_empty((tokens, words), dtype=torch.int64)
    positions = torch.empty_like(parents)
    _run(device, "plan_tree", load_library().exl3_plan_tree, parents.data_ptr(), starts.data_ptr(),
         lengths.data_ptr(), requests, tokens, words, masks.data_ptr(), positions.data_ptr())
    return masks, positions


def accept_drafts(tokens, choices, parents, starts, lengths, certain, words: int) -> tuple:
    """Places, lengths and next tokens (exl3_accept_trees)."""
    torch = _torch()
    requests, device = _ranges(starts, lengths), starts.device
    _vector(parents, "parents", (torch.int32,), None, device)
    count = parents.numel()
    _vector(tokens, "tokens", (torch.int32, torch.int64), count, device)
    _vector(choices, "choices", (tokens.dtype,), count, device)
    if certain is not None:
        _vector(certain, "certain", (torch.int32,), requests, device)
    places, kept = torch.empty_like(parents), torch.empty_like(lengths)
    following = lengths.new_empty(requests, dtype=tokens.dtype)
    _run(device, "accept_drafts", load_library().exl3_accept_trees, tokens.data_ptr(),
         choices.data_ptr(), tokens.dtype == torch.int64, parents.data_ptr(), starts.data_ptr(),
         lengths.data_ptr(), None if certain is None else certain.data_ptr(), requests, count, words,
         places.data_ptr(), kept.data_ptr(), following.data_ptr())
    return places, kept, following


def cache_keep(pages, slots, starts, places) -> None:
    """Entries of kept tokens moved together (exl3_cache_keep)."""
    torch = _torch()
    n, page_size, heads, dim = _pages(pages)
    device = pages.device
    requests = _ranges(starts)
    if starts.device != device:
        raise RuntimeError("starts must be on the cache's device")
    _vector(slots, "slots", (torch.int64,), None, device)
    _vector(places, "places", (torch.int32,), slots.numel(), device)
    _run(device, "keep_tokens", load_library().exl3_cache_keep, pages.data_ptr(), n, page_size, heads,
         dim, slots.data_ptr(), starts.data_ptr(), places.data_ptr(), requests, slots.numel())
    _written(pages)


def release_pages(before, after, tables, free_pages, taken, page_size: int):
    """The new ``taken`` (exl3_release_pages)."""
    torch = _torch()
    dev = tables.device if isinstance(tables, torch.Tensor) else None
    if (dev is None or dev.type != "cuda" or tables.dim() != 2 or tables.dtype != torch.int32
            or not tables.is_contiguous()):
        raise RuntimeError("tables must be a contiguous 2-D int32 GPU (cuda) tensor")
    requests, width = tables.shape
    _vector(before, "before", (torch.int32,), requests, dev)
    _vector(after, "after", (torch.int32,), requests, dev)
    _vector(free_pages, "free_pages", (torch.int32,), None, dev)
    _vector(taken, "taken", (torch.int32,), 1, dev)
    out = torch.empty_like(taken)
    _run(dev, "release_pages", load_library().exl3_release_pages, before.data_ptr(), after.data_ptr(),
         requests, tables.data_ptr(), width, page_size, free_pages.data_ptr(), free_pages.numel(),
         taken.data_ptr(), out.data_ptr())
    _written(tables, free_pages)
    return out


# ------------------------------------------------- products with stored weights

def linear(x, trellis, su, sv, K: int, cb: int):
    """x (..., in) times a stored weight (exl3_linear)."""
    torch = _torch()
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() < 1:
        raise RuntimeError("x must be a GPU (cuda) tensor (..., in)")
    if x.dtype != torch.float16 and x.dtype != torch.bfloat16:
        raise RuntimeError(f"x must be float16 or bfloat16, got {x.dtype}")
    device = x.device
    if not 1 <= K <= 8:
        raise ValueError(f"K must be in 1..8, got {K}")
    if cb not in (0, 1, 2):
        raise ValueError(f"Unknown codebook {cb}")
    if (not isinstance(trellis, torch.Tensor) or trellis.dtype != torch.int16 or trellis.dim() != 3
            or not trellis.is_contiguous() or trellis.device != device):
        raise RuntimeError(f"trellis must be a contiguous 3-D int16 tensor on {device}")
    tk, tn, words = trellis.shape
    if words != 16 * K:
        raise ValueError(f"Trellis last dimension {words} does not match 16 * K = {16 * K}")
    k, n = 16 * tk, 16 * tn
    if k % 128 or n % 128 or not k or not n:
        raise ValueError(f"both dimensions must be divisible by 128, got {(k, n)}")
    shape = x.shape
    if shape[-1] != k:
        raise ValueError(f"x must have {k} input channels, got {tuple(shape)}")
    scales = (torch.float16, torch.float32)
    # As columns and rows too, as quantisation returns them.
    if isinstance(su, torch.Tensor) and su.dim() == 2:
        su = su.flatten()
    if isinstance(sv, torch.Tensor) and sv.dim() == 2:
        sv = sv.flatten()
    _vector(su, "suh", scales, k, device)
    _vector(sv, "svh", scales, n, device)
    # The kernel reads 16 bytes at a time; rows that start elsewhere are copied.
    rows = x if x.dim() == 2 else x.reshape(-1, k)
    stride, at, words_at, su_at, sv_at = rows.stride(), rows.data_ptr(), trellis.data_ptr(), su.data_ptr(), sv.data_ptr()
    if stride[1] != 1 or stride[0] % 8 or at % 16:
        rows = rows.clone(memory_format=torch.contiguous_format)
        stride, at = rows.stride(), rows.data_ptr()
    if (words_at | su_at | sv_at) % 16:
        trellis, su, sv = (t.clone() if t.data_ptr() % 16 else t for t in (trellis, su, sv))
        words_at, su_at, sv_at = trellis.data_ptr(), su.data_ptr(), sv.data_ptr()
    count = rows.shape[0]
    lib = load_library()
    code = _types()[x.dtype]
    size = lib.exl3_linear_workspace(count, k, n, code)
    if size < 0:
        raise RuntimeError(f"quantized_linear: {count} rows of {k} by {n} are too many")
    out = x.new_empty((*shape[:-1], n))
    workspace = trellis.new_empty(size // 2)
    _run(device, "quantized_linear", lib.exl3_linear, at, stride[0], count, code, words_at, su_at, sv_at,
         (su.dtype == torch.float16) + 2 * (sv.dtype == torch.float16), k, n, K, cb,
         out.data_ptr(), workspace.data_ptr(), size)
    return out
