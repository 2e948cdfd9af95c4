"""What a layer runs around its SeedDelta projections, on device buffers (include/seeddelta_hip.h, "around the projections"):

  * ``rms_norm_device`` — residual addition, root-mean-square norm and weight in one pass, output in F32 (what SeedDelta tensors
    read) and / or in 8 bits with scales (what dense Q8_0 tensors read); ``q8_quantize_device`` — the 8-bit conversion alone;
  * ``dense_forward_q8_device`` — a dense Q8_0 weight (``scan.DenseWeight``) times 8-bit activations: the projections of a layer
    that have no payload;
  * ``LoraSet`` — low-rank adapters of many requests beside one projection, SeedDelta or dense, the adapter chosen per token
    (``build_lora_mm``, src/llama-graph.cpp:672-746).

Pointers are raw device pointers, strides are in elements, ``stream`` is a hipStream_t (0: the legacy default stream), as in
``seeddelta``. Calls are asynchronous, allocate nothing and can be recorded into a HIP graph.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import seeddelta as sd


def Q8View(q_ptr: int, ldq: int, d_ptr: int, ldd: int) -> sd.SdhQ8:
    """8-bit activations in device memory: quants int8 (T, n) with row stride ldq, scales float32 (T, n / 32) with row stride ldd."""
    return sd.SdhQ8(q_ptr or None, ldq, d_ptr or None, ldd)


def rms_norm_device(x_ptr: int, ldx: int, n: int, T: int, weight_ptr: int = 0, eps: float = 1e-6, res_ptr: int = 0, ldr: int = 0,
                    sum_ptr: int = 0, lds: int = 0, y_ptr: int = 0, ldy: int = 0, q8=None, stream: int = 0):
    """s = x + res; z = s * weight / sqrt(mean(s^2) + eps). Writes s to `sum_ptr`, z to `y_ptr` (F32) and to `q8` (a Q8View);
    pointers that are 0 and q8 = None are left out."""
    rc = sd.load_library().sdh_rms_norm(x_ptr or None, ldx, res_ptr or None, ldr, weight_ptr or None, eps, n, T, sum_ptr or None, lds,
                                        y_ptr or None, ldy, None if q8 is None else C.byref(q8), stream or None)
    if rc:
        sd._check(rc, "sdh_rms_norm")


def q8_quantize_device(x_ptr: int, ldx: int, n: int, T: int, q8, stream: int = 0):
    rc = sd.load_library().sdh_q8_quantize(x_ptr or None, ldx, n, T, None if q8 is None else C.byref(q8), stream or None)
    if rc:
        sd._check(rc, "sdh_q8_quantize")


def dense_forward_q8_device(weight, x8, T: int, y_ptr: int, ldy: int, stream: int = 0):
    """y (T, n_out) = x (T, n_in) W^T for a Q8_0 `scan.DenseWeight` and a Q8View x8."""
    rc = sd.load_library().sdh_dense_forward_q8(weight._h, None if x8 is None else C.byref(x8), T, y_ptr or None, ldy, stream or None)
    if rc:
        sd._check(rc, "sdh_dense_forward_q8")


class LoraSet:
    """The adapters of one projection: a list of (A (r, n_in), B (n_out, r), scale), numpy float16 / float32, ranks may differ.
    scale = alpha / r times the user's scale, as llama_adapter_lora_weight::get_scale computes it."""

    def __init__(self, adapters):
        lib = sd.load_library()
        if sd._inited_device is None:
            sd.init(0)
        adapters = list(adapters)
        if not adapters or any(a.ndim != 2 or b.ndim != 2 for a, b, _ in adapters):
            raise sd.SeedDeltaError("LoraSet: a list of (A (r, n_in), B (n_out, r), scale) with one adapter at least")
        self.n_in, self.n_out = adapters[0][0].shape[1], adapters[0][1].shape[0]
        descs = (sd.SdhLoraDesc * len(adapters))()
        for d, (a, b, scale) in zip(descs, adapters):
            d.a, d.b, d.scale = sd.tensor_of(a), sd.tensor_of(b), float(scale)
        h = C.c_void_p()
        sd._check(lib.sdh_lora_create(self.n_in, self.n_out, descs, len(adapters), C.byref(h)), "sdh_lora_create")
        self._h = h
        self.n_adapters = len(adapters)
        self.stored_bytes = int(lib.sdh_lora_bytes(h))

    def workspace_bytes(self, T: int) -> int:
        n = int(sd.load_library().sdh_lora_workspace_bytes(self._h, T))
        if n < 0:
            sd._check(n, "sdh_lora_workspace_bytes")
        return n

    def apply_device(self, ids_ptr: int, x_ptr: int, ldx: int, T: int, y_ptr: int, ldy: int, base_ptr: int = 0, ldb: int = 0,
                     ws_ptr: int = 0, ws_bytes: int = 0, stream: int = 0):
        """y = base + scale_a B_a (A_a x) with a = ids[t] (int32 on the device; outside the set: y = base). base_ptr = y_ptr adds in
        place, base_ptr = 0 writes the adapters' part alone, ids_ptr = 0 gives every token adapter 0."""
        rc = sd.load_library().sdh_lora_apply(self._h, ids_ptr or None, x_ptr or None, ldx, T, base_ptr or None, ldb, y_ptr or None, ldy,
                                              ws_ptr or None, ws_bytes, stream or None)
        if rc:
            sd._check(rc, "sdh_lora_apply")

    def close(self):
        if getattr(self, "_h", None):
            sd.load_library().sdh_lora_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
