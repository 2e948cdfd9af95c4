"""What the operators around the projections refuse, without a GPU: every check of arguments comes before the first use of the
device, so a bad call is an SDH_ERR_INVALID here and a good one ends at the missing device."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from llama_cpp_amd import scan, sublayer
from llama_cpp_amd import seeddelta as sd

BAD, NO_DEVICE = r"\(-1\)", r"\(-2\)"
P = 4096                                     # a pointer that is never read: 16-byte aligned

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that passes the checks would run")


def norm(n=64, T=2, **k):
    a = dict(ldx=64, weight_ptr=P, eps=1e-6, y_ptr=4 * P, ldy=64)
    a.update(k)
    x_ptr, ldx = a.pop("x_ptr", P), a.pop("ldx")
    sublayer.rms_norm_device(x_ptr, ldx, n, T, **a)


Q8 = sublayer.Q8View(P, 64, 2 * P, 2)


@pytest.mark.parametrize("k", [
    dict(x_ptr=0), dict(y_ptr=0), dict(n=0), dict(n=-1), dict(T=-1), dict(n=65), dict(ldy=63), dict(res_ptr=P, ldr=63), dict(sum_ptr=2 * P, lds=63),
    dict(eps=-1.0), dict(eps=float("nan")), dict(x_ptr=P + 2), dict(y_ptr=P + 1), dict(weight_ptr=P + 2),
    dict(sum_ptr=P, lds=128), dict(y_ptr=P, ldy=128), dict(sum_ptr=4 * P, lds=64), dict(res_ptr=2 * P, ldr=64, sum_ptr=2 * P, lds=65),
    dict(n=63, q8=Q8), dict(q8=sublayer.Q8View(0, 64, P, 2)), dict(q8=sublayer.Q8View(P, 64, 0, 2)), dict(q8=sublayer.Q8View(P, 63, P, 2)),
    dict(q8=sublayer.Q8View(P, 64, P, 1)), dict(q8=sublayer.Q8View(P + 1, 64, P, 2)), dict(q8=sublayer.Q8View(P, 66, P, 2)),
    dict(T=1 << 31), dict(n=1 << 31, ldx=1 << 32, ldy=1 << 32),
])
def test_norm_refuses(k):
    with pytest.raises(sd.SeedDeltaError, match=BAD):
        norm(**k)


@pytest.mark.parametrize("k", [dict(), dict(T=0, x_ptr=0, y_ptr=0), dict(q8=Q8), dict(q8=Q8, y_ptr=0), dict(sum_ptr=P, lds=64), dict(y_ptr=P), dict(weight_ptr=0), dict(n=1),
                               dict(res_ptr=2 * P, ldr=70, sum_ptr=2 * P, lds=70)])
def test_norm_takes(k):
    with pytest.raises(sd.SeedDeltaError, match=NO_DEVICE):
        norm(**k)


@pytest.mark.parametrize("args", [(0, 64, 64, 2, Q8), (P, 63, 64, 2, Q8), (P, 64, 64, 2, None), (P, 64, 48, 2, Q8), (P, 64, 0, 2, Q8), (P, 64, 64, -1, Q8), (P + 2, 64, 64, 1, Q8)])
def test_quantize_refuses(args):
    with pytest.raises(sd.SeedDeltaError, match=BAD):
        sublayer.q8_quantize_device(*args)


def test_dense_refuses_null():
    lib = sd.load_library()
    assert lib.sdh_dense_forward_q8(None, C.byref(Q8), 1, P, 64, None) == -1
    assert b"null" in lib.sdh_last_error()


def ab(r=4, n_in=32, n_out=48, ta=np.float16, tb=np.float16):
    return np.zeros((r, n_in), ta), np.zeros((n_out, r), tb), 1.0


@pytest.mark.parametrize("adapters", [
    [], [ab(), ab(n_in=33)], [ab(), ab(n_out=47)], [(np.zeros((4, 32), np.float16), np.zeros((48, 5), np.float16), 1.0)],
    [ab(r=513)], [ab(ta=np.int16)], [ab(tb=np.int32)], [(np.zeros((4, 32, 1), np.float16), np.zeros((48, 4), np.float16), 1.0)], [ab(r=1)] * 4097,
    [(np.zeros((0, 32), np.float16), np.zeros((48, 0), np.float16), 1.0)],
])
def test_adapter_sets_refused(adapters, monkeypatch):
    monkeypatch.setattr(sd, "_inited_device", 0)
    with pytest.raises(sd.SeedDeltaError, match=BAD if adapters and adapters[0][0].ndim == 2 else "LoraSet"):
        sublayer.LoraSet(adapters)


def test_adapter_sets_taken_up_to_the_device(monkeypatch):
    monkeypatch.setattr(sd, "_inited_device", 0)
    for adapters in ([ab()], [ab(), ab(r=1), ab(r=512, ta=np.float32)]):
        with pytest.raises(sd.SeedDeltaError, match=NO_DEVICE):
            sublayer.LoraSet(adapters)


def test_adapter_sets_have_a_largest_size():
    lib, d = sd.load_library(), (sd.SdhLoraDesc * 1)()
    h = C.c_void_p()
    for n_in, n_out in ((0, 48), (32, 0), (-1, 48), ((1 << 24) + 1, 48), (32, (1 << 24) + 1)):
        assert lib.sdh_lora_create(n_in, n_out, d, 1, C.byref(h)) == -1 and b"dims" in lib.sdh_last_error()


def test_lora_entry_points_without_a_set():
    lib = sd.load_library()
    assert lib.sdh_lora_bytes(None) == -1 and lib.sdh_lora_workspace_bytes(None, 4) == -1
    lib.sdh_lora_destroy(None)
    assert lib.sdh_lora_create(32, 48, None, 1, C.byref(C.c_void_p())) == -1
    assert lib.sdh_lora_apply(None, None, P, 32, 1, None, 0, P, 48, P, 1 << 20, None) == -1


def test_struct_layouts_match_the_header():
    assert C.sizeof(sd.SdhQ8) == 32 and C.sizeof(sd.SdhLoraDesc) == 2 * C.sizeof(sd.SdhTensor) + 8


@pytest.mark.parametrize("W", [np.zeros((3, 100), np.uint8), np.zeros((3, 33), np.uint8), np.zeros(68, np.uint8), np.zeros((2, 3, 34), np.uint8), np.zeros(64, np.float32)])
def test_dense_weights_of_ragged_rows_are_refused(W, monkeypatch):
    monkeypatch.setattr(sd, "_inited_device", 0)
    with pytest.raises(sd.SeedDeltaError, match="DenseWeight"):
        scan.DenseWeight(W)
    with pytest.raises(sd.SeedDeltaError, match="DenseWeight|raw Q8_0 rows"):
        sd.SeedDeltaContext().add_dense("up", W)


def test_dense_weights_of_whole_blocks_end_at_the_device():
    with pytest.raises(sd.SeedDeltaError, match=NO_DEVICE):
        scan.DenseWeight(np.zeros((3, 68), np.uint8))


def test_device_code_is_compiled_without_packed_fp32():
    """Every line that compiles HIP code, the measurement helpers' included, switches the packed instructions off."""
    root, lines = Path(__file__).resolve().parent.parent, []
    for f in [root / "llama.cpp_amd/csrc/Makefile", *root.glob("tools/*.sh"), *root.glob("tools/*.hip"), *root.glob("tools/gpu/*")]:
        text = f.read_text()
        lines += [(f.name, line) for line in text.splitlines() if re.search(r"hipcc\b.*\.hip\b|^CFLAGS", line) and " -shared " not in line]
    assert len(lines) >= 9
    assert [x for x in lines if "-Xclang -target-feature -Xclang -packed-fp32-ops" not in x[1]] == []
