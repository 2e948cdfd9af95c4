"""What the library does when the HIP runtime says no, on the CPU: hip_stub.c takes the runtime's place in a process of its own (kernels do
not run; a test says which call fails, which device is current, whether a capture is under way)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
START = """
import ctypes as C, sys
import numpy as np
stub = C.CDLL({stub!r}, C.RTLD_GLOBAL)
sys.path.insert(0, {root!r})
import llama_cpp_amd
from llama_cpp_amd import scan, sublayer, seeddelta as sd
from llama_cpp_amd.dense import make_dense
from llama_cpp_amd.payload import make_payload
def refused(fn, code):
    try:
        fn()
    except sd.SeedDeltaError as e:
        assert f"({{code}})" in str(e), e
        return str(e)
    raise AssertionError("not refused")
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.check_call(["gcc", "-std=c11", "-shared", "-fPIC", "-O1", "-I/opt/rocm/include", "-o", out, os.path.join(HERE, "hip_stub.c")])

    def run(code):
        p = subprocess.run([sys.executable, "-c", START.format(stub=out, root=os.path.dirname(HERE)) + code + "\nprint('done')"],
                           capture_output=True, text=True, timeout=240)
        assert p.returncode == 0 and p.stdout.endswith("done\n"), p.stdout + p.stderr
    return run


def test_dense_upload_that_fails_is_an_error_and_leaves_nothing(stub):
    """Whichever copy fails, and whether or not the runtime keeps the error of a call that others follow."""
    stub("""
sd.init(0)
before = stub.stub_live()
for W, copies in ((make_dense(1024, 3000), 6), (make_dense(96, 50), 2), (make_dense(64, 33, "f16"), 1), (make_dense(64, 33, "f32"), 1)):
    for keep in (0, 1):
        for n in range(copies):
            stub.stub_fail_copy(n, keep)
            assert "failed" in refused(lambda: scan.DenseWeight(W), -3)
            assert stub.stub_live() == before, (n, keep)
    stub.stub_fail_copy(-1, 1)
    w = scan.DenseWeight(W)
    w.close()
    assert stub.stub_live() == before
""")


def test_dense_upload_is_not_blamed_for_an_earlier_error(stub):
    stub("""
sd.init(0)
stub.stub_stale_error()
scan.DenseWeight(make_dense(96, 50)).close()
""")


def test_dense_weight_of_another_device_is_refused(stub):
    """The kernels run on the device that the library is bound to; a handle that was made while another one was current is not theirs to read."""
    stub("""
sd.init(0)
x8 = sublayer.Q8View(4096, 96, 8192, 3)
here = scan.DenseWeight(make_dense(96, 50))
stub.stub_set_device(1)
there = scan.DenseWeight(make_dense(96, 50))
assert "current device" in refused(lambda: sublayer.dense_forward_q8_device(here, x8, 4, 16384, 50), -1)
stub.stub_set_device(0)
n = stub.stub_launches()
assert "made on device 1" in refused(lambda: sublayer.dense_forward_q8_device(there, x8, 4, 16384, 50), -1)
assert stub.stub_launches() == n
sublayer.dense_forward_q8_device(here, x8, 4, 16384, 50)
assert stub.stub_launches() == n + 1
""")


def test_worker_threads_of_a_scan_run_on_the_bound_device(stub):
    """The current device is a thread's own and 0 in a new one: a rank bound to device 1 uploads and evaluates there from its pool too."""
    stub("""
sd.init(1)
ev = scan.Evaluator(lambda layer, kind: make_dense(96, 50), scan.ScanParams())
assert set(ev._workers(4).map(lambda _: stub.stub_device(), range(32))) == {1}
W = ev._workers(4).submit(lambda: scan.DenseWeight(make_dense(96, 50))).result()
sublayer.dense_forward_q8_device(W, sublayer.Q8View(4096, 96, 8192, 3), 4, 16384, 50)
stub.stub_set_device(0)
sd.init(1)                                    # once more in a thread: binds the thread
assert stub.stub_device() == 1
""")


def test_an_error_is_reported_once(stub):
    """The call that meets an error of the runtime returns it; the next one, which looks at its launch, does not find it again."""
    stub("""
sd.init(0)
norm = lambda: sublayer.rms_norm_device(4096, 64, 64, 2, y_ptr=8192, ldy=64)
for make in (lambda: scan.DenseWeight(make_dense(96, 50)), lambda: scan.DenseWeight(make_dense(64, 33, "f16")),
             lambda: sublayer.LoraSet([(np.zeros((4, 32), np.float16), np.zeros((48, 4), np.float16), 1.0)])):
    stub.stub_fail_copy(0, 1)
    refused(make, -3)
    norm()
    stub.stub_fail_copy(-1, 1)
    stub.stub_capture(1)                                # an allocation is refused
    refused(make, -3)
    stub.stub_capture(0)
    norm()
""")


def test_workspace_that_a_graph_holds_outlives_a_larger_one(stub):
    """A call with more tokens than before takes a larger workspace. One whose address a graph has recorded stays until the handle goes."""
    stub("""
sd.init(0)
def grown(recorded):
    before = stub.stub_live()
    w = sd.SeedDeltaWeight(make_payload(1024, 2048, scheme="coo", K=16, base=True, seed=1))
    call = lambda T: w.forward_device(4096, 1024, T, 8192, 2048, sd.FWD_NO_MFMA)
    call(16)
    if recorded:
        stub.stub_capture(1); call(16); stub.stub_capture(0)
    a = stub.stub_live()
    call(64)
    b = stub.stub_live()
    stub.stub_capture(1)                            # within the new size: nothing is allocated or freed
    call(64)
    refused(lambda: call(200), -3)                  # a larger one is (this mode of capture does not allow it)
    stub.stub_capture(0)
    call(200)
    w.close()
    assert stub.stub_live() == before
    return b - a
assert grown(False) == 0 and grown(True) == 1
""")


def test_ffn_workspace_that_a_graph_holds_outlives_a_larger_one(stub):
    stub("""
sd.init(0)
mk = lambda i, o, s: sd.SeedDeltaWeight(make_payload(i, o, scheme="coo", K=16, base=True, seed=s))
g, u, d = mk(1024, 2048, 1), mk(1024, 2048, 2), mk(2048, 1024, 3)
call = lambda T: sd.ffn_forward_device(g, u, d, sd.ACT_SILU, 4096, 1024, T, 8192, 1024, sd.FWD_NO_MFMA)
call(16)
a = stub.stub_live()
call(24)
assert stub.stub_live() == a
stub.stub_capture(1); call(24); stub.stub_capture(0)
call(64)
assert stub.stub_live() == a + 4                   # the three handles' and the block's own
""")


def test_folded_layout_is_not_built_under_capture(stub):
    stub("""
sd.init(0)
w = sd.SeedDeltaWeight(make_payload(1024, 2048, scheme="coo", K=16, base=True, seed=1))
call = lambda T: w.forward_device(4096, 1024, T, 8192, 2048, sd.FWD_MFMA_FOLD)
w.forward_device(4096, 1024, 2048, 8192, 2048, sd.FWD_NO_MFMA)      # a workspace that is large enough
live = stub.stub_live()
stub.stub_capture(1)
assert "eagerly" in refused(lambda: call(16), -4)
stub.stub_capture(0)
assert stub.stub_live() == live
""")


def test_no_memset_node_is_recorded(stub):
    """The ring of non-finite counters is cleared by a kernel: a call of any number may be the one that is recorded."""
    stub("""
sd.init(0)
w = sd.SeedDeltaWeight(make_payload(256, 512, scheme="coo", K=16, base=False, seed=1))
stub.stub_capture(1)
n = stub.stub_memsets()
for _ in range(600):
    w.forward_device(4096, 256, 1, 8192, 512)
assert stub.stub_memsets() == n and stub.stub_launches() >= 600
""")


def test_no_tokens_are_no_work_for_any_key(stub):
    """An empty batch has null pointers (an empty tensor's); a payload, a dense weight and adapters take it alike."""
    stub("""
sd.init(0)
ctx = sd.SeedDeltaContext()
assert ctx.try_add("up", make_payload(256, 512, scheme="coo", K=16, base=True, seed=1))
ctx.add_dense("gate", make_dense(256, 512))
for k in ("up", "gate"):
    ctx.add_adapters(k, [(np.zeros((4, 256), np.float16), np.zeros((512, 4), np.float16), 1.0)])
n = stub.stub_launches()
for k in ("up", "gate"):
    for ids in (0, 4096):
        assert ctx.mul_mat_device(k, 0, 256, 0, 0, 512, x8=sublayer.Q8View(0, 256, 0, 8), ids_ptr=ids) is True
assert ctx.mul_mat_device("down", 0, 256, 0, 0, 512) is False
assert stub.stub_launches() == n
""")


def test_mul_mat_device_launches_nothing_on_another_device(stub):
    stub("""
sd.init(0)
ctx = sd.SeedDeltaContext()
assert ctx.try_add("up", make_payload(256, 512, scheme="coo", K=16, base=True, seed=1))
ctx.add_dense("gate", make_dense(256, 512))
call = lambda k: ctx.mul_mat_device(k, 4096, 256, 16, 8192, 512, x8=sublayer.Q8View(4096, 256, 8192, 8))
n = stub.stub_launches()
stub.stub_set_device(1)
for k in ("up", "gate"):
    assert "current device is 1" in refused(lambda: call(k), -1)
assert stub.stub_launches() == n
stub.stub_set_device(0)
for k in ("up", "gate"):
    assert call(k)
assert stub.stub_launches() > n
""")


def test_adapters_of_another_device_are_refused(stub):
    """A set that was made before the library was bound to another device is in the first one's memory."""
    stub("""
sd.init(0)
s = sublayer.LoraSet([(np.zeros((4, 32), np.float16), np.zeros((48, 4), np.float16), 1.0)])
call = lambda: s.apply_device(0, 4096, 32, 8, 8192, 48, ws_ptr=16384, ws_bytes=1 << 20)
call()
sd.init(1)
n = stub.stub_launches()
assert "made on device 0" in refused(call, -1)
assert stub.stub_launches() == n
sd.init(0)
call()
assert stub.stub_launches() > n
""")
