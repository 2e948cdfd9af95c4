"""GPU tests of the operators around the projections: sdh_rms_norm, sdh_q8_quantize, sdh_dense_forward_q8, sdh_lora_*, against
plain implementations in 64 bits on the CPU.

Tolerances (u = 2^-24, half a step of F32):
  * norm: s is one F32 addition, compared bit for bit. z is formed in double and rounded once: u |z| (plus 1e-12 |z| for the
    double arithmetic, and half the smallest subnormal). Scales: the same. A quant is the nearest integer of z / d; it may differ
    by one where z / d lies within 1e-9 of a border.
  * dense: the integer sums are exact. Per block one rounding of the product of the two scales and one of the fused
    multiply-add; the sums along a lane, over lanes and over waves round once per addition, at most nblk + 8 of them:
    (nblk + 10) u sum_b |term_b|.
  * adapters: u_r is a sum of n_in products (each rounded at most once with its addition), y a sum of r products and the base:
    (n_in + r + 20) u |scale| sum_r |B| sum_k |A x| + (r + 4) u |base|.
"""
import numpy as np
import pytest
import torch

from conftest import bits
from llama_cpp_amd import scan, sublayer
from llama_cpp_amd.dense import dequantize_q8_0, make_dense
from llama_cpp_amd.payload import make_payload
import oracle_py as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def padded(a, pad=0, shift=0, fill=float("nan")):
    """`a` (T, n) inside a larger device buffer: row stride n + pad, first element `shift` elements behind an aligned address,
    everything else `fill`. -> (buffer, pointer, stride)"""
    T, n = a.shape
    buf = torch.full((T * (n + pad) + shift + 64,), fill, dtype=torch.from_numpy(a[:0]).dtype, device="cuda")
    buf[shift:shift + T * (n + pad)].view(T, n + pad)[:, :n] = dev(a)
    return buf, buf.data_ptr() + shift * buf.element_size(), n + pad


class Out:
    """A (T, n) output inside a larger buffer of `fill`; get() returns it and checks that nothing else was written."""

    def __init__(self, T, n, pad=0, shift=0, dtype=torch.float32, fill=-77):
        self.T, self.n, self.pad, self.shift, self.fill = T, n, pad, shift, fill
        self.buf = torch.full((T * (n + pad) + shift + 64,), fill, dtype=dtype, device="cuda")
        self.ptr, self.ld = self.buf.data_ptr() + shift * self.buf.element_size(), n + pad

    def get(self):
        torch.cuda.synchronize()
        h = self.buf.cpu().numpy()
        body = h[self.shift:self.shift + self.T * self.ld].reshape(self.T, self.ld)
        assert np.all(h[:self.shift] == self.fill) and np.all(h[self.shift + self.T * self.ld:] == self.fill), "written outside the rows"
        assert np.all(body[:, self.n:] == self.fill), "written between the rows"
        return body[:, :self.n].copy()


# ---- norm -----------------------------------------------------------------------------------------------------------
def norm_ref(x, res, w):
    """-> (s F32, z in 64 bits)"""
    with np.errstate(all="ignore"):
        s = x if res is None else (x + res).astype(np.float32)
        s64 = s.astype(np.float64)
        z = s64 / np.sqrt((s64 * s64).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
        return s, z if w is None else z * w.astype(np.float64)


def check_q8(q, d, z):
    """quants (T, n) int8 and scales (T, n / 32) against z in 64 bits"""
    b = z.reshape(z.shape[0], -1, 32)
    with np.errstate(all="ignore"):
        amax = np.abs(b).max(2)
        want = amax / 127.0
    fine = np.isfinite(amax)
    assert np.all(~np.isfinite(d[~fine]))
    assert np.all(np.abs(d[fine] - want[fine]) <= (U + 1e-12) * want[fine] + 2.0 ** -150)
    q = q.reshape(b.shape)
    live = fine & (want.astype(np.float32) > 0)
    assert np.all(q[~live] == 0)
    r = b[live] * (127.0 / amax[live])[:, None]
    near = np.abs(np.abs(r - np.floor(r)) - 0.5) < 1e-9
    assert np.all((q[live] == np.rint(r)) | (near & (np.abs(q[live] - r) < 0.5 + 1e-8)))
    assert q.max(initial=0) <= 127 and q.min(initial=0) >= -127


def run_norm(T, n, res, w, f32, q8, seed=0, pad=0, shift=0, x=None, with_sum=True):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, n)).astype(np.float32) if x is None else x
    r = rng.standard_normal((T, n)).astype(np.float32) if res else None
    wt = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32) if w else None
    keep = [padded(x, pad, shift), padded(r, pad, shift) if res else (None, 0, 0), padded(wt[None], 0, shift) if w else (None, 0, 0)]
    s_out = Out(T, n, pad, shift) if res and with_sum else None
    y_out = Out(T, n, pad, shift) if f32 else None
    q_out, d_out = (Out(T, n, 4 * bool(pad), 4 * bool(shift), torch.int8), Out(T, n // 32, pad, shift)) if q8 else (None, None)
    sublayer.rms_norm_device(keep[0][1], keep[0][2], n, T, weight_ptr=keep[2][1], eps=EPS, res_ptr=keep[1][1], ldr=keep[1][2],
                             sum_ptr=s_out.ptr if s_out else 0, lds=s_out.ld if s_out else 0, y_ptr=y_out.ptr if f32 else 0, ldy=y_out.ld if f32 else 0,
                             q8=sublayer.Q8View(q_out.ptr, q_out.ld, d_out.ptr, d_out.ld) if q8 else None)
    s, z = norm_ref(x, r, wt)
    if s_out:
        assert np.array_equal(bits(s_out.get()), bits(s))
    got = {}
    if f32:
        got["y"] = y = y_out.get()
        ok = np.isfinite(z)
        assert np.all(np.abs(y[ok] - z[ok]) <= (U + 1e-12) * np.abs(z[ok]) + 2.0 ** -150)
        assert np.array_equal(np.isnan(y), np.isnan(z))
    if q8:
        got["q"], got["d"] = q_out.get(), d_out.get()
        check_q8(got["q"], got["d"], z)
    return got


@pytest.mark.parametrize("n", [1, 2, 3, 5, 31, 63, 100, 257, 1153, 4095, 4097, 8190, 16385, 40001])
@pytest.mark.parametrize("T", [1, 3])
def test_norm_odd_lengths(hip, n, T):
    run_norm(T, n, res=True, w=True, f32=True, q8=False, seed=n)


@pytest.mark.parametrize("n", [32, 64, 96, 256, 1152, 4096, 4128, 8192, 8224, 16384, 16416, 40000])
@pytest.mark.parametrize("res, w, pad, shift", [(True, True, 0, 0), (False, True, 4, 0), (True, False, 3, 1), (True, True, 0, 3), (False, False, 0, 0)])
def test_norm_all_outputs(hip, n, res, w, pad, shift):
    run_norm(5, n, res, w, True, True, seed=n, pad=pad, shift=shift)


@pytest.mark.parametrize("n", [1152, 4096, 20000])
def test_norm_outputs_do_not_depend_on_each_other(hip, n):
    both = run_norm(3, n, True, True, True, True, seed=4)
    a, b = run_norm(3, n, True, True, True, False, seed=4, with_sum=False), run_norm(3, n, True, True, False, True, seed=4, with_sum=False)
    assert np.array_equal(bits(both["y"]), bits(a["y"])) and np.array_equal(both["q"], b["q"]) and np.array_equal(bits(both["d"]), bits(b["d"]))


def test_norm_sum_alone_and_many_rows(hip):
    rng = np.random.default_rng(1)
    x, r = rng.standard_normal((2, 70001, 36)).astype(np.float32)
    s = Out(70001, 36)
    xd, rd = dev(x), dev(r)
    sublayer.rms_norm_device(xd.data_ptr(), 36, 36, 70001, res_ptr=rd.data_ptr(), ldr=36, sum_ptr=s.ptr, lds=s.ld)
    assert np.array_equal(bits(s.get()), bits(x + r))
    run_norm(70001, 32, False, True, True, True, seed=2)


@pytest.mark.parametrize("n", [64, 4096, 20000])
@pytest.mark.parametrize("into", ["sum=x", "sum=res", "y=x", "y=res", "sum=res,y=x"])
def test_norm_in_place(hip, n, into):
    rng = np.random.default_rng(n)
    x, r = rng.standard_normal((2, 4, n)).astype(np.float32)
    xd, rd = dev(x), dev(r)
    s, z = norm_ref(x, r, None)
    sum_t = {"sum=x": xd, "sum=res": rd}.get(into.split(",")[0])
    y_t = xd if "y=x" in into else rd if "y=res" in into else torch.empty_like(xd)
    sublayer.rms_norm_device(xd.data_ptr(), n, n, 4, eps=EPS, res_ptr=rd.data_ptr(), ldr=n, sum_ptr=0 if sum_t is None else sum_t.data_ptr(), lds=n, y_ptr=y_t.data_ptr(), ldy=n)
    torch.cuda.synchronize()
    if sum_t is not None:
        assert np.array_equal(bits(sum_t.cpu().numpy()), bits(s))
    assert np.all(np.abs(y_t.cpu().numpy() - z) <= (U + 1e-12) * np.abs(z))


def test_norm_extreme_values(hip):
    n = 256
    rng = np.random.default_rng(3)
    x = rng.standard_normal((9, n)).astype(np.float32)
    x[0] = 0.0
    x[1] *= np.float32(1e-38)          # eps decides
    x[2] *= np.float32(1e30)           # the squares leave F32
    x[3, 5] = np.inf
    x[4, 7] = np.nan
    x[5, :32] = 0.0                    # one block of zeros
    x[6] = 0.0
    x[6, 40] = np.float32(1e-45)       # the smallest subnormal alone
    x[7, 3] = np.float32(3e38)
    run_norm(9, n, False, True, True, True, x=x)
    run_norm(9, n, False, False, True, True, x=x)


@pytest.mark.parametrize("T, n, pad, shift", [(1, 32, 0, 0), (7, 96, 0, 0), (3, 6912, 5, 1), (2, 14336, 0, 0), (2, 20000, 4, 0)])
def test_quantize(hip, T, n, pad, shift):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((T, n)) * 10.0 ** rng.integers(-30, 30, (T, 1))).astype(np.float32)
    x[0, :32] = np.arange(32) - 16.5                     # d = 16.5 / 127
    if T > 2:
        x[1, 3], x[2, 40] = np.nan, -np.inf
        x[1, 64:96] = 0
    xs, q, d = padded(x, pad, shift), Out(T, n, 4 * bool(pad), 4 * bool(shift), torch.int8), Out(T, n // 32, pad, shift)
    sublayer.q8_quantize_device(xs[1], xs[2], n, T, sublayer.Q8View(q.ptr, q.ld, d.ptr, d.ld))
    check_q8(q.get(), d.get(), x.astype(np.float64))


def test_quantize_ties_go_to_the_even_step(hip):
    x = np.zeros((1, 32), np.float32)
    x[0, 0] = 127.0                                       # d = 1
    x[0, 1:9] = [0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5]
    q, d = Out(1, 32, dtype=torch.int8), Out(1, 1)
    xd = dev(x)
    sublayer.q8_quantize_device(xd.data_ptr(), 32, 32, 1, sublayer.Q8View(q.ptr, 32, d.ptr, 1))
    assert d.get()[0, 0] == 1.0
    assert q.get()[0, :9].tolist() == [127, 0, 2, 2, 0, -2, -2, 126, -126]


def test_norm_scale_past_the_range(hip):
    """A block of z whose scale leaves F32 is not finite: quants of zero, as where a value itself is not finite."""
    n = 20000
    x, w = np.zeros((2, n), np.float32), np.full(n, 3.4e38, np.float32)
    x[:, 40] = 1.0                                        # z = 3.4e38 * sqrt(20000) = 4.8e40, z / 127 = 3.8e38
    x[1, 41] = 1.0                                        # z = 3.4e40, z / 127 = 2.7e38: still in range
    q, d, xd, wd = Out(2, n, dtype=torch.int8), Out(2, n // 32), dev(x), dev(w)
    sublayer.rms_norm_device(xd.data_ptr(), n, n, 2, weight_ptr=wd.data_ptr(), eps=0.0, q8=sublayer.Q8View(q.ptr, q.ld, d.ptr, d.ld))
    q, d = q.get(), d.get()
    assert np.isinf(d[0, 1]) and not q[0].any() and not d[0, 2:].any()
    assert np.isfinite(d[1]).all() and q[1, 40] == q[1, 41] == 127 and np.count_nonzero(q[1]) == 2


@pytest.mark.parametrize("n", [2016, 20000])
def test_quantize_exact_ties_whatever_the_step(hip, n):
    """A block of maximum 127 k has the step k exactly, and (j + 1/2) k lies exactly between two steps, however 127 / (127 k) rounds:
    the even one for every k and j. Their neighbours in F32 on either side go to the step that is nearer."""
    rng = np.random.default_rng(n)
    T = 40
    k = rng.integers(1, 2000, (T, n // 32, 1)).astype(np.float32)
    k[0, :4, 0] = 49, 98, 103, 107                       # 73.5 / 49 = 1.5, where 73.5 * (127 / 6223) is below it
    k *= np.float32(2.0) ** rng.integers(-20, 20, k.shape).astype(np.float32)
    j = rng.integers(-127, 127, (T, n // 32, 32)).astype(np.float32)
    x = (j + np.float32(0.5)) * k                        # exact: 8 + 11 bits
    side = rng.integers(-1, 2, x.shape).astype(np.float32)
    x = np.where(side == 0, x, np.nextafter(x, np.copysign(np.float32(np.inf), side)))
    x[0, :4, 1] = 1.5 * k[0, :4, 0]
    x[:, :, :1] = 127 * k
    q, d = Out(T, n, dtype=torch.int8), Out(T, n // 32)
    xd = dev(x.reshape(T, n))
    sublayer.q8_quantize_device(xd.data_ptr(), n, n, T, sublayer.Q8View(q.ptr, q.ld, d.ptr, d.ld))
    assert np.array_equal(d.get(), k[:, :, 0])
    # x / k in 64 bits is exact at a tie and on the right side of it elsewhere (a neighbour is 2^-24 of it away)
    assert np.array_equal(q.get(), np.rint(x.astype(np.float64) / k).astype(np.int8).reshape(T, n))


# ---- dense ----------------------------------------------------------------------------------------------------------
def dense_case(n_in, n_out, T, seed=0, extreme=False):
    rng = np.random.default_rng(seed)
    W = make_dense(n_in, n_out, "q8_0", seed, structure=0.0)
    q = rng.integers(-127, 128, (T, n_in)).astype(np.int8)
    d = (np.abs(rng.standard_normal((T, n_in // 32))) * 0.02 * (10.0 ** rng.integers(-4, 5, (T, 1)))).astype(np.float32)
    if extreme:
        blk = W.reshape(n_out, -1, 34)
        blk[:, :, 2:] = np.uint8(0x80)                   # every weight -128
        q[:] = -127
        q[:, ::2] = 127
        q[0] = 127
    return W, q, d


def dense_ref(W, q, d):
    """-> (y, sum of the blocks' magnitudes), 64 bits"""
    n_out = W.shape[0]
    blk = W.reshape(n_out, -1, 34)
    wd = np.ascontiguousarray(blk[:, :, :2]).view(np.float16).astype(np.float64)[:, :, 0]
    wq = np.ascontiguousarray(blk[:, :, 2:]).view(np.int8).astype(np.float64)
    T, nb = d.shape
    y, mag = np.zeros((T, n_out)), np.zeros((T, n_out))
    for b in range(nb):
        term = (q[:, 32 * b:32 * b + 32].astype(np.float64) @ wq[:, b].T) * wd[:, b] * d[:, b, None].astype(np.float64)
        y += term
        mag += np.abs(term)
    return y, mag


def run_dense(n_in, n_out, T, seed=0, pad=0, shift=0, extreme=False):
    W, q, d = dense_case(n_in, n_out, T, seed, extreme)
    w = scan.DenseWeight(W)
    qs, ds, y = padded(q, 16 * pad, 16 * shift, fill=99), padded(d, pad, shift), Out(T, n_out, pad, shift)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qs[1], qs[2], ds[1], ds[2]), T, y.ptr, y.ld)
    got = y.get()
    want, mag = dense_ref(W, q, d)
    bound = (n_in // 32 + 10) * U * mag
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300)))
    w.close()


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("n_in, n_out", [(32, 1), (64, 33), (96, 257), (160, 64), (1152, 130)])
def test_dense_small(hip, n_in, n_out, T):
    run_dense(n_in, n_out, T, seed=n_in + T)


@pytest.mark.parametrize("n_in, n_out, T", [(4096, 515, 1), (14336, 128, 3), (2592, 1000, 12), (6912, 300, 40), (1152, 1100, 300), (4096, 129, 513), (4128, 640, 130), (128, 384, 1025)])
@pytest.mark.parametrize("pad, shift", [(0, 0), (1, 1), (4, 0)])
def test_dense_larger_strided(hip, n_in, n_out, T, pad, shift):
    run_dense(n_in, n_out, T, seed=7, pad=pad, shift=shift)


@pytest.mark.parametrize("T", [1, 6, 33, 140])
def test_dense_largest_quants(hip, T):
    run_dense(256, 160, T, extreme=True)


@pytest.mark.parametrize("T", [1, 4, 40, 200])
def test_dense_scale_that_is_not_finite_stays_in_its_row(hip, T):
    W, q, d = dense_case(320, 200, T, 5)
    bad = T - 1
    d[bad, 3], q[bad, 96:128] = np.nan, 0                # what the norm writes for a block that is not finite
    w, qd, dd, y = scan.DenseWeight(W), dev(q), dev(d), Out(T, 200)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qd.data_ptr(), 320, dd.data_ptr(), 10), T, y.ptr, y.ld)
    got = y.get()
    assert np.all(np.isnan(got[bad]))
    want, mag = dense_ref(W, q[:bad], d[:bad])
    assert np.all(np.abs(got[:bad] - want) <= 20 * U * mag)
    w.close()


@pytest.mark.parametrize("T", [1, 2, 4, 40, 200])
@pytest.mark.parametrize("n_in", [96, 320, 1056])
def test_dense_infinite_scales_stay_infinite(hip, n_in, T):
    """An infinite scale, of the weight or of x, meets no zero that the formula does not have: the output is infinite and not NaN."""
    W, q, d = dense_case(n_in, 200, T, 6)
    nb = n_in // 32
    blk = W.reshape(200, nb, 34)
    for o, b, v in ((0, nb - 1, 5), (3, max(0, nb - 3), 251), (199, 0, 5), (70, nb // 2, 5)):
        blk[o, b, :2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
        blk[o, b, 2:] = v                                # all 5, or all -5
    q[:] = np.maximum(np.abs(q), 1)                      # no sum of these blocks is zero
    blk[:, max(0, nb - 3), 2:][blk[:, max(0, nb - 3), 2:] == 0] = 1
    for b, t in ((nb - 1, 0), (max(0, nb - 3), T - 1)):
        d[t, b] = np.inf
    w, qd, dd, y = scan.DenseWeight(W), dev(q), dev(d), Out(T, 200)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qd.data_ptr(), n_in, dd.data_ptr(), nb), T, y.ptr, y.ld)
    got = y.get()
    with np.errstate(invalid="ignore"):
        want, mag = dense_ref(W, q, d)
    for value in (np.inf, -np.inf):
        assert np.array_equal(got == value, want == value)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isinf(want).any()
    fin = np.isfinite(want)
    assert np.all(np.abs(got - np.where(fin, want, 0))[fin] <= ((nb + 10) * U * mag)[fin])
    w.close()


# enough workgroups for each form to be the cheapest one: 16 x 16, 32 x 32, 64 x 64, 64 x 128, 128 x 128 tiles, rows of one and two blocks,
# tiles of 48 and 64 rows
FORMS = [(160, 13000, 2), (416, 5000, 70), (1056, 2900, 300), (160, 5000, 700), (288, 4500, 1500), (32, 2900, 300), (64, 4500, 1500),
         (2080, 10001, 9), (2112, 14003, 16), (2080, 10010, 29), (2112, 14001, 25)]


@pytest.mark.parametrize("n_in, n_out, T", FORMS)
@pytest.mark.parametrize("pad, shift", [(0, 0), (1, 1)])
def test_dense_many_workgroups(hip, n_in, n_out, T, pad, shift):
    run_dense(n_in, n_out, T, seed=n_in, pad=pad, shift=shift)


@pytest.mark.parametrize("n_in, n_out, T", FORMS[:5] + FORMS[7:])
def test_dense_many_workgroups_infinite_scales(hip, n_in, n_out, T):
    """In the first and the last block, where steps end: infinite outputs stay infinite, the others what they are."""
    W, q, d = dense_case(n_in, n_out, T, 8)
    nb = n_in // 32
    blk = W.reshape(n_out, nb, 34)
    q[:] = np.maximum(np.abs(q), 1)
    for o, b, v in ((0, nb - 1, 5), (n_out - 1, 0, 251), (n_out // 2, nb - 1, 7)):
        blk[o, b, :2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
        blk[o, b, 2:] = v                                # one sign, so no sum of theirs is zero
    d[T - 1, nb - 1] = np.inf
    w, qd, dd, y = scan.DenseWeight(W), dev(q), dev(d), Out(T, n_out)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qd.data_ptr(), n_in, dd.data_ptr(), nb), T, y.ptr, y.ld)
    got = y.get()
    with np.errstate(invalid="ignore"):
        want, mag = dense_ref(W, q, d)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isinf(want[:, 0]).all()
    for value in (np.inf, -np.inf):
        assert np.array_equal(got == value, want == value)
    fin = np.isfinite(want)
    assert np.all(np.abs(got - np.where(fin, want, 0))[fin] <= ((nb + 10) * U * mag)[fin])
    w.close()


@pytest.mark.parametrize("n_in, n_out, T", [(160, 64, 1), (96, 64, 5), (320, 200, 9)] + FORMS[:5])
@pytest.mark.parametrize("scale", [1e-36, 1e-39])
def test_dense_scales_below_the_normal_range(hip, n_in, n_out, T, scale):
    """Products of scales in F32's subnormal range keep its resolution of 2^-149: half a step per block, times the block's integer sum."""
    W, q, d = dense_case(n_in, n_out, T, 9)
    d[:] = (np.abs(np.random.default_rng(1).standard_normal(d.shape)) * scale).astype(np.float32)
    w, qd, dd, y = scan.DenseWeight(W), dev(q), dev(d), Out(T, n_out)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qd.data_ptr(), n_in, dd.data_ptr(), n_in // 32), T, y.ptr, y.ld)
    got = y.get()
    want, mag = dense_ref(W, q, d)
    ones = W.reshape(n_out, -1, 34).copy()
    ones[:, :, :2] = np.frombuffer(np.float16(1).tobytes(), np.uint8)
    _, sums = dense_ref(ones.reshape(W.shape), q, np.ones_like(d))
    nb = n_in // 32
    assert np.all(np.abs(got.astype(np.float64) - want) <= (nb + 10) * U * mag + 2.0 ** -150 * sums + nb * 2.0 ** -149)
    w.close()


def test_dense_refusals(hip):
    q, d, y = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, device="cuda"), torch.zeros(4, 48, device="cuda")
    w = scan.DenseWeight(make_dense(64, 48, "q8_0"))
    args = lambda qp=q.data_ptr(), ldq=64, ldd=2: sublayer.Q8View(qp, ldq, d.data_ptr(), ldd)  # noqa: E731
    for x8, T, ldy in ((args(ldq=48), 4, 48), (args(ldq=72), 4, 48), (args(ldd=1), 4, 48), (args(qp=q.data_ptr() + 8), 2, 48), (args(qp=0), 4, 48), (args(), 4, 47), (args(), -1, 48), (None, 4, 48)):
        with pytest.raises(hip.SeedDeltaError, match=r"\(-1\)"):
            sublayer.dense_forward_q8_device(w, x8, T, y.data_ptr(), ldy)
    for kind in ("f16", "f32"):
        v = scan.DenseWeight(make_dense(64, 48, kind))
        with pytest.raises(hip.SeedDeltaError, match=r"\(-4\)"):
            sublayer.dense_forward_q8_device(v, args(), 4, y.data_ptr(), 48)
        v.close()
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(0, 64, 0, 2), 0, 0, 48)          # no tokens: nothing happens
    w.close()
    torch.cuda.synchronize()
    assert not y.any()


# ---- adapters -------------------------------------------------------------------------------------------------------
def make_adapters(n_in, n_out, ranks, types, seed=0):
    rng = np.random.default_rng(seed)
    t = {"h": np.float16, "f": np.float32}
    return [((rng.standard_normal((r, n_in)) / np.sqrt(n_in)).astype(t[ty[0]]), (0.5 * rng.standard_normal((n_out, r))).astype(t[ty[-1]]), 0.25 * (i + 1) * (-1) ** i)
            for i, (r, ty) in enumerate(zip(ranks, types))]


def lora_ref(adapters, ids, x, base, n_out):
    """-> (y, bound), 64 bits"""
    T, n_in = x.shape
    y = np.zeros((T, n_out)) if base is None else base.astype(np.float64)
    bound = np.zeros((T, n_out))
    for k, (a, b, scale) in enumerate(adapters):
        at = np.nonzero(ids == k)[0]
        if not at.size:
            continue
        a, b, xs, scale, r = a.astype(np.float64), b.astype(np.float64), x[at].astype(np.float64), float(np.float32(scale)), a.shape[0]
        if base is not None:
            bound[at] += (r + 4) * U * np.abs(base[at])
        y[at] += scale * (xs @ a.T) @ b.T
        bound[at] += (n_in + r + 20) * U * abs(scale) * (np.abs(xs) @ np.abs(a).T) @ np.abs(b).T
    return y, bound


def run_lora(adapters, ids, T, base="apart", pad=0, shift=0, seed=0, x=None, stream=0):
    n_in, n_out = adapters[0][0].shape[1], adapters[0][1].shape[0]
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, n_in)).astype(np.float32) if x is None else x
    b = None if base is None else rng.standard_normal((T, n_out)).astype(np.float32)
    s = sublayer.LoraSet(adapters)
    xs, y = padded(x, pad, shift), Out(T, n_out, pad, shift)
    bs = padded(b, pad, shift) if base == "apart" else None
    if base == "in place":
        y.buf[shift:shift + T * y.ld].view(T, y.ld)[:, :n_out] = dev(b)
    idd = None if ids is None else dev(np.asarray(ids, np.int32))
    ws = torch.full((s.workspace_bytes(T) + 64,), 0x5b, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    s.apply_device(0 if ids is None else idd.data_ptr(), xs[1], xs[2], T, y.ptr, y.ld, base_ptr=0 if base is None else y.ptr if base == "in place" else bs[1],
                   ldb=0 if base is None else y.ld if base == "in place" else bs[2], ws_ptr=ws.data_ptr(), ws_bytes=ws.numel() - 64, stream=stream)
    got = y.get()
    assert torch.all(ws[-64:] == 0x5b), "written behind the workspace"
    want, bound = lora_ref(adapters, np.zeros(T, int) if ids is None else np.asarray(ids), x, b, n_out)
    s.close()
    return got, want, bound


def check_lora(*a, **k):
    got, want, bound = run_lora(*a, **k)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300)))


def some_ids(T, n, order, seed=0):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, n, T)
    if order == "runs":
        ids = np.sort(ids)
    if order == "gaps":
        ids[rng.random(T) < 0.3] = -1
        ids[rng.random(T) < 0.1] = n
        ids[rng.random(T) < 0.05] = -2 ** 31
    return ids


@pytest.mark.parametrize("T", [1, 2, 3, 8, 31, 32, 33, 63, 64, 65, 96, 130, 300])
@pytest.mark.parametrize("order", ["each", "runs", "gaps"])
def test_lora_token_counts(hip, T, order):
    ads = make_adapters(160, 260, [8, 16, 3, 40, 1], ["h", "f", "h", "hf", "fh"], seed=T)
    check_lora(ads, some_ids(T, 5, order, T), T, seed=T)


@pytest.mark.parametrize("rank", [1, 2, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 130, 512])
@pytest.mark.parametrize("ty", ["h", "f"])
@pytest.mark.parametrize("T", [1, 5, 70])
def test_lora_ranks(hip, rank, ty, T):
    check_lora(make_adapters(96, 132, [rank, 5], [ty, "h"], seed=rank), some_ids(T, 2, "each", rank), T)


@pytest.mark.parametrize("n_in, n_out", [(1, 1), (3, 5), (8, 4), (31, 33), (33, 1024), (127, 1025), (130, 1028), (544, 2052), (1000, 999)])
@pytest.mark.parametrize("T", [1, 6, 100])
@pytest.mark.parametrize("pad, shift", [(0, 0), (4, 0), (3, 1)])
def test_lora_shapes_and_strides(hip, n_in, n_out, T, pad, shift):
    check_lora(make_adapters(n_in, n_out, [4, 20], ["h", "f"], seed=n_in), some_ids(T, 2, "gaps", T), T, pad=pad, shift=shift)


@pytest.mark.parametrize("T", [1, 4, 64, 65, 200])
@pytest.mark.parametrize("base", [None, "in place"])
def test_lora_base_forms(hip, T, base):
    for n_out in (256, 259):
        check_lora(make_adapters(64, n_out, [16, 8], ["h", "f"]), some_ids(T, 2, "gaps", 3 * T + 1), T, base=base)


@pytest.mark.parametrize("T", [1, 5, 64, 65, 500])
def test_lora_all_none_and_null_ids(hip, T):
    ads = make_adapters(64, 100, [16, 8], ["h", "f"])
    for base in ("apart", "in place", None):
        got, want, _ = run_lora(ads, np.full(T, -1), T, base=base)
        assert np.array_equal(got, want)                 # the base itself, or zeros
    check_lora(ads, None, T)


@pytest.mark.parametrize("T", [65, 127, 128, 129, 200, 255, 256, 257, 513])
@pytest.mark.parametrize("n", [1, 2, 7, 9, 10, 15, 16, 63])
@pytest.mark.parametrize("order", ["runs", "gaps"])
def test_lora_some_hundred_tokens(hip, T, n, order):
    check_lora(make_adapters(40, 70, [1 + 7 * i % 20 for i in range(n)], ["h", "f"] * n, seed=n), some_ids(T, n, order, T), T, base="in place" if T % 2 else None)


@pytest.mark.parametrize("T", [66, 96, 511, 2000])
@pytest.mark.parametrize("base", ["apart", "in place", None])
def test_lora_one_adapter_for_all_tokens(hip, T, base):
    check_lora(make_adapters(200, 300, [20, 8], ["f", "h"]), None, T, base=base, pad=1, shift=1)


@pytest.mark.parametrize("T", [1, 40, 64, 200])
def test_lora_many_adapters(hip, T):
    n = 4096 if T != 40 else 1000
    rng = np.random.default_rng(T)
    ads = [(rng.standard_normal((2, 32)).astype(np.float16), rng.standard_normal((36, 2)).astype(np.float16), 1.0) for _ in range(n)]
    ids = rng.integers(0, n, T)
    ids[-1] = n - 1
    check_lora(ads, ids, T)


@pytest.mark.parametrize("T", [3, 40, 100])
@pytest.mark.parametrize("rank", [5, 16, 70])
def test_lora_values_that_are_not_finite_stay_with_their_token(hip, T, rank):
    ads = make_adapters(96, 140, [rank, 9], ["h", "f"])
    ids = some_ids(T, 2, "each", 8)
    x = np.random.default_rng(1).standard_normal((T, 96)).astype(np.float32)
    x[T // 2, 11] = np.inf
    x[0, 95] = np.nan
    got, want, bound = run_lora(ads, ids, T, x=x)
    bad = np.zeros(T, bool)
    bad[[0, T // 2]] = True
    assert np.all(~np.isfinite(got[bad]))
    assert np.all(np.abs(got[~bad] - want[~bad]) <= bound[~bad])


@pytest.mark.parametrize("T", [4, 64, 90])
def test_lora_a_token_does_not_depend_on_the_others(hip, T):
    ads = make_adapters(300, 500, [16, 8, 24], ["h", "f", "h"])
    rng = np.random.default_rng(0)
    x = rng.standard_normal((T, 300)).astype(np.float32)
    ids = some_ids(T, 3, "each", 1)
    a = run_lora(ads, ids, T, x=x)[0]
    perm = rng.permutation(T)
    # another order and other neighbours (same generator: the same base row belongs to another token, so compare without a base)
    a = run_lora(ads, ids, T, x=x, base=None)[0]
    b = run_lora(ads, ids[perm], T, x=x[perm], base=None)[0]
    assert np.array_equal(bits(a[perm]), bits(b))
    other = ids.copy()
    other[1:] = -1
    assert np.array_equal(bits(run_lora(ads, other, T, x=x, base=None)[0][0]), bits(a[0]))


# ---- adapters, tokens sorted by the plan ----------------------------------------------------------------------------
# More than 256 tokens, or more than 64 of more adapters than a wave deals by itself, are sorted by lora_plan_kernel. The workspace begins with
# its permutation of the tokens, so a test sees that it ran.
def tokens_in_order(ws, T):
    """The workspace's first T numbers, if they are a permutation of the tokens; None: nothing was sorted."""
    perm = ws[:4 * T].cpu().numpy().view(np.int32)
    return perm if np.array_equal(np.sort(perm), np.arange(T)) else None


def run_planned(adapters, ids, x, base=None, pad=0, shift=0):
    """-> (y, 64-bit y, bound); the plan is checked: tokens of an adapter in a row, adapters in order, those without one last"""
    T, n_out, n = len(ids), adapters[0][1].shape[0], len(adapters)
    s, idd = sublayer.LoraSet(adapters), dev(np.asarray(ids, np.int32))
    xs, y = padded(x, pad, shift), Out(T, n_out, pad, shift)
    bs = (None, 0, 0) if base is None else padded(base, pad, shift)
    ws = torch.full((s.workspace_bytes(T) + 64,), 0x5b, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    s.apply_device(idd.data_ptr(), xs[1], xs[2], T, y.ptr, y.ld, base_ptr=bs[1], ldb=bs[2], ws_ptr=ws.data_ptr(), ws_bytes=ws.numel() - 64)
    got = y.get()
    assert torch.all(ws[-64:] == 0x5b), "written behind the workspace"
    perm = tokens_in_order(ws, T)
    assert perm is not None, "not sorted by the plan: the dispatch rule has changed"
    bins = np.where((ids >= 0) & (ids < n), ids, n)
    assert np.all(np.diff(bins[perm]) >= 0)
    s.close()
    return got, *lora_ref(adapters, np.asarray(ids), x, base, n_out)


@pytest.mark.parametrize("T, n, planned", [(64, 40, False), (65, 15, False), (65, 16, True), (128, 16, True), (256, 7, False), (256, 8, True), (257, 1, True), (300, 0, False)])
def test_lora_which_calls_sort_tokens(hip, T, n, planned):
    """n = 0: no ids"""
    s = sublayer.LoraSet(make_adapters(32, 40, [4] * max(n, 1), ["h"] * max(n, 1)))
    x, y, ids = torch.randn(T, 32, device="cuda"), torch.empty(T, 40, device="cuda"), dev(some_ids(T, max(n, 1), "each", T).astype(np.int32))
    ws = torch.full((s.workspace_bytes(T),), 0x5b, dtype=torch.uint8, device="cuda")
    s.apply_device(ids.data_ptr() if n else 0, x.data_ptr(), 32, T, y.data_ptr(), 40, ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
    torch.cuda.synchronize()
    assert (tokens_in_order(ws, T) is not None) == planned
    assert planned or torch.all(ws[:4 * T] == 0x5b)
    s.close()


@pytest.mark.parametrize("T", [65, 300, 1024, 4095, 4096, 4097, 9000])
@pytest.mark.parametrize("n", [16, 40, 1000, 4096])
@pytest.mark.parametrize("order", ["runs", "gaps"])
def test_lora_planned_token_and_adapter_counts(hip, T, n, order):
    rng = np.random.default_rng(T + n)
    ads = [(rng.standard_normal((1 + i % 5, 20)).astype(np.float16), rng.standard_normal((24, 1 + i % 5)).astype(np.float32 if i % 3 else np.float16), 0.5 + i % 4) for i in range(n)]
    got, want, bound = run_planned(ads, some_ids(T, n, order, T), rng.standard_normal((T, 20)).astype(np.float32), rng.standard_normal((T, 24)).astype(np.float32))
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("ids", [np.full(300, -1), np.full(300, 2), np.full(5000, 7), np.arange(300) % 3, np.r_[np.zeros(4999, int), 1], np.r_[2, np.full(4999, -5)]])
def test_lora_planned_lopsided_batches(hip, ids):
    rng = np.random.default_rng(len(ids))
    x, base = rng.standard_normal((len(ids), 70)).astype(np.float32), rng.standard_normal((len(ids), 90)).astype(np.float32)
    got, want, bound = run_planned(make_adapters(70, 90, [16, 3, 40], ["h", "f", "h"]), ids, x, base)
    assert np.all(np.abs(got - want) <= bound)
    none = (ids < 0) | (ids >= 3)
    assert np.array_equal(got[none], base[none])


@pytest.mark.parametrize("rank", [1, 8, 9, 16, 33, 64, 65, 100, 130, 512])
@pytest.mark.parametrize("ty", ["h", "f"])
def test_lora_planned_ranks(hip, rank, ty):
    rng = np.random.default_rng(rank)
    got, want, bound = run_planned(make_adapters(96, 132, [rank, 5], [ty, "h"], seed=rank), some_ids(300, 2, "each", rank), rng.standard_normal((300, 96)).astype(np.float32))
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("n_in, n_out", [(1, 1), (3, 5), (31, 33), (127, 1025), (130, 1028), (544, 2052), (1000, 999)])
@pytest.mark.parametrize("pad, shift", [(4, 0), (3, 1), (0, 2)])
def test_lora_planned_shapes_and_strides(hip, n_in, n_out, pad, shift):
    rng = np.random.default_rng(n_in)
    x, base = rng.standard_normal((300, n_in)).astype(np.float32), rng.standard_normal((300, n_out)).astype(np.float32)
    got, want, bound = run_planned(make_adapters(n_in, n_out, [4, 20], ["h", "f"], seed=n_in), some_ids(300, 2, "gaps", 5), x, base, pad=pad, shift=shift)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("T", [300, 5000])
@pytest.mark.parametrize("rank", [5, 16, 70])
def test_lora_planned_values_that_are_not_finite_stay_with_their_token(hip, T, rank):
    x = np.random.default_rng(1).standard_normal((T, 96)).astype(np.float32)
    x[T // 2, 11], x[0, 95] = np.inf, np.nan
    with np.errstate(invalid="ignore"):
        got, want, bound = run_planned(make_adapters(96, 140, [rank, 9], ["h", "f"]), some_ids(T, 2, "each", 8), x)
    bad = np.zeros(T, bool)
    bad[[0, T // 2]] = True
    assert np.all(~np.isfinite(got[bad]))
    assert np.all(np.abs(got[~bad] - want[~bad]) <= bound[~bad])


@pytest.mark.parametrize("T", [300, 5000])
def test_lora_planned_token_does_not_depend_on_its_place(hip, T):
    """The atomics give a token its place in its adapter's run: another order of the tokens, other neighbours and a second run of the same
    call give every token the same bits."""
    ads = make_adapters(300, 500, [16, 8, 24], ["h", "f", "h"])
    rng = np.random.default_rng(0)
    x, ids, perm = rng.standard_normal((T, 300)).astype(np.float32), some_ids(T, 3, "gaps", 1), rng.permutation(T)
    a = run_planned(ads, ids, x)[0]
    assert np.array_equal(bits(run_planned(ads, ids, x)[0]), bits(a))
    assert np.array_equal(bits(run_planned(ads, ids[perm], x[perm])[0]), bits(a[perm]))
    other = ids.copy()
    other[1::2] = -1
    assert np.array_equal(bits(run_planned(ads, other, x)[0][::2]), bits(a[::2]))


@pytest.mark.parametrize("T", [300, 5000])
def test_lora_planned_captured_and_replayed(hip, T):
    """Recorded as the set's first call; every replay sorts the ids that it finds, with eager calls on the same set in between."""
    n_in, n_out, rng = 160, 264, np.random.default_rng(T)
    s = sublayer.LoraSet(make_adapters(n_in, n_out, [16, 4, 33], ["h", "f", "h"]))
    mk = lambda: dict(x=torch.empty(T, n_in, device="cuda"), y=torch.empty(T, n_out, device="cuda"), ids=torch.zeros(T, dtype=torch.int32, device="cuda"),  # noqa: E731
                      ws=torch.full((s.workspace_bytes(T),), 0x5b, dtype=torch.uint8, device="cuda"))
    call = lambda b, st: s.apply_device(b["ids"].data_ptr(), b["x"].data_ptr(), n_in, T, b["y"].data_ptr(), n_out, base_ptr=b["y"].data_ptr(), ldb=n_out, ws_ptr=b["ws"].data_ptr(), ws_bytes=b["ws"].numel(), stream=st)  # noqa: E731
    cap, eager, side = mk(), mk(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(cap, torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        x, y, ids = rng.standard_normal((T, n_in)).astype(np.float32), rng.standard_normal((T, n_out)).astype(np.float32), some_ids(T, 3, ("each", "runs", "gaps", "gaps")[rep], rep)
        for b in (cap, eager):
            b["x"].copy_(dev(x)); b["y"].copy_(dev(y)); b["ids"].copy_(dev(ids.astype(np.int32)))
        g.replay()
        call(eager, 0)
        torch.cuda.synchronize()
        assert torch.equal(cap["y"], eager["y"]), rep
        assert tokens_in_order(cap["ws"], T) is not None
        want, bound = lora_ref(make_adapters(n_in, n_out, [16, 4, 33], ["h", "f", "h"]), ids, x, y, n_out)
        assert np.all(np.abs(cap["y"].cpu().numpy() - want) <= bound)
    s.close()


def test_lora_planned_on_two_streams_at_once(hip):
    T, n_in, n_out = 600, 512, 1024
    s = sublayer.LoraSet(make_adapters(n_in, n_out, [16, 8], ["h", "f"]))
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(T, n_in, generator=g, device="cuda") for _ in range(2)]
    ids = [torch.randint(-1, 2, (T,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    ws = [torch.empty(s.workspace_bytes(T), dtype=torch.uint8, device="cuda") for _ in range(2)]
    run = lambda k, y, st: s.apply_device(ids[k].data_ptr(), xs[k].data_ptr(), n_in, T, y.data_ptr(), n_out, ws_ptr=ws[k].data_ptr(), ws_bytes=ws[k].numel(), stream=st)  # noqa: E731
    lone, both, streams = [torch.empty(T, n_out, device="cuda") for _ in range(2)], [torch.empty(T, n_out, device="cuda") for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        run(k, lone[k], 0)
    torch.cuda.synchronize()
    for _ in range(5):
        for k in range(2):
            run(k, both[k], streams[k].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(lone[0], both[0]) and torch.equal(lone[1], both[1])
    assert all(tokens_in_order(w, T) is not None for w in ws)
    s.close()


def test_lora_strided_host_views(hip):
    rng = np.random.default_rng(0)
    big_a, big_b = rng.standard_normal((40, 200)).astype(np.float16), rng.standard_normal((12, 300)).astype(np.float16)
    a, b = big_a[::2, 3:99], big_b.T[::3]                # rows 400 bytes apart; columns strided
    assert not b.flags.c_contiguous
    check_lora([(a[:12], b, 0.5), (a[:7].astype(np.float32), np.ascontiguousarray(b[:, :7]), 1.0)], np.array([0, 1, 1, 0, -1]), 5)


def test_lora_more_tokens_than_one_pass(hip):
    """Over 2^20 tokens the call takes them in passes; the workspace it asks for covers each."""
    T = (1 << 20) + 700
    rng = np.random.default_rng(0)
    ads = make_adapters(3, 4, [2, 9], ["h", "f"])
    ids = rng.integers(-1, 3, T)
    ids[-700:] = 1
    check_lora(ads, ids, T, x=rng.standard_normal((T, 3)).astype(np.float32))


def test_lora_workspace_of_the_most_tokens_serves_fewer(hip):
    s = sublayer.LoraSet(make_adapters(4096, 64, [16, 8], ["h", "h"]))
    counts = sorted({max(1, c + d) for e in range(0, 22) for c in [1 << e] for d in (-1, 0, 1)} | {3000, 5000, 3 << 20})
    need = [s.workspace_bytes(T) for T in counts]
    assert need == sorted(need)
    T, most = 2048, 2049                                    # the shorter call has twice the splits
    x = torch.randn(T, 4096, device="cuda")
    y = torch.zeros(T, 64, device="cuda")
    ws = torch.empty(s.workspace_bytes(most), dtype=torch.uint8, device="cuda")
    s.apply_device(0, x.data_ptr(), 4096, T, y.data_ptr(), 64, ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
    torch.cuda.synchronize()
    assert torch.isfinite(y).all() and (y != 0).any(dim=1).all()


def test_lora_wide_output(hip):
    """A million columns: few tokens a pass."""
    ads = make_adapters(4, 1 << 20, [3, 1], ["f", "h"])
    check_lora(ads, some_ids(70, 2, "gaps", 1), 70)


def test_lora_refusals(hip):
    ads = make_adapters(64, 48, [8], ["h"])
    s = sublayer.LoraSet(ads)
    assert s.stored_bytes == 8 * (64 + 48) * 2 and s.workspace_bytes(0) == 0
    x, y, ids = torch.zeros(4, 64, device="cuda"), torch.zeros(4, 48, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    n = s.workspace_bytes(4)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    good = dict(ids_ptr=ids.data_ptr(), x_ptr=x.data_ptr(), ldx=64, T=4, y_ptr=y.data_ptr(), ldy=48, base_ptr=0, ldb=0, ws_ptr=ws.data_ptr(), ws_bytes=n)
    for k in (dict(x_ptr=0), dict(y_ptr=0), dict(ws_ptr=0), dict(ws_bytes=n - 1), dict(ws_ptr=ws.data_ptr() + 8), dict(ldx=63), dict(ldy=47), dict(T=-1),
              dict(base_ptr=y.data_ptr(), ldb=49, ldy=48), dict(base_ptr=x.data_ptr(), ldb=47), dict(ids_ptr=ids.data_ptr() + 2), dict(x_ptr=x.data_ptr() + 1), dict(x_ptr=y.data_ptr(), ldx=64)):
        with pytest.raises(hip.SeedDeltaError, match=r"\(-1\)"):
            s.apply_device(**{**good, **k})
    with pytest.raises(hip.SeedDeltaError):
        s.workspace_bytes(-1)
    s.apply_device(0, 0, 64, 0, 0, 48)                   # no tokens: nothing happens
    s.apply_device(**good)
    torch.cuda.synchronize()
    s.close()


# ---- streams and graphs ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 6, 100])
def test_context_runs_build_lora_mm_on_the_device(hip, T):
    """SeedDeltaContext.mul_mat_device: a payload, a dense weight and a key without either, with and without adapters; the results
    are those of the calls it is made of, bit for bit."""
    n, n_out = 256, 512
    ctx = hip.SeedDeltaContext()
    p, W, ads = make_payload(n, n_out, scheme="coo", K=16, base=True, seed=1), make_dense(n, n_out, "q8_0", 2), make_adapters(n, n_out, [8, 20], ["h", "f"])
    assert ctx.try_add("up", p)
    ctx.add_dense("gate", W)
    with pytest.raises(hip.SeedDeltaError):
        ctx.add_dense("gate16", make_dense(n, n_out, "f16"))
    for k in ("up", "gate"):
        ctx.add_adapters(k, ads)
    x = torch.randn(T, n, device="cuda")
    q, d, ids = torch.empty(T, n, dtype=torch.int8, device="cuda"), torch.empty(T, n // 32, device="cuda"), dev(some_ids(T, 2, "gaps", T).astype(np.int32))
    x8 = sublayer.Q8View(q.data_ptr(), n, d.data_ptr(), n // 32)
    sublayer.q8_quantize_device(x.data_ptr(), n, n, T, x8)
    ws = torch.empty(ctx.workspace_bytes("up", T), dtype=torch.uint8, device="cuda")
    assert ctx.workspace_bytes("down", T) == 0
    assert not ctx.mul_mat_device("down", x.data_ptr(), n, T, 0, n_out)
    w, dw, s = hip.SeedDeltaWeight(p), scan.DenseWeight(W), sublayer.LoraSet(ads)
    for key in ("up", "gate"):
        for with_ids in (False, True):
            got, want = torch.empty(T, n_out, device="cuda"), torch.empty(T, n_out, device="cuda")
            i = ids.data_ptr() if with_ids else 0
            assert ctx.mul_mat_device(key, x.data_ptr(), n, T, got.data_ptr(), n_out, x8=x8, ids_ptr=i, ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
            if key == "up":
                w.forward_device(x.data_ptr(), n, T, want.data_ptr(), n_out)
            else:
                sublayer.dense_forward_q8_device(dw, x8, T, want.data_ptr(), n_out)
            if with_ids:
                s.apply_device(i, x.data_ptr(), n, T, want.data_ptr(), n_out, base_ptr=want.data_ptr(), ldb=n_out, ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
            torch.cuda.synchronize()
            assert torch.equal(got, want), (key, with_ids)
    ctx.enabled = False                                   # payloads off: "up" has no dense weight to go to
    assert not ctx.mul_mat_device("up", x.data_ptr(), n, T, 0, n_out)
    for v in (w, dw, s):
        v.close()


@pytest.mark.parametrize("dims", [(512, 512), (128, 512), (256, 544)])
def test_context_refuses_adapters_of_another_projection(hip, dims):
    ctx = hip.SeedDeltaContext()
    ctx.add_dense("up", make_dense(256, 512, "q8_0", 2))
    ctx.add_adapters("up", make_adapters(*dims, [8], ["h"]))
    x, y = torch.zeros(2, 512, device="cuda"), torch.full((2, 544), 7.0, device="cuda")
    with pytest.raises(hip.SeedDeltaError, match="adapters of"):
        ctx.mul_mat_device("up", x.data_ptr(), 512, 2, y.data_ptr(), 544)
    assert torch.all(y == 7.0)


@pytest.mark.parametrize("T", [1, 6, 100])
def test_context_captured_and_replayed(hip, T):
    """mul_mat_device of a payload and of a dense key, with adapters, recorded after one eager call of as many tokens. Eager calls of more
    tokens between the replays take larger workspaces of the payload's handle: the graph keeps its own."""
    n, n_out, most = 1024, 2048, 5 * T + 3
    ctx, rng = hip.SeedDeltaContext(), np.random.default_rng(T)
    assert ctx.try_add("up", make_payload(n, n_out, scheme="coo", K=16, base=True, seed=1))
    ctx.add_dense("gate", make_dense(n, n_out, "q8_0", 2))
    ads = make_adapters(n, n_out, [8, 20], ["h", "f"])
    for k in ("up", "gate"):
        ctx.add_adapters(k, ads)

    def buffers(T):
        return dict(T=T, x=torch.zeros(T, n, device="cuda"), q=torch.empty(T, n, dtype=torch.int8, device="cuda"), d=torch.empty(T, n // 32, device="cuda"),
                    ids=torch.zeros(T, dtype=torch.int32, device="cuda"), up=torch.empty(T, n_out, device="cuda"), gate=torch.empty(T, n_out, device="cuda"),
                    ws=torch.empty(ctx.workspace_bytes("up", T), dtype=torch.uint8, device="cuda"))

    def call(b, st):
        x8 = sublayer.Q8View(b["q"].data_ptr(), n, b["d"].data_ptr(), n // 32)
        sublayer.q8_quantize_device(b["x"].data_ptr(), n, n, b["T"], x8, stream=st)
        for k in ("up", "gate"):
            assert ctx.mul_mat_device(k, b["x"].data_ptr(), n, b["T"], b[k].data_ptr(), n_out, x8=x8, ids_ptr=b["ids"].data_ptr(), ws_ptr=b["ws"].data_ptr(), ws_bytes=b["ws"].numel(), stream=st)

    cap, eager, more = buffers(T), buffers(T), [buffers(m) for m in (T + 1, 2 * T, most)]
    call(eager, 0)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        call(cap, torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        x, ids = dev(rng.standard_normal((T, n)).astype(np.float32)), dev(rng.integers(-1, 3, T).astype(np.int32))
        for b in (cap, eager):
            b["x"].copy_(x); b["ids"].copy_(ids)
        for k in ("up", "gate"):
            cap[k].fill_(-7.0)
        g.replay()
        call(eager, 0)
        torch.cuda.synchronize()
        for k in ("up", "gate"):
            assert torch.equal(cap[k], eager[k]), (rep, k)
        if rep < len(more):
            call(more[rep], 0)
            torch.cuda.synchronize()


def test_norm_more_rows_than_one_launch(hip):
    """Over 2^21 rows: the launch is cut."""
    T, n = (1 << 21) + 5, 4
    x = torch.randn(T, n, device="cuda")
    y = torch.empty_like(x)
    sublayer.rms_norm_device(x.data_ptr(), n, n, T, eps=EPS, y_ptr=y.data_ptr(), ldy=n)
    torch.cuda.synchronize()
    z = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + float(np.float32(EPS)))
    assert torch.all((y - z).abs() <= (U + 1e-12) * z.abs())


@pytest.mark.parametrize("T", [1, 9, 80])
def test_operators_captured_and_replayed(hip, T):
    """The four calls recorded into one graph as their very first call, replayed with changing inputs and ids, eager work on the same
    handles in between; every replay equals the eager result bit for bit."""
    n, n_out, rng = 256, 384, np.random.default_rng(T)
    w, s = scan.DenseWeight(make_dense(n, n_out, "q8_0")), sublayer.LoraSet(make_adapters(n, n_out, [16, 4, 33], ["h", "f", "h"]))
    mk = lambda: dict(x=torch.empty(T, n, device="cuda"), r=torch.empty(T, n, device="cuda"), y=torch.empty(T, n, device="cuda"),  # noqa: E731
                      q=torch.empty(T, n, dtype=torch.int8, device="cuda"), d=torch.empty(T, n // 32, device="cuda"), o=torch.empty(T, n_out, device="cuda"),
                      ids=torch.zeros(T, dtype=torch.int32, device="cuda"), ws=torch.empty(s.workspace_bytes(T), dtype=torch.uint8, device="cuda"))

    def call(b, st):
        q8 = sublayer.Q8View(b["q"].data_ptr(), n, b["d"].data_ptr(), n // 32)
        sublayer.rms_norm_device(b["x"].data_ptr(), n, n, T, res_ptr=b["r"].data_ptr(), ldr=n, sum_ptr=b["x"].data_ptr(), lds=n, y_ptr=b["y"].data_ptr(), ldy=n, q8=q8, stream=st)
        sublayer.dense_forward_q8_device(w, q8, T, b["o"].data_ptr(), n_out, stream=st)
        s.apply_device(b["ids"].data_ptr(), b["y"].data_ptr(), n, T, b["o"].data_ptr(), n_out, base_ptr=b["o"].data_ptr(), ldb=n_out, ws_ptr=b["ws"].data_ptr(), ws_bytes=b["ws"].numel(), stream=st)
        sublayer.q8_quantize_device(b["x"].data_ptr(), n, n, T, q8, stream=st)

    cap, eager, side = mk(), mk(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(cap, torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        x, r, ids = rng.standard_normal((T, n)).astype(np.float32), rng.standard_normal((T, n)).astype(np.float32), rng.integers(-1, 4, T).astype(np.int32)
        for b in (cap, eager):
            b["x"].copy_(dev(x)); b["r"].copy_(dev(r)); b["ids"].copy_(dev(ids))
        g.replay()
        call(eager, 0)
        torch.cuda.synchronize()
        for k in ("x", "y", "q", "d", "o"):
            assert torch.equal(cap[k], eager[k]), (rep, k)
    w.close(); s.close()


def test_two_streams_at_once(hip):
    """One set, two streams, a workspace each: both results are the lone ones."""
    T, n_in, n_out = 200, 512, 1024
    s = sublayer.LoraSet(make_adapters(n_in, n_out, [16, 8], ["h", "f"]))
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(T, n_in, generator=g, device="cuda") for _ in range(2)]
    ids = [torch.randint(-1, 2, (T,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    ws = [torch.empty(s.workspace_bytes(T), dtype=torch.uint8, device="cuda") for _ in range(2)]
    run = lambda k, y, st: s.apply_device(ids[k].data_ptr(), xs[k].data_ptr(), n_in, T, y.data_ptr(), n_out, ws_ptr=ws[k].data_ptr(), ws_bytes=ws[k].numel(), stream=st)  # noqa: E731
    lone, both, streams = [torch.empty(T, n_out, device="cuda") for _ in range(2)], [torch.empty(T, n_out, device="cuda") for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        run(k, lone[k], 0)
    torch.cuda.synchronize()
    for _ in range(5):
        for k in range(2):
            run(k, both[k], streams[k].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(lone[0], both[0]) and torch.equal(lone[1], both[1])
    s.close()


# ---- rows far apart -------------------------------------------------------------------------------------------------
def far(T, n, dtype, align=4):
    """(T, n) rows whose last one begins past 2^32 elements of a buffer -> (buffer, view, stride)"""
    ld = (2 ** 32 // (T - 1) + n + align) // align * align
    buf = torch.empty((T - 1) * ld + n, dtype=dtype, device="cuda")
    return buf, buf.as_strided((T, n), (ld, 1)), ld


@pytest.mark.parametrize("T", [3, 40, 700])
def test_rows_past_32_bits_norm_and_dense(hip, T):
    n, n_out = 256, 320
    rng = np.random.default_rng(T)
    x = rng.standard_normal((T, n)).astype(np.float32)
    W = make_dense(n, n_out, "q8_0", 3)
    keep, xv, ldx = far(T, n, torch.float32)
    xv.copy_(dev(x))
    kq, qv, ldq = far(T, n, torch.int8, 16)
    d, y = torch.empty(T, n // 32, device="cuda"), torch.empty(T, n, device="cuda")
    sublayer.rms_norm_device(xv.data_ptr(), ldx, n, T, eps=EPS, sum_ptr=xv.data_ptr(), lds=ldx, y_ptr=y.data_ptr(), ldy=n, q8=sublayer.Q8View(qv.data_ptr(), ldq, d.data_ptr(), n // 32))
    torch.cuda.synchronize()
    s, z = norm_ref(x, None, None)
    assert np.array_equal(bits(xv.contiguous().cpu().numpy()), bits(s)) and np.all(np.abs(y.cpu().numpy() - z) <= (U + 1e-12) * np.abs(z))
    q, dh = qv.contiguous().cpu().numpy(), d.cpu().numpy()
    check_q8(q, dh, z)
    del keep, xv
    ko, ov, ldo = far(T, n_out, torch.float32)
    w = scan.DenseWeight(W)
    sublayer.dense_forward_q8_device(w, sublayer.Q8View(qv.data_ptr(), ldq, d.data_ptr(), n // 32), T, ov.data_ptr(), ldo)
    want, mag = dense_ref(W, q, dh)
    assert np.all(np.abs(ov.contiguous().cpu().numpy() - want) <= (n // 32 + 10) * U * mag)
    w.close()


@pytest.mark.parametrize("T", [3, 40, 130, 700])
def test_rows_past_32_bits_adapters(hip, T):
    n_in, n_out = 160, 300
    ads, ids, rng = make_adapters(n_in, n_out, [8, 20, 33], ["h", "f", "h"]), some_ids(T, 3, "gaps", T), np.random.default_rng(T)
    ids[-1] = 1
    x, base = rng.standard_normal((T, n_in)).astype(np.float32), rng.standard_normal((T, n_out)).astype(np.float32)
    (kx, xv, ldx), (ky, yv, ldy) = far(T, n_in, torch.float32), far(T, n_out, torch.float32)
    xv.copy_(dev(x)); yv.copy_(dev(base))
    s, idd = sublayer.LoraSet(ads), dev(ids.astype(np.int32))
    ws = torch.empty(s.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    s.apply_device(idd.data_ptr(), xv.data_ptr(), ldx, T, yv.data_ptr(), ldy, base_ptr=yv.data_ptr(), ldb=ldy, ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
    want, bound = lora_ref(ads, ids, x, base, n_out)
    assert np.all(np.abs(yv.contiguous().cpu().numpy() - want) <= bound)
    s.close()


# ---- a run of them together -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 3, 40])
def test_ffn_sublayer_with_a_dense_gate_and_adapters(hip, T):
    """One FFN sublayer of a model whose gate stayed dense while up and down have payloads, every projection with adapters:
    residual + norm (F32 for up, 8 bit for gate) -> gate / up + adapters -> act(g) u -> down + adapters, added to the stream. Each
    step is held to its own tolerance on the values that the step before it left on the device."""
    n_embd, n_ff, rng = 256, 640, np.random.default_rng(T)
    Wg = make_dense(n_embd, n_ff, "q8_0", 1)
    pu, pd = make_payload(n_embd, n_ff, scheme="coo", K=32, base=True, seed=2), make_payload(n_ff, n_embd, scheme="block", K=64, block=16, base=True, seed=3)
    wg, wu, wd = scan.DenseWeight(Wg), hip.SeedDeltaWeight(pu), hip.SeedDeltaWeight(pd)
    ads = {k: make_adapters(i, o, [8, 16], ["h", "f"], seed=5) for k, i, o in (("gate", n_embd, n_ff), ("up", n_embd, n_ff), ("down", n_ff, n_embd))}
    sets = {k: sublayer.LoraSet(v) for k, v in ads.items()}
    ids = some_ids(T, 2, "gaps", T)
    idd = dev(ids.astype(np.int32))
    x, att = rng.standard_normal((2, T, n_embd)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(n_embd)).astype(np.float32)
    xd, ad, wt = dev(x), dev(att), dev(w)
    stream_d, norm_d = torch.empty(T, n_embd, device="cuda"), torch.empty(T, n_embd, device="cuda")
    q, d = torch.empty(T, n_embd, dtype=torch.int8, device="cuda"), torch.empty(T, n_embd // 32, device="cuda")
    q8 = sublayer.Q8View(q.data_ptr(), n_embd, d.data_ptr(), n_embd // 32)
    sublayer.rms_norm_device(xd.data_ptr(), n_embd, n_embd, T, weight_ptr=wt.data_ptr(), eps=EPS, res_ptr=ad.data_ptr(), ldr=n_embd,
                             sum_ptr=stream_d.data_ptr(), lds=n_embd, y_ptr=norm_d.data_ptr(), ldy=n_embd, q8=q8)
    proj = {k: torch.empty(T, o, device="cuda") for k, o in (("gate", n_ff), ("up", n_ff), ("down", n_embd))}
    full = {k: torch.empty_like(v) for k, v in proj.items()}

    def adapt(k, inp):
        ws = torch.empty(sets[k].workspace_bytes(T), dtype=torch.uint8, device="cuda")
        sets[k].apply_device(idd.data_ptr(), inp.data_ptr(), inp.shape[1], T, full[k].data_ptr(), full[k].shape[1], base_ptr=proj[k].data_ptr(), ldb=proj[k].shape[1], ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())

    sublayer.dense_forward_q8_device(wg, q8, T, proj["gate"].data_ptr(), n_ff)
    adapt("gate", norm_d)
    wu.forward_device(norm_d.data_ptr(), n_embd, T, proj["up"].data_ptr(), n_ff)
    adapt("up", norm_d)
    h = torch.empty(T, n_ff, device="cuda")
    hip.glu_device(hip.ACT_SILU, full["gate"].data_ptr(), full["up"].data_ptr(), h.data_ptr(), T * n_ff)
    wd.forward_device(h.data_ptr(), n_ff, T, proj["down"].data_ptr(), n_embd)
    adapt("down", h)
    out = torch.empty(T, n_embd, device="cuda")
    sublayer.rms_norm_device(full["down"].data_ptr(), n_embd, n_embd, T, res_ptr=stream_d.data_ptr(), ldr=n_embd, sum_ptr=out.data_ptr(), lds=n_embd)
    torch.cuda.synchronize()
    host = lambda t: t.cpu().numpy()  # noqa: E731
    s, z = norm_ref(x, att, w)
    assert np.array_equal(bits(host(stream_d)), bits(s))
    assert np.all(np.abs(host(norm_d) - z) <= (U + 1e-12) * np.abs(z))
    check_q8(host(q), host(d), z)
    want, mag = dense_ref(Wg, host(q), host(d))
    assert np.all(np.abs(host(proj["gate"]) - want) <= (n_embd // 32 + 10) * U * mag)
    from test_gpu_forward import fast_tolerance
    for k, p, inp in (("up", pu, norm_d), ("down", pd, h)):
        i = host(inp)
        assert np.all(np.abs(host(proj[k]) - O.forward(p, i)) <= fast_tolerance(p, i, None))
    for k, inp in (("gate", norm_d), ("up", norm_d), ("down", h)):
        want, bound = lora_ref(ads[k], ids, host(inp), host(proj[k]), proj[k].shape[1])
        assert np.all(np.abs(host(full[k]) - want) <= bound), k
    assert np.array_equal(bits(host(out)), bits(host(full["down"]) + host(stream_d)))
    # the dense gate against the same weight in F32: 8-bit activations are within half a step of each value
    g64 = z @ dequantize_q8_0(Wg).astype(np.float64).T
    step = np.repeat(np.abs(z).reshape(T, -1, 32).max(2) / 127, 32, axis=1)
    assert np.all(np.abs(host(proj["gate"]) - g64) <= (0.5 + 1e-6) * step @ np.abs(dequantize_q8_0(Wg)).astype(np.float64).T + 1e-5 * np.abs(g64).max())
    for v in (wg, wu, wd, *sets.values()):
        v.close()
