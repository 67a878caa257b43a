"""The 8-bit KV cache (iek_dev_kv8_*) on the device against tests/kv8_ref.py in 64 bits.

Bars: codes, scales, kept slots, lengths and moved weights equal (scales are powers of two, so a value is rounded once);
attention within the f32 error bound that kv8_ref derives, weights within 2^-24 of the same terms."""
import numpy as np
import pytest

import kv8_ref
from inference_engine_rust_amd import engine as E

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"i8": E.I8, "e4m3": E.E4M3}
STALE = 0x7F  # what unwritten slots hold: NaN as e4m3, 127 as int8


def dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).to("cuda")


HELD = []  # small arrays given by address only: alive until their test ends


@pytest.fixture(autouse=True)
def _let_go():
    yield
    HELD.clear()


def ints(x):
    HELD.append(dev(np.asarray(x, np.int32)))
    return HELD[-1]


def stream():
    return torch.cuda.current_stream().cuda_stream


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


class Dev:
    """A cache's buffers on the device, unwritten slots and scales filled with what must not be read."""

    def __init__(self, batch, kv, cap, hd, dtype, ref=None):
        self.shape, self.dtype, self.cap = (batch, kv, cap, hd), dtype, cap
        self.code = [torch.full(self.shape, STALE, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.scale = [torch.full((batch, kv, -(-cap // 32)), float("nan"), device="cuda") for _ in range(2)]
        self.w = torch.full((batch, kv, cap), 5.0, device="cuda")
        self.h = E.KV8Cache(DT[dtype], batch, kv, cap, hd, *(x.data_ptr() for x in self.code + self.scale))
        if ref is not None:
            for i in range(2):
                v = torch.from_numpy(ref.code[i])
                c = v.to(torch.int8) if dtype == "i8" else v.to(torch.float8_e4m3fn)
                self.code[i].copy_(c.view(torch.uint8))
                self.scale[i].copy_(torch.from_numpy(ref.scale[i]))

    def stale_from(self, lens):
        for b, n in enumerate(lens):
            for i in range(2):
                self.code[i][b, :, n:] = STALE
                self.scale[i][b, :, -(-n // 32):] = float("nan")

    def check(self, ref, lens):
        """The live slots hold what the reference holds; the others are as they were."""
        for i in range(2):
            code, scale = host(self.code[i]), host(self.scale[i])
            for b, n in enumerate(lens):
                nb = -(-n // 32)
                assert np.array_equal(scale[b, :, :nb], ref.scale[i][b, :, :nb].astype(np.float32), equal_nan=True), (i, b)
                assert np.isnan(scale[b, :, nb:]).all(), (i, b)
                ok = ~np.isnan(np.repeat(ref.scale[i][b, :, :nb], 32, 1)[:, :n])
                got, want = kv8_ref.decode(code[b, :, :n], self.dtype), ref.code[i][b, :, :n]
                assert np.array_equal(got[ok], want[ok]), (i, b, np.argwhere((got != want) & ok[..., None])[:4])
                assert (code[b, :, n:] == STALE).all(), (i, b)


def filled(seed, batch, kv, cap, hd, dtype, lens):
    """A reference cache with random rows (values of very different size from block to block)."""
    rng = np.random.default_rng(seed)
    ref = kv8_ref.Cache(batch, kv, cap, hd, dtype)
    x = [rng.standard_normal((batch, cap, kv, hd)).astype(np.float32) for _ in range(2)]
    for y in x:
        y *= np.exp2(rng.integers(-6, 3, (batch, -(-cap // 32), kv, 1))).repeat(32, 1)[:, :cap]
    ref.append(x[0], x[1], [0] * batch, lens)
    return ref


# ---- append and load ----

@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 64), (8, 128), (2, 256), (1, 512)])
def test_append_matches_and_leaves_the_rest(gpu, dtype, kv, hd):
    rng = np.random.default_rng(kv * hd)
    batch, cap, n = 5, 133, 70
    start, count = [0, 5, 31, 64, 100], [70, 33, 1, 0, 33]  # (100 + 33: the last slot; 64 + 0: nothing)
    lens0 = [0, 5, 31, 64, 100]
    ref = filled(1, batch, kv, cap, hd, dtype, lens0)
    d = Dev(batch, kv, cap, hd, dtype, ref)
    d.stale_from(lens0)
    pad = 12
    fused = (rng.standard_normal((batch, n, 2 * kv * hd + pad)) * np.exp2(rng.integers(-3, 5, (batch, n, 1)))).astype(np.float32)
    x = dev(fused)
    len_out = ints([-7] * batch)
    E.kv8_append(d.h, x.data_ptr(), x.data_ptr() + 4 * kv * hd, n, fused.shape[2], ints(start).data_ptr(),
                 ints(count).data_ptr(), len_out.data_ptr(), d.w.data_ptr(), stream())
    k, v = (fused[..., i * kv * hd:(i + 1) * kv * hd].reshape(batch, n, kv, hd) for i in range(2))
    want = ref.append(k, v, start, count)
    assert want == [70, 38, 32, 64, 133] and host(len_out).tolist() == want
    d.check(ref, want)
    w = host(d.w)
    for b in range(batch):
        assert (w[b, :, start[b]:want[b]] == 0).all() and (w[b, :, :start[b]] == 5).all() and (w[b, :, want[b]:] == 5).all()
    # and back as values, some rows of it
    out = [torch.full((batch, 50, kv * hd + 4), -3.0, device="cuda") for _ in range(2)]
    s, c = [20, 0, 30, 60, 90], [50, 38, 2, 0, 43]
    E.kv8_load(d.h, 50, kv * hd + 4, ints(s).data_ptr(), ints(c).data_ptr(), out[0].data_ptr(), out[1].data_ptr(), stream())
    for i in range(2):
        got = host(out[i])
        for b in range(batch):
            rows = np.stack([ref.value(i, b, h, want[b]) for h in range(kv)], 1)[s[b]:s[b] + c[b]]
            assert np.array_equal(got[b, :c[b], :kv * hd], rows.reshape(c[b], kv * hd).astype(np.float32)), (i, b)
            assert (got[b, c[b]:] == -3).all() and (got[b, :, kv * hd:] == -3).all()


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_append_token_by_token(gpu, dtype):
    rng = np.random.default_rng(8)
    kv, hd, steps = 2, 128, 75
    ref, d = kv8_ref.Cache(2, kv, 96, hd, dtype), Dev(2, kv, 96, hd, dtype)
    lens = ints([0, 3])
    ref.append(np.ones((2, 3, kv, hd), np.float32), np.ones((2, 3, kv, hd), np.float32), [0, 0], [0, 3])
    one = torch.ones((2, 3, kv, hd), device="cuda")
    E.kv8_append(d.h, one.data_ptr(), one.data_ptr(), 3, kv * hd, 0, ints([0, 3]).data_ptr(), 0, 0, stream())
    at = [0, 3]
    for i in range(steps):
        # growing, shrinking, and now and then a row of zeros or of very small values
        x = rng.standard_normal((2, 2, 1, kv, hd)) * 2.0 ** rng.integers(-4, 6)
        x *= [0.0, 1e-33][i % 2] if i % 11 == 5 else 1.0
        x = x.astype(np.float32)
        k, v = dev(x[0]), dev(x[1])
        E.kv8_append(d.h, k.data_ptr(), v.data_ptr(), 1, kv * hd, lens.data_ptr(), 0, lens.data_ptr(), 0, stream())
        at = ref.append(x[0], x[1], at, [1, 1])
        torch.cuda.synchronize()
    assert host(lens).tolist() == at == [75, 78]
    d.check(ref, at)


def test_append_outside_the_cache(gpu):
    ref, d = kv8_ref.Cache(5, 1, 40, 64, "i8"), Dev(5, 1, 40, 64, "i8")
    x = np.random.default_rng(0).standard_normal((5, 20, 1, 64)).astype(np.float32)
    start, count = [-1, 40, 41, 30, 2 ** 31 - 1], [20, 20, 20, 20, 20]
    lens, t = ints([9] * 5), dev(x)
    E.kv8_append(d.h, t.data_ptr(), t.data_ptr(), 20, 64, ints(start).data_ptr(), ints(count).data_ptr(), lens.data_ptr(),
                 d.w.data_ptr(), stream())
    assert host(lens).tolist() == ref.append(x, x, start, count) == [0, 40, 40, 40, 40]
    code, s = host(d.code[0]), host(d.scale[0])
    for b in range(5):
        first = 30 if b == 3 else 40
        # slots 30 .. 39 of sequence 3 (its block 0 also holds what was there before: NaN scale, kept)
        assert (code[b, 0, :first] == STALE).all()
        assert np.isnan(s[b, 0, 0]) and np.isnan(s[b, 0, 1]) == (b != 3)
    assert np.array_equal(kv8_ref.decode(code[3, :, 32:], "i8")[0], ref.code[0][3, 0, 32:])
    E.kv8_append(d.h, t.data_ptr(), t.data_ptr(), 20, 64, 0, ints([-5, 0, 7, 99, 20]).data_ptr(), lens.data_ptr(), 0, stream())
    assert host(lens).tolist() == [0, 0, 7, 20, 20]


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_scale_borders_and_non_finite(gpu, dtype):
    """Largest values on, just below and just above what a scale holds; infinities and NaN make the scale NaN."""
    top = kv8_ref.TOP[dtype]
    up = np.nextafter(np.float32(top), np.float32(np.inf))
    tops = [top, up, top / 2, 2.0 ** 20 * top, 2.0 ** -100 * top, 2.0 ** -101 * top, 1e-44, 0.0, 3.4028234e38, np.inf, -np.inf,
            np.nan, 1.0, 2.0 ** -90]
    n = 32 * len(tops)
    rng = np.random.default_rng(2)
    x = rng.uniform(-1, 1, (1, n, 1, 64)).astype(np.float32)
    for i, a in enumerate(tops):
        x[0, 32 * i:32 * i + 32] *= np.float32(a if np.isfinite(a) else 1)
        x[0, 32 * i + 7, 0, 9] = a
    ref, d, t = kv8_ref.Cache(1, 1, n, 64, dtype), Dev(1, 1, n, 64, dtype), dev(x)
    E.kv8_append(d.h, t.data_ptr(), t.data_ptr(), n, 64, 0, 0, 0, 0, stream())
    ref.append(x, x, [0], [n])
    assert np.isnan(ref.scale[0][0, 0]).tolist() == [not np.isfinite(a) for a in tops]
    d.check(ref, [n])
    # a NaN scale stays when rows join its block, and reaches every output of its KV head
    E.kv8_append(d.h, t.data_ptr(), t.data_ptr(), 3, 64, ints([32 * 9 + 20]).data_ptr(), 0, 0, 0, stream())
    assert np.isnan(host(d.scale[0])[0, 0, 9])
    for at in (9, 11):
        c = Dev(1, 2, 64, 64, dtype, filled(3, 1, 2, 64, 64, dtype, [64]))
        c.scale[at == 11][0, 1, 1] = float("nan")
        out, _ = attend(c, np.ones((1, 1, 4, 64), np.float32), [64], 0, 0.1)
        assert np.isfinite(out[0, 0, :2]).all() and np.isnan(out[0, 0, 2:]).all()


# ---- attention ----

def attend(d, q, lens, window, scale, w_in=None, w_out=None, max_len=None, q_pad=0):
    batch, n_q, heads, hd = q.shape
    rows = dev(np.concatenate([q.reshape(batch, n_q, -1), np.zeros((batch, n_q, q_pad), np.float32)], 2))
    max_len = max(lens) if max_len is None else max_len
    size = E.kv8_attention_workspace(d.h, heads, n_q, max_len, w_out is not None)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")  # NaN to whoever reads it unwritten
    out = torch.full(q.shape, 77.0, device="cuda")
    E.kv8_attention(d.h, rows.data_ptr(), heads, n_q, heads * hd + q_pad, ints(lens).data_ptr(), max_len, window, scale,
                    out.data_ptr(), w_in.data_ptr() if w_in is not None else 0, w_out.data_ptr() if w_out is not None else 0,
                    ws.data_ptr(), size, stream())
    return host(out), ws


def check_attention(seed, dtype, kv, group, hd, n_q, lens, window, cap=None, weights=True, max_len=None, q_pad=0):
    rng = np.random.default_rng(seed)
    batch, cap = len(lens), cap or max(lens) + 5
    ref = filled(seed, batch, kv, cap, hd, dtype, lens)
    d = Dev(batch, kv, cap, hd, dtype, ref)
    d.stale_from(lens)
    q = (rng.standard_normal((batch, n_q, kv * group, hd)) * np.exp2(rng.integers(-4, 2, (batch, n_q, kv * group, 1)))).astype(np.float32)
    scale = 1 / np.sqrt(hd)
    want, w, bound = ref.attention(q, lens, window, scale)
    w0 = rng.uniform(0, 3, w.shape).astype(np.float32)
    w_in, w_out = dev(w0), torch.full(w.shape, -4.0, device="cuda")
    got, _ = attend(d, q, lens, window, scale, w_in if weights else None, w_out if weights else None, max_len, q_pad)
    worst = np.max(np.abs(got - want) - bound)
    assert worst <= 0, (worst, np.argwhere(np.abs(got - want) > bound)[:5])
    if weights:
        got = host(w_out)
        for b, n in enumerate(lens):
            assert (got[b, :, n:] == -4).all()
            # each share off by the score's error as in the bound of the output, the sum by an ulp an addend
            size = scale * np.abs(q[b]).sum(-1).max() * max([np.abs(ref.value(0, b, h, n)).max() for h in range(kv)] if n else [0])
            rel = (2 * (hd + 16) * size + 32 + n / 32 + 300 + group * n_q) * 2.0 ** -24
            assert (np.abs(got[b, :, :n] - w0[b, :, :n] - w[b, :, :n]) <= rel * w[b, :, :n] + 2.0 ** -22 * w0[b, :, :n] + 1e-30).all()


LENS = [0, 1, 2, 31, 32, 33, 64, 95, 127, 128, 129, 257, 531]


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("kv,group", [(1, 8), (2, 4), (3, 1)])
def test_attention_one_token(gpu, dtype, hd, kv, group):
    check_attention(hd + group, dtype, kv, group, hd, 1, LENS, 0, q_pad=8)


@pytest.mark.parametrize("hd,kv,group,n_q", [(64, 2, 4, 5), (128, 1, 3, 7), (128, 2, 8, 2), (128, 1, 8, 33), (256, 1, 5, 3),
                                             (512, 1, 8, 4), (64, 1, 1, 64)])
@pytest.mark.parametrize("dtype,window", [("i8", 0), ("e4m3", 40)])
def test_attention_several_tokens(gpu, dtype, window, hd, kv, group, n_q):
    check_attention(n_q, dtype, kv, group, hd, n_q, [0, 1, n_q - 1, n_q, 40, 300], window)


@pytest.mark.parametrize("hd,kv,group,n_q,lens", [(64, 2, 8, 9, [4000, 0, 3111]), (128, 1, 8, 33, [5000, 40, 1701]),
                                                  (256, 1, 5, 21, [3000, 1, 2222]), (512, 1, 8, 16, [1500, 700, 15])])
@pytest.mark.parametrize("window", [0, 40, 1400])
def test_attention_several_tokens_long(gpu, hd, kv, group, n_q, lens, window):
    """Enough work for the workgroups that take sixteen columns (without a window and with a long one)."""
    check_attention(hd + window, "e4m3" if window else "i8", kv, group, hd, n_q, lens * 8, window)


@pytest.mark.parametrize("window", [1, 31, 32, 33, 512, 513])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_window(gpu, window, hd):
    check_attention(window, "i8", 1, 8, hd, 1, [1, 33, 511, 512, 513, 1000, 4099], window)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("hd,kv,group", [(128, 8, 4), (512, 1, 8)])
def test_attention_long(gpu, dtype, hd, kv, group):
    check_attention(5, dtype, kv, group, hd, 1, [20011, 9000], 0)


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
@pytest.mark.parametrize("hd,kv,group,n_q,window", [(64, 1, 8, 1, 0), (64, 2, 8, 3, 0), (128, 1, 2, 1, 300)])
def test_attention_many_sequences(gpu, batch, hd, kv, group, n_q, window):
    lens = [(37 * i * i + 5) % 1200 if i % 7 else 0 for i in range(batch)]
    check_attention(batch, "e4m3", kv, group, hd, n_q, lens, window)


def test_attention_max_len_beyond_and_below_the_lengths(gpu):
    check_attention(6, "i8", 2, 4, 128, 1, [40, 700], 0, cap=3000, max_len=3000)
    # lengths above max_len count as max_len
    ref = filled(7, 2, 1, 200, 64, "i8", [200, 200])
    d = Dev(2, 1, 200, 64, "i8", ref)
    q = np.random.default_rng(1).standard_normal((2, 1, 4, 64)).astype(np.float32)
    got, _ = attend(d, q, [200, -3], 0, 0.125, max_len=90)
    want, _, bound = ref.attention(q, [90, 0], 0, 0.125)
    assert (np.abs(got - want) <= bound).all()
    got, _ = attend(d, q, [200, 200], 0, 0.125, max_len=0)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_attention_sizes_of_values(gpu, dtype):
    """Queries and blocks of values whose sizes differ by many powers of two: the shares and the sums keep 32 bits."""
    rng = np.random.default_rng(4)
    ref = filled(4, 1, 1, 256, 128, dtype, [256])
    ref.scale[1][0, 0] = np.exp2([0, -40, 30, -90, 60, -20, 10, -60])
    d = Dev(1, 1, 256, 128, dtype, ref)
    q = rng.standard_normal((1, 1, 8, 128)).astype(np.float32)
    for size in (1.0, 1e-30, 0.0):
        want, _, bound = ref.attention(q * np.float32(size), [256], 0, 0.05)
        got, _ = attend(d, q * np.float32(size), [256], 0, 0.05)
        assert (np.abs(got - want) <= bound).all(), size
    # the large blocks out of sight: what is left is small, and exact to its own size
    ref.code[0][0, 0, :, 0] = np.where(np.isin(np.arange(256) // 32, [1, 3, 7]), 100.0, -100.0) if dtype == "i8" else \
        np.where(np.isin(np.arange(256) // 32, [1, 3, 7]), 104.0, -104.0)
    ref.code[0][0, 0, :, 1:] = 0
    ref.scale[0][0, 0] = 1
    d = Dev(1, 1, 256, 128, dtype, ref)
    q = np.zeros((1, 1, 8, 128), np.float32)
    q[..., 0] = 20.0
    want, _, bound = ref.attention(q, [256], 0, 0.05)
    got, _ = attend(d, q, [256], 0, 0.05)
    assert np.abs(want).max() < 1e-7 and (np.abs(got - want) <= bound).all()
    # large queries: one entry takes everything
    q = (rng.standard_normal((1, 1, 8, 128)) * 1e30).astype(np.float32)
    ref = filled(9, 1, 1, 100, 128, dtype, [100])
    want, _, _ = ref.attention(q, [100], 0, 0.05)
    got, _ = attend(Dev(1, 1, 100, 128, dtype, ref), q, [100], 0, 0.05)
    assert np.allclose(got, want, rtol=1e-6, atol=0)


def test_weights_in_place_and_from_nothing(gpu):
    lens = [70, 3]
    ref = filled(2, 2, 2, 80, 64, "i8", lens)
    d = Dev(2, 2, 80, 64, "i8", ref)
    q = np.random.default_rng(2).standard_normal((2, 1, 4, 64)).astype(np.float32)
    _, w, _ = ref.attention(q, lens, 0, 0.125)
    fresh = torch.full((2, 2, 80), 9.0, device="cuda")
    attend(d, q, lens, 0, 0.125, None, fresh)
    same = fresh.clone()
    attend(d, q, lens, 0, 0.125, same, same)
    a, b = host(fresh), host(same)
    for i, n in enumerate(lens):
        assert np.allclose(a[i, :, :n], w[i, :, :n], rtol=1e-4, atol=1e-9) and (a[i, :, n:] == 9).all()
        assert np.allclose(b[i, :, :n], 2 * w[i, :, :n], rtol=1e-4, atol=1e-9) and (b[i, :, n:] == 9).all()
        assert np.allclose(a[i, :, :n].sum(1), 2, rtol=1e-5)  # two heads a KV head


# ---- eviction ----

def run_evict(d, w, lens, keep, first, last, to=None, max_len=None, index=True, alias=False):
    max_len = d.cap if max_len is None else max_len
    t = to or d
    size = E.kv8_evict_workspace(d.h, max_len, keep)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    ln = ints(lens)
    out = ln if alias else ints([-1] * len(lens))
    idx = torch.full((*d.shape[:2], max(keep, 1)), -9, dtype=torch.int32, device="cuda")
    E.kv8_evict(d.h, t.h, w.data_ptr(), t.w.data_ptr() if to else w.data_ptr(), ln.data_ptr(), out.data_ptr(), max_len, keep,
                first, last, idx.data_ptr() if index else 0, ws.data_ptr(), size, stream())
    return host(out).tolist(), host(idx)


def check_evict(seed, dtype, kv, hd, lens, keep, first, last, w, in_place, cap=None, to_cap=None, alias=False):
    batch, cap = len(lens), cap or max(lens) + 7
    ref = filled(seed, batch, kv, cap, hd, dtype, lens)
    d = Dev(batch, kv, cap, hd, dtype, ref)
    d.stale_from(lens)
    dw = dev(w)
    to = None if in_place else Dev(batch, kv, to_cap or keep + 3, hd, dtype)
    got, idx = run_evict(d, dw, lens, keep, first, last, to, index=not alias, alias=alias)
    left, w_out, want, index = ref.evict(w, lens, keep, first, last, to_cap or (cap if in_place else keep + 3))
    assert got == want
    if not alias:
        for (b, h), slots in index.items():
            assert np.array_equal(idx[b, h, :len(slots)], slots), (b, h)
            assert (idx[b, h, len(slots):] == -9).all()
    ws = host(dw if in_place else to.w)
    for b, n in enumerate(want):
        assert np.array_equal(ws[b, :, :n], w_out[b, :, :n].astype(np.float32), equal_nan=True)
        if not in_place:
            assert (ws[b, :, n:] == 5).all()
    if in_place:  # what lies behind the new length no longer matters
        d.stale_from(want)
    (d if in_place else to).check(left, want)


def some_weights(seed, shape):
    rng = np.random.default_rng(seed)
    w = np.exp(3 * rng.standard_normal(shape)).astype(np.float32)
    return np.where(rng.random(shape) < 0.3, np.float32(0.25), w)  # many equal ones


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("kv,hd", [(2, 64), (3, 128), (1, 256), (1, 512)])
def test_evict(gpu, dtype, kv, hd, in_place):
    lens = [0, 1, 31, 100, 101, 133, 700, 2049]
    for keep, first, last in ((100, 4, 33), (100, 0, 0), (100, 60, 40), (1, 0, 1), (1, 0, 0), (33, 33, 0), (700, 1, 2)):
        check_evict(keep, dtype, kv, hd, lens, keep, first, last, some_weights(keep, (len(lens), kv, 2056)), in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_lengths_in_place_of_themselves_and_nothing_kept(gpu, in_place):
    w = some_weights(1, (3, 2, 207))
    check_evict(2, "i8", 2, 64, [200, 40, 99], 64, 2, 8, w, in_place, alias=True)
    check_evict(2, "e4m3", 2, 64, [200, 40, 0], 0, 0, 0, w, in_place, to_cap=None if in_place else 32)
    check_evict(2, "i8", 2, 64, [200, 40, 99], 200, 5, 100, w, in_place)


def test_evict_order_of_weights(gpu):
    """Infinities, NaN, negative and signed zero weights; all equal; near equal in the last bits."""
    w = np.zeros((4, 1, 1030), np.float32)
    w[0, 0] = np.random.default_rng(0).choice(np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-45, -1e-45, -3, 7], np.float32), 1030)
    w[1, 0] = 1.0
    w[2, 0] = (np.float32(1).view(np.int32) + np.random.default_rng(1).integers(0, 40, 1030)).astype(np.int32).view(np.float32)
    w[3, 0] = -np.arange(1030)
    for keep in (1, 5, 64, 500, 1000, 1022):
        check_evict(1, "i8", 1, 64, [1023, 1023, 1023, 1023], keep, 0, 0, w, False)
        check_evict(1, "i8", 1, 64, [1023, 1023, 1000, 1023], keep, 1, 0, w, True)


def test_evict_long(gpu):
    for in_place in (False, True):
        w = some_weights(3, (2, 2, 40007))
        check_evict(4, "i8", 2, 64, [40000, 33001], 20011, 4, 1024, w, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_very_long(gpu, in_place):
    """Segments of more than one piece; the smallest weight that stays is one of very many, or one of few."""
    w = some_weights(7, (2, 1, 140008))
    w[1] = np.exp(np.random.default_rng(8).standard_normal(140008)).astype(np.float32)
    check_evict(4, "i8", 1, 64, [140001, 131000], 70001, 3, 50, w, in_place)
    check_evict(4, "i8", 1, 64, [33000, 0, 900, 32769], 1000, 1000, 0, some_weights(9, (4, 1, 33007)), in_place)


@pytest.mark.parametrize("hd", [64, 128])
def test_evict_of_many_blocks(gpu, hd):
    check_evict(5, "e4m3", 4, hd, [20000, 17001], 16500, 0, 100, some_weights(5, (2, 4, 20007)), False)


def test_evict_keeps_a_poisoned_block_poisoned(gpu):
    ref = filled(1, 1, 1, 128, 64, "i8", [128])
    ref.scale[0][0, 0, 1] = np.nan
    d, to = Dev(1, 1, 128, 64, "i8", ref), Dev(1, 1, 100, 64, "i8")
    w = np.ones((1, 1, 128), np.float32)
    w[..., 40:60] = 0
    run_evict(d, dev(w), [128], 100, 0, 0, to)
    left, _, _, _ = ref.evict(w, [128], 100, 0, 0, 100)
    assert np.isnan(left.scale[0][0, 0]).any() and not np.isnan(left.scale[0][0, 0]).all()
    to.check(left, [100])


# ---- together ----

@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_a_request_with_a_budget(gpu, dtype):
    """Two prompts, then decoding: each step appends, attends with weights and, over budget, evicts in place."""
    rng = np.random.default_rng(11)
    kv, group, hd, cap, keep = 2, 4, 128, 160, 96
    ref, d = kv8_ref.Cache(2, kv, cap, hd, dtype), Dev(2, kv, cap, hd, dtype)
    w = np.zeros((2, kv, cap))
    prompt = rng.standard_normal((2, 2, 90, kv, hd)).astype(np.float32)
    k, v = dev(prompt[0]), dev(prompt[1])
    lens_dev = ints([0, 0])
    E.kv8_append(d.h, k.data_ptr(), v.data_ptr(), 90, kv * hd, lens_dev.data_ptr(), ints([90, 71]).data_ptr(),
                 lens_dev.data_ptr(), d.w.data_ptr(), stream())
    lens = ref.append(prompt[0], prompt[1], [0, 0], [90, 71])
    for step in range(80):
        x = (rng.standard_normal((2, 2, 1, kv, hd)) * 2.0 ** rng.integers(-2, 3)).astype(np.float32)
        q = (rng.standard_normal((2, 1, kv * group, hd)) * 1.5).astype(np.float32)
        k, v = dev(x[0]), dev(x[1])
        E.kv8_append(d.h, k.data_ptr(), v.data_ptr(), 1, kv * hd, lens_dev.data_ptr(), 0, lens_dev.data_ptr(), d.w.data_ptr(), stream())
        for b in range(2):
            w[b, :, lens[b]] = 0
        lens = ref.append(x[0], x[1], lens, [1, 1])
        got, _ = attend(d, q, lens, 0, 0.09, d.w, d.w, max_len=cap)
        want, step_w, bound = ref.attention(q, lens, 0, 0.09)
        assert (np.abs(got - want) <= bound).all(), step
        w += step_w
        if max(lens) > 120:
            # the selection is checked on the device's own weights: they differ from 64 bits in the last places
            on_dev = host(d.w)
            for b, n in enumerate(lens):
                assert np.allclose(on_dev[b, :, :n], w[b, :, :n], rtol=1e-4, atol=1e-7)
            lens_dev.copy_(ints(lens))
            size = E.kv8_evict_workspace(d.h, cap, keep)
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            E.kv8_evict(d.h, d.h, d.w.data_ptr(), d.w.data_ptr(), lens_dev.data_ptr(), lens_dev.data_ptr(), cap, keep, 4, 32, 0,
                        ws.data_ptr(), size, stream())
            ref, _, lens, index = ref.evict(on_dev, lens, keep, 4, 32)
            for (b, h), slots in index.items():
                w[b, h, :len(slots)] = w[b, h, slots]
            assert host(lens_dev).tolist() == lens
    d.stale_from(lens)
    d.check(ref, lens)


def test_captured_step_replays(gpu):
    """append, attention and an eviction in place of one step captured into a graph, replayed with other rows and lengths,
    eager calls with their own workspace between the replays, against a second cache driven eagerly."""
    kv, group, hd, cap, keep = 2, 4, 64, 128, 64
    ref = filled(5, 2, kv, cap, hd, "i8", [70, 90])
    caches = [Dev(2, kv, cap, hd, "i8", ref) for _ in range(2)]
    for c in caches:
        c.w.copy_(dev(some_weights(1, (2, kv, cap))))
    x = torch.zeros((2, 2, 1, kv * hd), device="cuda")
    q = torch.zeros((2, 1, kv * group * hd), device="cuda")
    state = []
    for c in caches:
        a, e = E.kv8_attention_workspace(c.h, kv * group, 1, cap, True), E.kv8_evict_workspace(c.h, cap, keep)
        state.append(dict(c=c, lens=ints([70, 90]), out=torch.zeros((2, 1, kv * group * hd), device="cuda"),
                          ws=torch.empty(a, dtype=torch.uint8, device="cuda"), es=torch.empty(e, dtype=torch.uint8, device="cuda")))

    def step(s):
        c = s["c"]
        E.kv8_append(c.h, x[0].data_ptr(), x[1].data_ptr(), 1, kv * hd, s["lens"].data_ptr(), 0, s["lens"].data_ptr(),
                     c.w.data_ptr(), stream())
        E.kv8_attention(c.h, q.data_ptr(), kv * group, 1, kv * group * hd, s["lens"].data_ptr(), cap, 0, 0.125,
                        s["out"].data_ptr(), c.w.data_ptr(), c.w.data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream())
        E.kv8_evict(c.h, c.h, c.w.data_ptr(), c.w.data_ptr(), s["lens"].data_ptr(), s["lens"].data_ptr(), cap, keep, 2, 16, 0,
                    s["es"].data_ptr(), s["es"].numel(), stream())

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(state[0])
    for i in range(6):
        g = torch.Generator(device="cuda").manual_seed(i)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        graph.replay()
        step(state[1])
        torch.cuda.synchronize()
        a, b = state
        assert a["lens"].tolist() == b["lens"].tolist() == [64, 64]
        assert torch.equal(a["out"], b["out"]) and torch.isfinite(a["out"]).all() and a["out"].abs().max() > 0
        assert torch.equal(a["c"].w[..., :64], b["c"].w[..., :64])
        for j in range(2):
            assert torch.equal(a["c"].code[j][:, :, :64], b["c"].code[j][:, :, :64])
            assert torch.equal(a["c"].scale[j][:, :, :2], b["c"].scale[j][:, :, :2])


@pytest.mark.parametrize("batch", [1, 3])
def test_captured_attention_follows_the_lengths(gpu, batch):
    """One captured attention with weights, launched for the whole capacity, replayed at lengths from none to all of it."""
    cap, kv, group, hd = 5000, 2, 4, 64
    ref = filled(12, batch, kv, cap, hd, "i8", [cap] * batch)
    d, lens = Dev(batch, kv, cap, hd, "i8", ref), ints([cap] * batch)
    q = np.random.default_rng(3).standard_normal((batch, 1, kv * group, hd)).astype(np.float32)
    dq, out, w = dev(q), torch.zeros((batch, kv * group * hd), device="cuda"), torch.zeros((batch, kv, cap), device="cuda")
    size = E.kv8_attention_workspace(d.h, kv * group, 1, cap, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        E.kv8_attention(d.h, dq.data_ptr(), kv * group, 1, kv * group * hd, lens.data_ptr(), cap, 0, 0.125, out.data_ptr(), 0,
                        w.data_ptr(), ws.data_ptr(), size, stream())
    for n in (1, 40, 0, 531, 5000, 33, 2049):
        now = [max(0, n - 7 * b) for b in range(batch)]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(9)
        w.fill_(-4)
        graph.replay()
        want, want_w, bound = ref.attention(q, now, 0, 0.125)
        assert (np.abs(host(out).reshape(q.shape) - want) <= bound).all(), n
        got = host(w)
        for b in range(batch):
            assert np.allclose(got[b, :, :now[b]], want_w[b, :, :now[b]], rtol=1e-4, atol=1e-9) and (got[b, :, now[b]:] == -4).all()


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with its own workspace and outputs over one cache, give what they give alone."""
    ref = filled(6, 2, 4, 1500, 128, "i8", [1500, 900])
    d, lens = Dev(2, 4, 1500, 128, "i8", ref), ints([1500, 900])
    size = E.kv8_attention_workspace(d.h, 16, 1, 1500, False)
    q = [torch.randn((2, 16 * 128), device="cuda") for _ in range(2)]
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    alone, both = [[torch.zeros((2, 16 * 128), device="cuda") for _ in range(2)] for _ in range(2)]

    def call(i, out, st):
        E.kv8_attention(d.h, q[i].data_ptr(), 16, 1, 16 * 128, lens.data_ptr(), 1500, 0, 0.09, out[i].data_ptr(), 0, 0,
                        ws[i].data_ptr(), size, st)

    for i in range(2):
        call(i, alone, stream())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            call(i, both, streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(alone[i], both[i])


def test_offsets_beyond_32_bits(gpu):
    """K and V of 4.5 GiB each: the last sequence's codes lie past 2^32 bytes (and a head's past 2^31)."""
    batch, kv, cap, hd = 3, 1, 3 * 2 ** 20, 512
    code = [torch.empty((batch, kv, cap, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scale = [torch.empty((batch, kv, cap // 32), device="cuda") for _ in range(2)]
    h = E.KV8Cache(E.I8, batch, kv, cap, hd, *(x.data_ptr() for x in code + scale))
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, batch, 64, kv, hd)).astype(np.float32)
    k, v = dev(x[0]), dev(x[1])
    start = [5, 2 ** 21, cap - 64]
    E.kv8_append(h, k.data_ptr(), v.data_ptr(), 64, hd, ints(start).data_ptr(), 0, 0, 0, stream())
    out = [torch.zeros((batch, 64, kv * hd), device="cuda") for _ in range(2)]
    E.kv8_load(h, 64, hd, ints(start).data_ptr(), 0, out[0].data_ptr(), out[1].data_ptr(), stream())
    for i in range(2):
        ref = kv8_ref.Cache(batch, kv, 64, hd, "i8")
        ref.append(x[0], x[1], [0] * 3, [64] * 3)
        got = host(out[i])
        for b in (1, 2):  # (these start on a block's border, as in the reference)
            assert np.array_equal(got[b], ref.value(i, b, 0, 64).astype(np.float32))
    # a window at the very end, of the length of the rows
    q = rng.standard_normal((batch, 1, 8, hd)).astype(np.float32)
    size = E.kv8_attention_workspace(h, 8, 1, cap, False)
    ws, res, dq = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros((batch, 8 * hd), device="cuda"), dev(q)
    E.kv8_attention(h, dq.data_ptr(), 8, 1, 8 * hd, ints([0, 2 ** 21 + 64, cap]).data_ptr(), cap, 64, 0.04, res.data_ptr(), 0, 0,
                    ws.data_ptr(), size, stream())
    want, _, bound = ref.attention(q, [0, 64, 64], 0, 0.04)
    got = host(res).reshape(batch, 1, 8, hd)
    assert (np.abs(got - want) <= bound).all()


# ---- blocks that hold an infinity or NaN, and queries that see none of them ----

def poisoned(seed, dtype, kv, group, hd, n_q, lens, at, which, window):
    """A cache whose slot at[b] of KV head kv - 1 (None: none) was appended with an infinity in K or V; queries; the reference."""
    rng = np.random.default_rng(seed)
    batch, cap = len(lens), max(lens) + 5
    ref, d = kv8_ref.Cache(batch, kv, cap, hd, dtype), Dev(batch, kv, cap, hd, dtype)
    x = rng.standard_normal((2, batch, cap, kv, hd)).astype(np.float32)
    for b, j in enumerate(at):
        if j is not None:
            x[which, b, j, kv - 1, 3] = np.inf
    k, v = dev(x[0]), dev(x[1])
    E.kv8_append(d.h, k.data_ptr(), v.data_ptr(), cap, kv * hd, 0, ints(lens).data_ptr(), 0, 0, stream())
    ref.append(x[0], x[1], [0] * batch, lens)
    q = rng.standard_normal((batch, n_q, kv * group, hd)).astype(np.float32)
    return ref, d, q, ref.attention(q, lens, window, 0.1)


def same_nan_and_near(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    ok = ~np.isnan(want)
    assert (np.abs(got - want) <= bound)[ok].all()
    return ok


BLIND = [  # (KV heads, group, head_dim, query tokens, lengths, the poisoned slots, window)
    # a block that begins with the last two of three tokens: the first sees none of it; in one chunk, and joined
    *[(2, 2, hd, 3, [32 * m + 2], [32 * m], 0) for hd in (64, 128, 256, 512) for m in (1, 70)],
    # a block whose last slot is the first that the first token's window holds: the others see none of it
    *[(1, 4, hd, 3, [32 * 9 - 1 + w + 2], [32 * 8 + 5], w) for hd in (64, 128, 256, 512) for w in (40, 1400)],
    # sequences beside it, tokens with no entries at all, a poisoned block that is everything
    (2, 4, 128, 5, [0, 3, 34, 35, 700, 33], [None, 1, 32, 32, 672, 0], 0),
    # sixteen columns a workgroup
    (2, 8, 64, 9, [4001, 0, 3113] * 8, [4000, None, 3104] * 8, 0),
    (1, 8, 128, 33, [4015, 41, 2975] * 8, [4000, 32, 2944] * 8, 0),
]


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("which", [0, 1], ids=["k", "v"])
@pytest.mark.parametrize("kv,group,hd,n_q,lens,at,window", BLIND)
def test_attention_of_tokens_that_see_none_of_a_poisoned_block(gpu, kv, group, hd, n_q, lens, at, window, which, dtype):
    ref, d, q, (want, _, bound) = poisoned(hd, dtype, kv, group, hd, n_q, lens, at, which, window)
    got, _ = attend(d, q, lens, window, 0.1)
    ok = same_nan_and_near(got, want, bound)
    assert not ok.all() and ok.any()


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
@pytest.mark.parametrize("where", ["k", "v", "q"])
@pytest.mark.parametrize("kv,group,hd,n_q,lens,at,window", BLIND)
def test_weights_of_entries_that_a_nan_token_does_not_see(gpu, kv, group, hd, n_q, lens, at, window, where, dtype):
    """A token whose scores are NaN (a NaN in its query, or in a key it sees) gives NaN to the entries it sees and
    nothing to the others; a NaN value gives none."""
    ref, d, q, (want, w, bound) = poisoned(hd, dtype, kv, group, hd, n_q, lens, at if where != "q" else [None] * len(lens),
                                           int(where == "v"), window)
    if where == "q":
        q[:, 0, 1, 5] = np.nan  # (the first token of a draft does not see the last entries, nor with a window all the first)
        want, w, bound = ref.attention(q, lens, window, 0.1)
    w_out = torch.full(w.shape, -4.0, device="cuda")
    got, _ = attend(d, q, lens, window, 0.1, None, w_out)
    same_nan_and_near(got, want, bound)
    got = host(w_out)
    for b, n in enumerate(lens):
        assert (got[b, :, n:] == -4).all()
        a, z = got[b, :, :n], w[b, :, :n]
        assert np.array_equal(np.isnan(a), np.isnan(z)), (b, np.argwhere(np.isnan(a) != np.isnan(z))[:4])
        ok = ~np.isnan(z)
        # (relative error of a share as in check_attention)
        keys = max([np.nanmax(np.abs(ref.value(0, b, h, n)), initial=0) for h in range(kv)])
        rel = (2 * (hd + 16) * 0.1 * np.nanmax(np.abs(q[b]).sum(-1)) * keys + 32 + n / 32 + 300 + group * n_q) * 2.0 ** -24
        assert (np.abs(a - z) <= rel * z + 1e-30)[ok].all()


# ---- evictions of more than 32768 entries, which several workgroups a head select ----

def many_weights(n):
    """Rows of n weights whose smallest kept one is hard to place: signs, infinities and NaN; all equal; equal but for a few;
    equal in all but the last bits; one size with many different last bits; NaN only."""
    rng = np.random.default_rng(n)
    w = np.zeros((7, 1, n), np.float32)
    w[0, 0] = rng.choice(np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-45, -1e-45, -3, 7], np.float32), n)
    w[1, 0] = 1.0
    w[2, 0, rng.integers(0, n, 900)] = rng.uniform(0, 1, 900)
    w[3, 0] = (np.float32(1).view(np.int32) + rng.integers(0, 40, n)).astype(np.int32).view(np.float32)
    w[4, 0] = rng.uniform(1, 1.12, n)
    w[5, 0] = np.nan
    w[6, 0] = -np.arange(n)
    return w


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,keep,first,last", [(40001, 1000, 0, 0), (33000, 32000, 4, 500), (70003, 20011, 1, 0), (70003, 1, 0, 0),
                                               (40001, 600, 100, 500), (135000, 90001, 0, 77)])
def test_evict_order_of_many_weights(gpu, n, keep, first, last, in_place):
    w = many_weights(n)
    if keep == first + last:  # (only what the caller names stays, whatever the weights)
        w[6] = np.nan
    lens = [n, n - 1, n - 300, n, n, n, 32769]
    check_evict(3, "i8", 1, 64, lens, keep, first, last, w, in_place, cap=n)


# ---- uses that the documentation names ----

@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_loaded_rows_are_the_caches_of_attention_decode(gpu, dtype):
    """Rows of one sequence read back are the f32 caches that iek_attention_decode takes: the same attention."""
    kv, group, hd, n = 2, 4, 128, 301
    ref = filled(21, 1, kv, 320, hd, dtype, [n])
    d = Dev(1, kv, 320, hd, dtype, ref)
    d.stale_from([n])
    q = np.random.default_rng(2).standard_normal((1, 1, kv * group, hd)).astype(np.float32)
    rows = [torch.full((n, kv, hd), 7.0, device="cuda") for _ in range(2)]
    E.kv8_load(d.h, n, kv * hd, 0, ints([n]).data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), stream())
    out = E.host_attention_decode(q.reshape(-1), host(rows[0]).reshape(-1), host(rows[1]).reshape(-1), kv * group, kv, hd, n, 0, 0.09)
    want, _, bound = ref.attention(q, [n], 0, 0.09)
    got, _ = attend(d, q, [n], 0, 0.09)
    # (bound is of f32 sums in any order: the plain kernel's too)
    assert (np.abs(np.asarray(out).reshape(q.shape) - want) <= bound).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_layers_share_their_lengths(gpu, dtype):
    """Three layers' caches of two sequences: each append reads the lengths before the step and writes those after it, which
    the attentions take; at the end of the step the latter become the former, by a copy or by the layers' evictions."""
    rng = np.random.default_rng(17)
    layers, kv, group, hd, cap, keep = 3, 2, 4, 64, 96, 60
    ref = [kv8_ref.Cache(2, kv, cap, hd, dtype) for _ in range(layers)]
    d = [Dev(2, kv, cap, hd, dtype) for _ in range(layers)]
    length, after, lens = ints([0, 0]), ints([-1, -1]), [0, 0]
    es = torch.empty(E.kv8_evict_workspace(d[0].h, cap, keep), dtype=torch.uint8, device="cuda")
    for step in range(40):
        n, count = (50, [50, 33]) if step == 0 else (1, [1, 1])
        for x, c in zip(ref, d):
            r = rng.standard_normal((2, 2, n, kv, hd)).astype(np.float32)
            k, v, q = dev(r[0]), dev(r[1]), rng.standard_normal((2, 1, kv * group, hd)).astype(np.float32)
            E.kv8_append(c.h, k.data_ptr(), v.data_ptr(), n, kv * hd, length.data_ptr(), ints(count).data_ptr(), after.data_ptr(),
                         c.w.data_ptr(), stream())
            now = x.append(r[0], r[1], lens, count)
            assert host(after).tolist() == now
            got, _ = attend(c, q, now, 0, 0.125, c.w, c.w, max_len=cap)
            want, _, bound = x.attention(q, now, 0, 0.125)
            assert (np.abs(got - want) <= bound).all()
        if max(now) > 80:
            for i, c in enumerate(d):
                w = host(c.w)
                E.kv8_evict(c.h, c.h, c.w.data_ptr(), c.w.data_ptr(), after.data_ptr(), length.data_ptr(), cap, keep, 2, 16, 0,
                            es.data_ptr(), es.numel(), stream())
                ref[i], _, now_left, _ = ref[i].evict(w, now, keep, 2, 16)
            now = now_left
        else:
            length.copy_(after)
        lens = now
        assert host(length).tolist() == lens
        HELD[2:] = []
    for x, c in zip(ref, d):
        c.stale_from(lens)
        c.check(x, lens)


def test_offsets_beyond_31_bits_within_a_head(gpu):
    """One head of 2.5 GiB of K and of V: rows appended, read back, attended to and moved from beyond 2^31 bytes of its start."""
    cap, hd, n = 5 * 2 ** 20, 512, 64
    code = [torch.empty((1, 1, cap, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scale = [torch.empty((1, 1, cap // 32), device="cuda") for _ in range(2)]
    w = torch.zeros((1, 1, cap), device="cuda")
    h = E.KV8Cache(E.I8, 1, 1, cap, hd, *(x.data_ptr() for x in code + scale))
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 1, n, 1, hd)).astype(np.float32)
    k, v, start, end = dev(x[0]), dev(x[1]), ints([cap - n]), ints([0])
    E.kv8_append(h, k.data_ptr(), v.data_ptr(), n, hd, start.data_ptr(), 0, end.data_ptr(), 0, stream())
    ref = kv8_ref.Cache(1, 1, n, hd, "i8")
    ref.append(x[0], x[1], [0], [n])
    to = Dev(1, 1, n, hd, "i8")
    len_out, ws = ints([0]), torch.empty(E.kv8_evict_workspace(h, cap, n), dtype=torch.uint8, device="cuda")
    E.kv8_evict(h, to.h, w.data_ptr(), to.w.data_ptr(), end.data_ptr(), len_out.data_ptr(), cap, n, 0, n, 0, ws.data_ptr(),
                ws.numel(), stream())
    assert host(end).tolist() == [cap] and host(len_out).tolist() == [n]
    to.check(ref, [n])
    out = [torch.zeros((n, hd), device="cuda") for _ in range(2)]
    E.kv8_load(h, n, hd, start.data_ptr(), 0, out[0].data_ptr(), out[1].data_ptr(), stream())
    for i in range(2):
        assert np.array_equal(host(out[i]), ref.value(i, 0, 0, n).astype(np.float32))
    q = rng.standard_normal((1, 1, 8, hd)).astype(np.float32)
    size = E.kv8_attention_workspace(h, 8, 1, cap, False)
    ws, res, dq = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros((8, hd), device="cuda"), dev(q)
    E.kv8_attention(h, dq.data_ptr(), 8, 1, 8 * hd, end.data_ptr(), cap, n, 0.04, res.data_ptr(), 0, 0, ws.data_ptr(), size, stream())
    want, _, bound = ref.attention(q, [n], 0, 0.04)
    assert (np.abs(host(res).reshape(q.shape) - want) <= bound).all()


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_attention_of_values_up_to_the_stated_limit(gpu, dtype):
    """300 entries of up to 2^110 (below 2^119 in all), the scores rising slowly from entry to entry, so that the running
    maximum is behind the largest one most of the time."""
    n, hd = 300, 64
    rng = np.random.default_rng(5)
    ref, d = kv8_ref.Cache(1, 1, n, hd, dtype), Dev(1, 1, n, hd, dtype)
    k = np.zeros((1, n, 1, hd), np.float32)
    k[0, :, 0, 0] = np.arange(n) / 8
    v = (rng.uniform(0.5, 1, (1, n, 1, hd)) * 2.0 ** 110).astype(np.float32)
    dk, dv = dev(k), dev(v)
    E.kv8_append(d.h, dk.data_ptr(), dv.data_ptr(), n, hd, 0, 0, 0, 0, stream())
    ref.append(k, v, [0], [n])
    q = np.zeros((1, 1, 8, hd), np.float32)
    q[..., 0] = np.arange(8)[None, None]
    want, _, bound = ref.attention(q, [n], 0, 0.3)
    got, _ = attend(d, q, [n], 0, 0.3)
    assert (np.abs(got - want) <= bound).all()
