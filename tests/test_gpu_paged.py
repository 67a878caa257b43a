"""The paged cache (iek_dev_paged_*) on the device against tests/paged_ref.py in 64 bits.

Bars: rows, lengths and what is left alone equal bit for bit (each rotation step is rounded to f32, an fp16 entry once);
attention within the bound on f32 errors that paged_ref derives."""
import numpy as np
import pytest

import paged_ref
from inference_engine_rust_amd import engine as E

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": (E.F32, torch.float32), "f16": (E.F16, torch.float16)}
HELD = []  # small arrays given by address only: alive until their test ends


@pytest.fixture(autouse=True)
def _let_go():
    yield
    HELD.clear()


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a)).to("cuda")


def ints(x):
    HELD.append(dev(np.asarray(x, np.int32)))
    return HELD[-1]


def stream():
    return torch.cuda.current_stream().cuda_stream


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


class Dev:
    """The pools on the device: those of a reference (NaN where it has nothing), its table, and their descriptor."""

    def __init__(self, ref):
        self.pool = [dev(x.astype(np.float32)).to(DT[ref.dtype][1]) for x in (ref.k, ref.v)]
        self.table = dev(ref.table.astype(np.int32))
        self.h = E.PagedKV(DT[ref.dtype][0], ref.n_pages, ref.kv, ref.page, ref.hd, self.pool[0].data_ptr(), self.pool[1].data_ptr(),
                           len(ref.table), ref.table.shape[1], self.table.data_ptr())

    def check(self, ref):
        for got, want in zip(self.pool, (ref.k, ref.v)):
            assert np.array_equal(host(got.float()), want.astype(np.float32), equal_nan=True)


def tables(rng, lens, page, max_pages, n_pages, common=0):
    """Page numbers in no order, the first `common` the same for all; behind a sequence's last page numbers that are none."""
    order = rng.permutation(n_pages)
    t = rng.choice([-1, -2 ** 31, n_pages, 2 ** 31 - 1], (len(lens), max_pages)).astype(np.int64)
    at = common
    for b, n in enumerate(lens):
        need = -(-n // page)
        t[b, :min(need, common)] = order[:min(need, common)]
        own = max(0, need - common)
        t[b, common:common + own] = order[at:at + own]
        at += own
    return t, order[:common]


def filled(seed, dtype, kv, hd, page, lens, max_pages=None, common=0):
    """A reference cache with the lengths' entries in place, and the pages that all sequences begin with."""
    rng = np.random.default_rng(seed)
    n_pages = common + sum(max(0, -(-n // page) - common) for n in lens) + 3
    max_pages = max_pages or max(1, max(-(-n // page) for n in lens)) + 1
    t, shared = tables(rng, lens, page, max_pages, n_pages, common)
    ref = paged_ref.Paged(n_pages, kv, page, hd, t, dtype)
    live = np.zeros((n_pages, page), bool)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            live[t[b, i], :n - i * page] = True
    size = np.exp2(rng.integers(-3, 3, (n_pages, kv, page, 1)))
    for x in (ref.k, ref.v):
        x[:] = np.where(live[:, None, :, None], ref.hold(rng.standard_normal(x.shape) * size), np.nan)
    return ref, shared


# ---- append ----

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd,rotary,page", [(1, 1, 64, 64, 16), (6, 3, 64, 2, 32), (32, 8, 128, 128, 64), (8, 2, 256, 64, 16),
                                                     (8, 1, 512, 512, 256), (0, 2, 128, 128, 16), (0, 1, 64, 0, 1024), (5, 5, 128, 66, 128)])
def test_append_matches_and_leaves_the_rest(gpu, dtype, heads, kv, hd, rotary, page):
    rng = np.random.default_rng(heads * hd)
    n, pages = 70, -(-133 // page)
    cap = pages * page
    start, count = [0, 5, 31, 64, cap - 7, cap, -1, cap + 1, 2 ** 31 - 1, 3], [70, 33, 1, 0, 20, 9, 9, 9, 9, -4]
    batch = len(start)
    n_pages = batch * pages + 2
    table = rng.permutation(n_pages)[:batch * pages].reshape(batch, pages).astype(np.int64)
    ref = paged_ref.Paged(n_pages, kv, page, hd, table, dtype)
    d = Dev(ref)
    pad = 8
    stride = (heads + 2 * kv) * hd + pad
    fused = (rng.standard_normal((batch, n, stride)) * np.exp2(rng.integers(-3, 5, (batch, n, 1)))).astype(np.float32)
    rope = rng.uniform(-1, 1, (cap + 3, rotary // 2, 2)).astype(np.float32)
    x, table_dev = dev(fused), dev(rope)
    q_out, q_stride = torch.full((batch, n, heads * hd + 4), -3.0, device="cuda"), heads * hd + 4
    len_out = ints([-7] * batch)
    base = x.data_ptr()
    E.paged_append(d.h, base if heads else 0, base + 4 * heads * hd, base + 4 * (heads + kv) * hd, heads, n, stride,
                   table_dev.data_ptr() if rotary else 0, cap + 3 if rotary else 0, rotary, ints(start).data_ptr(), ints(count).data_ptr(),
                   len_out.data_ptr(), q_out.data_ptr() if heads else 0, q_stride if heads else 0, stream())
    rows = fused[..., :stride - pad].reshape(batch, n, heads + 2 * kv, hd)
    at = np.clip(np.asarray(start)[:, None] + np.arange(n), 0, cap - 1)
    turned = paged_ref.rotated(rows[:, :, :heads + kv], rope[at]) if rotary else rows[:, :, :heads + kv]
    want = ref.append(turned[:, :, heads:], rows[:, :, heads + kv:], start, count)
    assert host(len_out).tolist() == want == [70, 38, 32, 64, cap, cap, 0, cap, cap, 3]
    d.check(ref)
    got = host(q_out)
    for b in range(batch):
        c = want[b] - min(max(start[b], 0), cap)
        assert np.array_equal(got[b, :c, :heads * hd], turned[b, :c, :heads].reshape(c, heads * hd))
        assert (got[b, c:] == -3).all() and (got[b, :, heads * hd:] == -3).all()


@pytest.mark.parametrize("n", [1, 3])
def test_append_in_place(gpu, n):
    """Queries over themselves, lengths over the starts; rows that all starts and counts are left out of."""
    rng = np.random.default_rng(n)
    heads, kv, hd, batch, page = 8, 2, 64, 70, 16
    table = rng.permutation(batch * 4).reshape(batch, 4).astype(np.int64)
    ref = paged_ref.Paged(batch * 4, kv, page, hd, table, "f32")
    d, stride = Dev(ref), (heads + 2 * kv) * hd
    start = [int(s) for s in rng.integers(-2, 70, batch)]
    rows = rng.standard_normal((batch, n, heads + 2 * kv, hd)).astype(np.float32)
    rope = E.rope_table(hd, hd, 10000.0, 64)
    x, table_dev, lens = dev(rows), dev(rope), ints(start)
    p = x.data_ptr()
    E.paged_append(d.h, p, p + 4 * heads * hd, p + 4 * (heads + kv) * hd, heads, n, stride, table_dev.data_ptr(), 64, hd, lens.data_ptr(),
                   0, lens.data_ptr(), p, stride, stream())
    turned = paged_ref.rotated(rows[:, :, :heads + kv], rope[np.clip(np.asarray(start)[:, None] + np.arange(n), 0, 63)])
    want = ref.append(turned[:, :, heads:], rows[:, :, heads + kv:], start, [n] * batch)
    assert host(lens).tolist() == want
    d.check(ref)
    got = host(x)
    for b in range(batch):
        c = want[b] - min(max(start[b], 0), 64)
        assert np.array_equal(got[b, :c, :heads], turned[b, :c, :heads]) and np.array_equal(got[b, c:], rows[b, c:])
        assert np.array_equal(got[b, :, heads:], rows[b, :, heads:])
    # and from the beginning, all of them
    E.paged_append(d.h, 0, p, p, 0, n, stride, 0, 0, 0, 0, 0, 0, 0, 0, stream())
    got = host(x)[:, :, :kv].astype(np.float64)
    for b in range(batch):
        assert np.array_equal(host(d.pool[0])[table[b, 0], :, :n], got[b].transpose(1, 0, 2))


def test_append_rotates_as_the_rope_op_does(gpu):
    rng = np.random.default_rng(0)
    hd, rotary, ff = 128, 96, rng.uniform(0.5, 4, 48).astype(np.float32)
    ref = paged_ref.Paged(8, 1, 16, hd, np.arange(8)[None], "f32")
    d = Dev(ref)
    x = rng.standard_normal((1, 100, 3, hd)).astype(np.float32)
    rope, q = dev(E.rope_table(hd, rotary, 1e4, 128, ff)), torch.zeros((100, hd), device="cuda")
    t = dev(x)
    E.paged_append(d.h, t.data_ptr(), t.data_ptr() + 4 * hd, t.data_ptr() + 8 * hd, 1, 100, 3 * hd, rope.data_ptr(), 128, rotary, 0, 0, 0,
                   q.data_ptr(), hd, stream())
    k = host(d.pool[0])[:, 0].reshape(128, hd)
    for pos in (0, 1, 17, 99):
        want = E.host_rope(x[0, pos, :2].copy(), 2, hd, rotary, 1e4, pos, ff)
        assert np.array_equal(host(q)[pos], want.reshape(2, hd)[0]) and np.array_equal(k[pos], want.reshape(2, hd)[1])


def test_append_of_values_at_fp16s_ends(gpu):
    vals = np.float32([0, -0.0, 1e-9, 2.0 ** -25, 2.0 ** -24, 3 * 2.0 ** -25, 6e-5, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 65504, 65519.9, 65520,
                       -1e9, np.inf, -np.inf, np.nan])
    ref = paged_ref.Paged(1, 1, 16, 64, np.zeros((1, 1)), "f16")
    d, x = Dev(ref), np.tile(vals, (1, 16, 1, 4)).astype(np.float32)
    t = dev(x)
    E.paged_append(d.h, 0, t.data_ptr(), t.data_ptr(), 0, 16, 64, 0, 0, 0, 0, 0, 0, 0, 0, stream())
    ref.append(x, x, [0], [16])
    d.check(ref)


def test_append_without_pages(gpu):
    """Rows whose page is none are dropped, the others of the sequence and its length are as ever."""
    rng = np.random.default_rng(2)
    table = np.asarray([[3, -1, 0, 7, 1], [7, 2 ** 31 - 1, -2 ** 31, 5, 4]])
    ref = paged_ref.Paged(7, 2, 16, 64, table, "f16")
    d, x = Dev(ref), rng.standard_normal((2, 80, 2, 64)).astype(np.float32)
    t, lens = dev(x), ints([0, 0])
    q, rope = torch.zeros((2, 80, 128), device="cuda"), dev(E.rope_table(64, 64, 1e4, 80))
    E.paged_append(d.h, t.data_ptr(), t.data_ptr(), t.data_ptr(), 2, 80, 128, rope.data_ptr(), 80, 64, 0, 0, lens.data_ptr(), q.data_ptr(),
                   128, stream())
    turned = paged_ref.rotated(x, host(rope)[None])
    assert ref.append(turned, x, [0, 0], [80, 80]) == host(lens).tolist() == [80, 80]
    d.check(ref)
    assert np.array_equal(host(q).reshape(x.shape), turned)


# ---- attention ----

def attend(d, q, lens, window, scale, shared=0, pages=(), max_shared=None, max_len=None, q_pad=0):
    batch, n_q, heads, hd = q.shape
    rows = dev(np.concatenate([q.reshape(batch, n_q, -1), np.zeros((batch, n_q, q_pad), np.float32)], 2))
    max_len = max(lens) if max_len is None else max_len
    max_shared = shared if max_shared is None else max_shared
    size = E.paged_attention_workspace(d.h, heads, n_q, max_len, max_shared)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")  # NaN to whoever reads it unwritten
    out = torch.full(q.shape, 77.0, device="cuda")
    p, n = (ints(pages).data_ptr(), ints([shared]).data_ptr()) if max_shared else (0, 0)
    E.paged_attention(d.h, rows.data_ptr(), heads, n_q, heads * hd + q_pad, ints(lens).data_ptr(), max_len, p, n, max_shared, window, scale,
                      out.data_ptr(), ws.data_ptr(), size, stream())
    return host(out)


def queries(rng, batch, n_q, heads, hd):
    return (rng.standard_normal((batch, n_q, heads, hd)) * np.exp2(rng.integers(-4, 2, (batch, n_q, heads, 1)))).astype(np.float32)


def check(got, want, bound):
    worst = np.max(np.abs(got - want) - bound)
    assert worst <= 0, (worst, np.argwhere(~(np.abs(got - want) <= bound))[:5])


def check_attention(seed, dtype, kv, group, hd, n_q, lens, window=0, page=16, shared=0, max_len=None, max_shared=None, q_pad=0):
    rng = np.random.default_rng(seed)
    common = -(-shared // page)
    # (a page that the shared part ends in is the shared one for all here: sequences go on in it, the same entries)
    ref, pages = filled(seed, dtype, kv, hd, page, lens, common=common)
    d = Dev(ref)
    q, scale = queries(rng, len(lens), n_q, kv * group, hd), 1 / np.sqrt(hd)
    want, bound = ref.attention(q, lens, window, scale, shared, pages)
    check(attend(d, q, lens, window, scale, shared, pages, max_shared, max_len, q_pad), want, bound)


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 95, 127, 128, 129, 257, 531]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 16), (256, 64), (512, 32)])
@pytest.mark.parametrize("kv,group", [(1, 8), (2, 4), (3, 1)])
def test_attention_one_token(gpu, dtype, hd, page, kv, group):
    check_attention(hd + group, dtype, kv, group, hd, 1, LENS, page=page, q_pad=8)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", [0, 1, 16, 31, 130, 700])
@pytest.mark.parametrize("hd", [64, 128, 512])
def test_attention_one_sequence(gpu, dtype, hd, n):
    check_attention(n, dtype, 2, 3, hd, 1, [n], page=32)


@pytest.mark.parametrize("dtype,window", [("f32", 0), ("f16", 40), ("f16", 0), ("f32", 33)])
@pytest.mark.parametrize("hd,kv,group,n_q", [(64, 2, 4, 5), (128, 1, 3, 7), (128, 2, 8, 2), (128, 1, 8, 33), (256, 1, 5, 3),
                                             (256, 1, 8, 9), (512, 1, 8, 4), (64, 1, 1, 64), (64, 2, 8, 64)])
def test_attention_several_tokens(gpu, dtype, window, hd, kv, group, n_q):
    check_attention(n_q, dtype, kv, group, hd, n_q, [0, 1, n_q - 1, n_q, 40, 300], window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 31, 33, 512, 513])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_window(gpu, dtype, window, hd):
    check_attention(window, dtype, 1, 8, hd, 1, [1, 33, 511, 512, 513, 1000, 4099], window, page=128)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_attention_long(gpu, dtype, page):
    check_attention(5, dtype, 2, 4, 128, 1, [20011, 9000], page=page)


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
@pytest.mark.parametrize("hd,kv,group,n_q,window,shared", [(64, 1, 8, 1, 0, 0), (64, 2, 8, 3, 0, 100), (128, 1, 2, 1, 300, 250)])
def test_attention_many_sequences(gpu, batch, hd, kv, group, n_q, window, shared):
    lens = [(37 * i * i + 5) % 1200 if i % 7 else 0 for i in range(batch)]
    check_attention(batch, "f16" if batch % 2 else "f32", kv, group, hd, n_q, lens, window, shared=shared)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shared", [1, 15, 16, 17, 32, 100, 128, 531, 700])
@pytest.mark.parametrize("kv,group,hd,n_q", [(2, 4, 64, 1), (1, 8, 128, 1), (2, 1, 128, 3), (1, 8, 256, 1), (1, 5, 512, 2)])
def test_attention_shared(gpu, dtype, shared, kv, group, hd, n_q):
    """Shared parts that end anywhere in a tile and a page, sequences shorter than them and empty ones among the batch."""
    check_attention(shared, dtype, kv, group, hd, n_q, [shared, shared + 1, 0, shared + 40, 5, shared + 333], page=32, shared=shared)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 100, 512])
@pytest.mark.parametrize("n_q", [1, 4])
def test_attention_shared_with_a_window(gpu, dtype, window, n_q):
    check_attention(window, dtype, 1, 8, 128, n_q, [600, 601, 0, 640, 1000, 1300, 700, 650, 3], window, shared=600)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("batch,heads,kv,hd", [(1, 8, 2, 64), (3, 8, 2, 64), (40, 32, 8, 128), (70, 8, 1, 256), (17, 8, 1, 512)])
def test_attention_shared_long(gpu, dtype, batch, heads, kv, hd):
    check_attention(batch, dtype, kv, heads // kv, hd, 1, [2501 + 13 * i % 200 for i in range(batch)], page=64, shared=2499)


def test_attention_shared_less_than_sized_for(gpu):
    """*shared below max_shared (0 too), above it, and negative: the words on the device decide."""
    ref, pages = filled(3, "f16", 2, 64, 16, [400, 500, 300], common=12)
    d, rng = Dev(ref), np.random.default_rng(3)
    q = queries(rng, 3, 1, 8, 64)
    want, bound = ref.attention(q, [400, 500, 300], 0, 0.125)
    for shared in (0, 5, 64, 192, 1000, -3):
        check(attend(d, q, [400, 500, 300], 0, 0.125, shared, pages, max_shared=192, max_len=500), want, bound)


def test_shared_entries_are_read_from_their_own_list(gpu):
    """Whatever the tables say of them: none, or other pages."""
    ref, pages = filled(4, "f32", 1, 128, 16, [100, 90], common=4)
    q = queries(np.random.default_rng(0), 2, 1, 4, 128)
    want, bound = ref.attention(q, [100, 90], 0, 0.1, 50, pages)
    ref.table[0, :3], ref.table[1, :3] = -1, ref.table[0, 5]
    check(attend(Dev(ref), q, [100, 90], 0, 0.1, 50, pages), want, bound)


def test_attention_max_len_beyond_and_below_the_lengths(gpu):
    check_attention(6, "f32", 2, 4, 128, 1, [40, 60], max_len=72)
    ref, _ = filled(7, "f16", 1, 64, 16, [200, 200])
    d, q = Dev(ref), queries(np.random.default_rng(1), 2, 1, 4, 64)
    want, bound = ref.attention(q, [90, 0], 0, 0.125)
    check(attend(d, q, [200, -3], 0, 0.125, max_len=90), want, bound)  # lengths above max_len count as max_len
    assert (attend(d, q, [200, 200], 0, 0.125, max_len=0) == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 32])
def test_attention_over_missing_pages(gpu, dtype, page):
    """Entries whose page is none are not seen: in the middle, at the end, all of a sequence's, of the shared list."""
    lens = [300, 300, 300, 40]
    for shared in (0, 64):
        ref, pages = filled(8, dtype, 2, 64, page, lens, common=shared // page)
        ref.table[0, 5], ref.table[0, 7], ref.table[1, -(-300 // page) - 1] = -1, ref.n_pages, 2 ** 31 - 1
        ref.table[2, shared // page:] = -5
        if shared:
            pages = pages.copy()
            pages[1] = ref.n_pages
        q = queries(np.random.default_rng(9), 4, 3, 8, 64)
        want, bound = ref.attention(q, lens, 0, 0.125, shared, pages)
        check(attend(Dev(ref), q, lens, 0, 0.125, shared, pages), want, bound)


BAD = [np.nan, np.inf, -np.inf]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("kv,group,hd,n_q,shared,window", [(1, 4, 64, 3, 0, 0), (2, 8, 128, 5, 0, 50), (1, 2, 256, 2, 0, 0), (1, 8, 512, 3, 0, 20),
                                                           (2, 4, 128, 1, 70, 0), (1, 8, 64, 2, 70, 33)])
def test_queries_that_do_not_see_a_bad_entry_take_nothing_of_it(gpu, kv, group, hd, n_q, shared, window, which, dtype):
    """A NaN or infinity in an entry: the queries that see it are not finite where the formula is not, the others as ever."""
    rng = np.random.default_rng(hd)
    lens = [90, 75, 71, 30, 200]
    for at, bad in ((89, np.nan), (70, np.inf), (74, -np.inf), (60, np.nan), (29, np.inf), (0, -np.inf)):
        ref, pages = filled(1, dtype, kv, hd, 16, lens, common=-(-shared // 16))
        q = queries(rng, len(lens), n_q, kv * group, hd)
        want, bound = ref.attention(q, lens, window, 0.01, shared, pages)
        b, dim = 0, 5
        page = pages[at // 16] if at < shared else ref.table[b, at // 16]
        (ref.k if which == "k" else ref.v)[page, kv - 1, at % 16, dim] = bad
        poisoned, _ = ref.attention(q, lens, window, 0.01, shared, pages)
        d = Dev(ref)
        got = attend(d, q, lens, window, 0.01, shared, pages)
        same = poisoned == want
        ends = [n - i for n in (lens if at < shared else lens[:1]) for i in range(n_q)]
        assert same.any() and same.all() == (not any((hi - window if window else 0) <= at < hi for hi in ends))
        assert (np.abs(got - want) <= bound)[same].all(), (at, np.argwhere(same & ~(np.abs(got - want) <= bound))[:4])
        if which == "v":
            # NaN or an infinity. (Which one cannot be told in fp16 pages: a weight is a pair hi + lo there, and with
            # lo <= 0 an infinity times it is inf - inf or inf * 0.)
            assert (np.isfinite(got) == np.isfinite(poisoned)).all()
        else:  # a score of NaN or +inf: NaN; of -inf: no weight (or +inf, by the query's sign)
            bad_rows = np.isnan(poisoned).all(-1)
            assert np.isnan(got[bad_rows]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_sizes_of_values(gpu, dtype):
    """Scores spread over hundreds, values over the type's whole range: the weights and the sums keep 32 bits."""
    rng = np.random.default_rng(4)
    ref, _ = filled(4, dtype, 2, 128, 16, [400, 333])
    ref.k *= 4
    small, big = (2.0 ** -20, 2.0 ** 10) if dtype == "f16" else (2.0 ** -100, 2.0 ** 100)
    for h, f in ((0, small), (1, big)):
        ref.v[:, h] = ref.hold(ref.v[:, h] * f)
    q = (queries(rng, 2, 1, 8, 128) * np.float32([2.0 ** e for e in (-30, -8, 0, 3, 4, 0, -20, 2)])[:, None]).astype(np.float32)
    want, bound = ref.attention(q, [400, 333], 0, 0.2)
    check(attend(Dev(ref), q, [400, 333], 0, 0.2), want, bound + 1e-300)


def test_one_large_weight_over_many_small_equal_ones(gpu):
    """fp16 pages: what thousands of equal shares far below the largest lose at fp16's lower end stays within the bound."""
    n = 16000
    ref, _ = filled(5, "f16", 1, 64, 64, [n])
    for x in (ref.k, ref.v):
        x[~np.isnan(x)] = 0
    ref.v[~np.isnan(ref.v)] = 1
    q = np.zeros((1, 1, 1, 64), np.float32)
    q[..., 0] = 1
    p0 = ref.table[0, 0]
    ref.k[p0, 0, 3, 0], ref.v[p0, 0, 3] = 18, 0
    want, bound = ref.attention(q, [n], 0, 1.0)
    assert 1e-4 < want[0, 0, 0, 0] < 1e-3
    check(attend(Dev(ref), q, [n], 0, 1.0), want, bound)


# ---- together ----

def test_a_decode_loop_with_a_shared_prompt(gpu):
    """A batch behind a common prompt: its entries appended once, then step by step one token a sequence: append, attention,
    a projection to logits, sampling. Every step against the 64-bit reference."""
    rng = np.random.default_rng(11)
    heads, kv, hd, batch, page, vocab, steps, prompt = 8, 2, 64, 5, 16, 300, 21, 37
    max_pages = 8
    t = np.full((batch, max_pages), -1, np.int64)
    free = list(rng.permutation(60))
    common = [int(free.pop()) for _ in range(prompt // page)]  # whole pages; the rest of the prompt is each one's own
    for b in range(batch):
        t[b, :len(common)] = common
        t[b, len(common):] = [free.pop() for _ in range(max_pages - len(common))]
    ref = paged_ref.Paged(60, kv, page, hd, t, "f16")
    d = Dev(ref)
    shared = len(common) * page
    rope_host = E.rope_table(hd, hd, 10000.0, max_pages * page)
    rope, width = dev(rope_host), (heads + 2 * kv) * hd
    rows = rng.standard_normal((batch, prompt, heads + 2 * kv, hd)).astype(np.float32)
    rows[1:, :shared] = rows[0, :shared]
    x, q_out = dev(rows), torch.zeros((batch, prompt, heads * hd), device="cuda")
    lens = ints([0] * batch)

    def put(x, n, start):
        p = x.data_ptr()
        E.paged_append(d.h, p, p + 4 * heads * hd, p + 4 * (heads + kv) * hd, heads, n, width, rope.data_ptr(), max_pages * page, hd,
                       start, 0, lens.data_ptr(), q_out.data_ptr(), heads * hd, stream())

    put(x, prompt, lens.data_ptr())
    turned = paged_ref.rotated(rows[:, :, :heads + kv], rope_host[None, :prompt])
    at = ref.append(turned[:, :, heads:], rows[:, :, heads + kv:], [0] * batch, [prompt] * batch)
    d.check(ref)
    head = rng.standard_normal((vocab, heads * hd)).astype(np.float32) * 0.3
    head_dev = dev(head)
    table = rng.standard_normal((vocab, width)).astype(np.float32)  # a token's next row
    out, logits = torch.zeros((batch, heads * hd), device="cuda"), torch.zeros((batch, vocab), device="cuda")
    opts = dict(t=[0.0, 0.7, 1.0, 1.3, 0.9], k=[0, 5, 0, 40, 300], p=[1.0, 0.9, 0.8, 1.0, 0.95], m=[0.0, 0.0, 0.05, 0.1, 0.0])
    par = {n: dev(np.asarray(v, np.int32 if n == "k" else np.float32)) for n, v in opts.items()}
    index, prob = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros(batch, device="cuda")
    ws = torch.empty(E.paged_attention_workspace(d.h, heads, 1, max_pages * page, shared) + E.sample_workspace(batch, vocab) + 16,
                     dtype=torch.uint8, device="cuda")
    shared_pages, shared_len = ints(common), ints([shared])
    tokens = list(range(batch))
    for step in range(steps):
        rows = table[tokens].reshape(batch, 1, heads + 2 * kv, hd)
        put(dev(rows), 1, lens.data_ptr())
        q = paged_ref.rotated(rows[:, :, :heads], rope_host[at][:, None])
        k = paged_ref.rotated(rows[:, :, heads:heads + kv], rope_host[at][:, None])
        at = ref.append(k, rows[:, :, heads + kv:], at, [1] * batch)
        E.paged_attention(d.h, q_out.data_ptr(), heads, 1, heads * hd, lens.data_ptr(), max_pages * page, shared_pages.data_ptr(),
                          shared_len.data_ptr(), shared, 0, 0.125, out.data_ptr(), ws.data_ptr(), ws.numel(), stream())
        want, bound = ref.attention(q, at, 0, 0.125, shared, common)
        check(host(out).reshape(batch, 1, heads, hd), want, bound)
        torch.matmul(out, head_dev.t(), out=logits)
        r = rng.random(batch).astype(np.float32)
        r_dev = dev(r)
        E.sample(logits.data_ptr(), batch, vocab, vocab, par["t"].data_ptr(), par["k"].data_ptr(), par["p"].data_ptr(), par["m"].data_ptr(),
                 r_dev.data_ptr(), index.data_ptr(), prob.data_ptr(), ws.data_ptr(), ws.numel(), stream())
        rows_of = host(logits)
        picks = [paged_ref.sample(rows_of[b], opts["t"][b], r[b], opts["k"][b], opts["p"][b], opts["m"][b]) for b in range(batch)]
        tokens = host(index).tolist()
        assert tokens == [i for i, _ in picks]
        assert np.abs(host(prob) / [p for _, p in picks] - 1).max() < 2.0 ** -23
    assert host(lens).tolist() == at == [prompt + steps] * batch
    d.check(ref)


def captured(body):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body(torch.cuda.current_stream().cuda_stream)
    return g


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_captured_step_replays(gpu, dtype):
    """Append, attention over a shared part, sampling, captured once: lengths, pages, shared part and draws from the device."""
    rng = np.random.default_rng(1)
    heads, kv, hd, batch, page, max_pages = 8, 2, 128, 3, 16, 40
    n_pages = 130
    ref = paged_ref.Paged(n_pages, kv, page, hd, np.full((batch, max_pages), -1), dtype)
    d = Dev(ref)
    width = (heads + 2 * kv) * hd
    rope_host = E.rope_table(hd, hd, 10000.0, max_pages * page)
    rope, x, q_out = dev(rope_host), torch.zeros((batch, 1, width), device="cuda"), torch.zeros((batch, heads * hd), device="cuda")
    start, lens, shared = ints([0] * batch), ints([0] * batch), ints([0])
    pages = ints([0] * max_pages)
    out = torch.zeros((batch, heads * hd), device="cuda")
    index, t, r = torch.zeros(batch, dtype=torch.int32, device="cuda"), dev(np.float32([0.8] * batch)), dev(np.float32([0.5] * batch))
    size = E.paged_attention_workspace(d.h, heads, 1, max_pages * page, max_pages * page)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    ss = torch.full((E.sample_workspace(batch, heads * hd) + 16,), 255, dtype=torch.uint8, device="cuda")

    def step(st):
        p = x.data_ptr()
        E.paged_append(d.h, p, p + 4 * heads * hd, p + 4 * (heads + kv) * hd, heads, 1, width, rope.data_ptr(), max_pages * page, hd,
                       start.data_ptr(), 0, lens.data_ptr(), q_out.data_ptr(), heads * hd, st)
        E.paged_attention(d.h, q_out.data_ptr(), heads, 1, heads * hd, lens.data_ptr(), max_pages * page, pages.data_ptr(), shared.data_ptr(),
                          max_pages * page, 0, 0.1, out.data_ptr(), ws.data_ptr(), size, st)
        E.sample(out.data_ptr(), batch, heads * hd, heads * hd, t.data_ptr(), 0, 0, 0, r.data_ptr(), index.data_ptr(), 0, ss.data_ptr(),
                 ss.numel(), st)

    g = captured(step)
    for turn, (at, common) in enumerate([([0, 0, 0], 0), ([5, 300, 599], 0), ([200, 177, 310], 160), ([639, 640, 2], 0), ([32, 16, 600], 16)]):
        ref2, sp = filled(turn, dtype, kv, hd, page, at, max_pages=max_pages, common=common // page)
        ref.k[:], ref.v[:] = np.nan, np.nan
        ref.k[:ref2.n_pages], ref.v[:ref2.n_pages], ref.table = ref2.k, ref2.v, ref2.table
        spare = iter(range(ref2.n_pages, n_pages))
        for b in range(batch):  # a page for the new row
            if at[b] < max_pages * page and at[b] % page == 0:
                ref.table[b, at[b] // page] = next(spare)
        for pool, have in zip(d.pool, (ref.k, ref.v)):
            pool.copy_(dev(have.astype(np.float32)))
        d.table.copy_(dev(ref.table.astype(np.int32)))
        rows, draws = rng.standard_normal((batch, 1, heads + 2 * kv, hd)).astype(np.float32), rng.random(batch).astype(np.float32)
        x.copy_(dev(rows.reshape(batch, 1, width)))
        r.copy_(dev(draws))
        start.copy_(ints(at))
        shared.copy_(ints([common]))
        if common:
            pages[:len(sp)] = ints(sp)
        g.replay()
        torch.cuda.synchronize()
        turned = paged_ref.rotated(rows[:, :, :heads + kv], rope_host[np.minimum(at, max_pages * page - 1)][:, None])
        after = ref.append(turned[:, :, heads:], rows[:, :, heads + kv:], at, [1] * batch)
        assert host(lens).tolist() == after
        d.check(ref)
        q = host(q_out).reshape(batch, 1, heads, hd)
        want, bound = ref.attention(q, after, 0, 0.1, common, sp)
        check(host(out).reshape(want.shape), want, bound)
        logits = host(out)
        assert host(index).tolist() == [paged_ref.sample(logits[b], 0.8, draws[b])[0] for b in range(batch)]


def test_two_streams_at_once(gpu):
    lens = [[700, 33, 2000], [1500, 0, 64]]
    cases = [filled(i, "f16", 2, 128, 32, lens[i], common=1) for i in range(2)]
    devs = [Dev(ref) for ref, _ in cases]
    q = [queries(np.random.default_rng(i), 3, 1, 8, 128) for i in range(2)]
    want = [ref.attention(q[i], lens[i], 0, 0.1, 32, p) for i, (ref, p) in enumerate(cases)]
    qd, ld, pd, sd = [dev(x) for x in q], [ints(x) for x in lens], [ints(p) for _, p in cases], ints([32])
    size = [E.paged_attention_workspace(devs[i].h, 8, 1, max(lens[i]), 32) for i in range(2)]
    ws = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in size]
    out = [torch.zeros(q[0].shape, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            E.paged_attention(devs[i].h, qd[i].data_ptr(), 8, 1, 8 * 128, ld[i].data_ptr(), max(lens[i]), pd[i].data_ptr(), sd.data_ptr(), 32,
                              0, 0.1, out[i].data_ptr(), ws[i].data_ptr(), size[i], s.cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        check(host(out[i]), *want[i])


def test_attention_repeats_bit_for_bit(gpu):
    ref, p = filled(2, "f16", 2, 128, 16, [900, 450, 1300, 333], common=20)
    d, q = Dev(ref), queries(np.random.default_rng(5), 4, 2, 8, 128)
    first = attend(d, q, [900, 450, 1300, 333], 0, 0.1, 320, p)
    for _ in range(3):
        assert np.array_equal(attend(d, q, [900, 450, 1300, 333], 0, 0.1, 320, p), first)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_offsets_beyond_32_bits(gpu, dtype):
    """A pool of more than 2^32 bytes: the last pages hold the rows."""
    kv, hd, page = 8, 128, 1024
    size = 2 if dtype == "f16" else 4
    n_pages = 2 ** 32 // (kv * hd * page * size) + 3
    last = [n_pages - 1, n_pages - 2]
    pool = [torch.zeros((n_pages, kv, page, hd), dtype=DT[dtype][1], device="cuda") for _ in range(2)]
    table = ints([last])
    h = E.PagedKV(DT[dtype][0], n_pages, kv, page, hd, pool[0].data_ptr(), pool[1].data_ptr(), 1, 2, table.data_ptr())
    rng = np.random.default_rng(0)
    n, start = 100, 1000
    rows = rng.standard_normal((1, n, 2 * kv, hd)).astype(np.float32)
    x = dev(rows)
    E.paged_append(h, 0, x.data_ptr(), x.data_ptr() + 4 * kv * hd, 0, n, 2 * kv * hd, 0, 0, 0, ints([start]).data_ptr(), 0, 0, 0, 0, stream())
    ref = paged_ref.Paged(2, kv, page, hd, [[0, 1]], dtype)
    ref.k[:], ref.v[:] = 0, 0
    ref.append(rows[:, :, :kv], rows[:, :, kv:], [start], [n])
    for got, want in zip(pool, (ref.k, ref.v)):
        for i, p in enumerate(last):
            assert np.array_equal(host(got[p].float()), want[i].astype(np.float32))
        assert not torch.any(got[:n_pages - 2]).item()
    q = queries(rng, 1, 1, 32, hd)
    qd, out = dev(q), torch.zeros(q.shape, device="cuda")
    need = E.paged_attention_workspace(h, 32, 1, 2048, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    E.paged_attention(h, qd.data_ptr(), 32, 1, 32 * hd, ints([start + n]).data_ptr(), 2048, 0, 0, 0, 0, 0.1, out.data_ptr(), ws.data_ptr(), need,
                      stream())
    check(host(out), *ref.attention(q, [start + n], 0, 0.1))
