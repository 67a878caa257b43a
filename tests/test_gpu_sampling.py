"""Sampling with temperature, top-k, top-p and min-p (iek_dev_sample, iek_sample, iek_session_sample) against
tests/paged_ref.py in 64 bits.

Bars: tokens equal (draws and limits within 2^-40 of a border do not come up in these inputs, and would be another
token's by right); probabilities within an f32 rounding, 2^-24, and the total's own 2^-44 (and below f32's normal range, a share of
1e-226 say, within f32's smallest step, 2^-149)."""
import numpy as np
import pytest

import paged_ref
from inference_engine_rust_amd import engine as E

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NONE = 0xFFFFFFFF


def dev(a, dtype):
    return torch.as_tensor(np.ascontiguousarray(a, dtype)).to("cuda")


def run(x, t, r, k=None, p=None, m=None, pad=0, fill=np.nan, prob=True, stream=None):
    """(tokens, probabilities) of the rows of x, the parameters as arrays."""
    rows, n = x.shape
    held = np.full((rows, n + pad), fill, np.float32)
    held[:, :n] = x
    logits, td, rd = dev(held, np.float32), dev(t, np.float32), dev(r, np.float32)
    kd, pd, md = (None if a is None else dev(a, b) for a, b in ((k, np.int32), (p, np.float32), (m, np.float32)))
    index, out = torch.full((rows,), -5, dtype=torch.int32, device="cuda"), torch.full((rows,), -5.0, device="cuda")
    ws = torch.full((E.sample_workspace(rows, n) + 16,), 255, dtype=torch.uint8, device="cuda")
    at = [0 if a is None else a.data_ptr() for a in (kd, pd, md)]
    E.sample(logits.data_ptr(), rows, n, n + pad, td.data_ptr(), *at, rd.data_ptr(), index.data_ptr(), out.data_ptr() if prob else 0,
             ws.data_ptr(), ws.numel(), stream or torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return index.cpu().numpy().view(np.uint32), out.cpu().numpy()


def check(x, t, r, k=None, p=None, m=None, pad=0):
    rows = len(x)
    got, prob = run(x, t, r, k, p, m, pad)
    for b in range(rows):
        want, share = paged_ref.sample(x[b], t[b], r[b], 0 if k is None else int(k[b]), 1.0 if p is None else p[b], 0.0 if m is None else m[b])
        assert got[b] == want, (b, got[b], want, prob[b], share)
        assert np.isnan(prob[b]) if np.isnan(share) else abs(prob[b] - share) <= 2.0 ** -23 * share + 2.0 ** -149, (b, prob[b], share)


def rows_of(rng, rows, n, kind):
    x = rng.standard_normal((rows, n)).astype(np.float32) * 2.5
    if kind == "peaked":
        x += 7 * np.maximum(rng.standard_normal((rows, n)) - 2.5, 0)
    elif kind == "ties":  # a few values, so that borders fall among equal logits
        x = np.round(x)
    elif kind == "half":
        x = x.astype(np.float16).astype(np.float32)
    elif kind == "equal":
        x[:] = -3.25
    elif kind == "banned":
        x[rng.random(x.shape) < 0.7] = -np.inf
        x[:, 0] = 1
    elif kind == "wide":  # weights from 1 down to nothing, logits of both signs and of every size
        x *= np.exp2(rng.integers(-30, 7, (rows, n)))
    elif kind == "far":  # all of them within a few steps of a large value
        x = np.float32(12345.0) + np.float32(2.0 ** -10) * rng.integers(-9, 9, (rows, n)).astype(np.float32)
    return x.astype(np.float32)


KINDS = ["peaked", "plain", "ties", "half", "equal", "banned", "wide", "far"]
SIZES = [1, 2, 63, 64, 65, 255, 1000, 4097, 32000, 32769, 65537, 70001]


def params(rng, rows, n):
    t = rng.choice([0.0, 0.2, 0.7, 1.0, 1.6, 30.0], rows).astype(np.float32)
    k = np.where(rng.random(rows) < 0.4, rng.choice([0, -1, n, n + 5, 2 ** 31 - 1], rows), np.exp(rng.uniform(0, np.log(n + 1), rows))).astype(np.int64)
    p = np.where(rng.random(rows) < 0.4, rng.choice([1.0, 2.0, 0.0, -1.0], rows), rng.random(rows)).astype(np.float32)
    m = np.where(rng.random(rows) < 0.5, rng.choice([0.0, -1.0, 1.0, 7.0], rows), rng.random(rows) ** 3).astype(np.float32)
    return t, k.astype(np.int32), p, m


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", SIZES)
def test_all_filters(gpu, n, kind):
    rng = np.random.default_rng(n + len(kind))
    rows = 40 if n < 10000 else 12
    x = rows_of(rng, rows, n, kind)
    t, k, p, m = params(rng, rows, n)
    check(x, t, rng.random(rows).astype(np.float32), k, p, m, pad=n % 3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1000, 32000, 100003])
@pytest.mark.parametrize("filters", ["none", "k", "p", "m", "kp"])
def test_each_filter_alone(gpu, n, filters, kind):
    rng = np.random.default_rng(n)
    rows = 6
    x = rows_of(rng, rows, n, kind)
    k = [1, 2, 50, 999, n // 2, n - 1] if "k" in filters else None
    p = [0.01, 0.3, 0.9, 0.99, 0.9999, np.nextafter(np.float32(1), np.float32(0))] if "p" in filters else None
    m = [1e-6, 0.001, 0.1, 0.5, 0.9, 1.0] if "m" in filters else None
    for r in ([0.0] * 6, [1 - 2.0 ** -24] * 6, rng.random(rows)):
        check(x, [0.3, 0.8, 1.0, 1.0, 1.3, 2.0], np.asarray(r, np.float32), k, p, m)


@pytest.mark.parametrize("rows,n", [(1, 262144), (5, 262144), (3, 262143), (2, 300001), (300, 2000), (1, 1048577)])
def test_sizes_of_batches(gpu, rows, n):
    rng = np.random.default_rng(rows)
    x = rows_of(rng, rows, n, "peaked")
    t, k, p, m = params(rng, rows, n)
    t[0], k[0], p[0], m[0] = 1.0, 0, 0.9, 0.0
    check(x, t, rng.random(rows).astype(np.float32), k, p, m, pad=1)


@pytest.mark.parametrize("n", [5, 3000, 40000, 140000])
def test_rows_without_a_token(gpu, n):
    """NaN, +inf or nothing but -inf in a row, and parameters out of their ranges: that row alone has no token."""
    x = np.random.default_rng(n).standard_normal((14, n)).astype(np.float32)
    t, r, p, m = np.full(14, 0.9, np.float32), np.full(14, 0.3, np.float32), np.full(14, 0.8, np.float32), np.full(14, 0.1, np.float32)
    x[1, n - 1], x[2, 0], x[3], x[4, n // 2] = np.nan, np.inf, -np.inf, -np.nan
    t[5], t[6], t[7] = -0.5, np.nan, np.inf
    r[8], r[9], r[10] = 1.0, -1e-9, np.nan
    p[11], m[12] = np.nan, np.nan
    check(x, t, r, None, p, m)
    got, prob = run(x, t, r, None, p, m)
    assert (got[1:13] == NONE).all() and np.isnan(prob[1:13]).all() and (got[[0, 13]] < n).all()


def test_greedy_takes_the_first_of_the_largest(gpu):
    x = np.full((4, 50000), -2.0, np.float32)
    x[0, [77, 40000]], x[1, [49999, 3]], x[2, 5], x[2, 900], x[3] = 1.5, 0.25, -0.0, 0.0, -np.inf
    x[2, :5] = -1
    x[3, 31234] = -1e30
    got, prob = run(x, [0.0] * 4, [0.99] * 4, [7] * 4, [0.1] * 4)
    assert got.tolist() == [77, 3, 5, 31234] and (prob == 1).all()


def test_zeros_of_both_signs_are_equal(gpu):
    x = np.zeros((1, 64), np.float32)
    x[0, 1::2] = -0.0
    for k in (1, 2, 5):
        got, _ = run(x, [1.0], [0.999], [k])
        assert got[0] == k - 1


def test_smallest_and_largest_temperatures(gpu):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 5000)).astype(np.float32) * 3
    check(x, [1e-45, 1e-30, 1e-3, 1e3, 1e30, 3.4e38], rng.random(6).astype(np.float32), None, [1, 0.5, 0.9, 0.9, 0.5, 0.7])
    x = np.float32([[3.4e38, -3.4e38, 3.39e38, 0]])
    check(x, [1e38], np.float32([0.6]))


def test_rows_repeat_bit_for_bit_and_do_not_depend_on_their_neighbours(gpu):
    rng = np.random.default_rng(3)
    x = rows_of(rng, 64, 32000, "half")
    t, k, p, m = params(rng, 64, 32000)
    r = rng.random(64).astype(np.float32)
    first = run(x, t, r, k, p, m)
    for a, b in zip(first, run(x, t, r, k, p, m, pad=7)):
        assert np.array_equal(a, b, equal_nan=True)
    for i in (0, 17, 63):
        one = run(x[i:i + 1], t[i:i + 1], r[i:i + 1], k[i:i + 1], p[i:i + 1], m[i:i + 1])
        assert one[0][0] == first[0][i] and np.array_equal(one[1][0], first[1][i], equal_nan=True)
    assert np.array_equal(run(x, t, r, k, p, m, prob=False)[0], first[0])


@pytest.mark.parametrize("rows,n", [(20, 2000), (3, 150000)])
def test_captured_and_replayed(gpu, rows, n):
    rng = np.random.default_rng(n)
    x, t, k, p, r = (torch.zeros((rows, n), device="cuda"), torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"),
                     torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda"))
    index, prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    ws = torch.full((E.sample_workspace(rows, n) + 16,), 255, dtype=torch.uint8, device="cuda")

    def body(st):
        E.sample(x.data_ptr(), rows, n, n, t.data_ptr(), k.data_ptr(), p.data_ptr(), 0, r.data_ptr(), index.data_ptr(), prob.data_ptr(),
                 ws.data_ptr(), ws.numel(), st)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        body(side.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body(torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        hx = rows_of(rng, rows, n, KINDS[turn])
        ht, hk, hp, _ = params(rng, rows, n)
        hr = rng.random(rows).astype(np.float32)
        for d, h in ((x, hx), (t, ht), (k, hk), (p, hp), (r, hr)):
            d.copy_(torch.from_numpy(h))
        g.replay()
        torch.cuda.synchronize()
        for b in range(rows):
            want, share = paged_ref.sample(hx[b], ht[b], hr[b], int(hk[b]), hp[b])
            assert index[b].item() == want and abs(prob[b].item() / share - 1) < 2.0 ** -23


def test_host_entry(gpu):
    rng = np.random.default_rng(9)
    for n in (1, 700, 100000):
        x = rows_of(rng, 1, n, "peaked")[0]
        for t, r, k, p, m in ((1.0, 0.3, 0, 1.0, 0.0), (0.7, 0.9, 40, 0.95, 0.02), (0.0, 0.5, 0, 1.0, 0.0)):
            got = E.host_sample(x, t, r, k, p, m)
            want = paged_ref.sample(x, t, r, k, p, m)
            assert got[0] == want[0] and abs(got[1] / want[1] - 1) < 2.0 ** -23
    for bad in ([1.0, np.nan], [np.inf, 0], [-np.inf, -np.inf]):
        with pytest.raises(E.EngineError) as e:
            E.host_sample(bad, 1.0, 0.5)
        assert e.value.kind == "Sampling"


def test_session_samples_its_own_logits(gpu, c0_path):
    model = E.LoadedModel.load(c0_path)
    s = E.InferenceSession(model)
    s.prefill([5, 9, 100, 7])
    rng = np.random.default_rng(2)
    for step in range(6):
        x = s.logits_last_token()
        r = float(np.float32(rng.random()))
        for t, k, p, m in ((0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (1.2, 0, 0.9, 0.0)):
            tok = E.sample_next_token(s, t, r, k, p, m)
            assert tok == paged_ref.sample(x, t, r, k, p, m)[0]
        s.decode_token(tok)
    assert E.sample_next_token(s, 0.0, 0.0) == E.greedy_next_token(s)
    for kw, kind in ((dict(temperature=-1.0, r=0.5), "Sampling"), (dict(temperature=1.0, r=1.0), "Op"), (dict(temperature=1.0, r=0.5, top_p=np.nan), "Op")):
        with pytest.raises(E.EngineError) as e:
            E.sample_next_token(s, **kw)
        assert e.value.kind == kind
    with pytest.raises(E.EngineError):
        E.sample_next_token(E.InferenceSession(model), 1.0, 0.5)  # no state yet
