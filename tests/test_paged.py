"""CPU checks of the paged cache's and the batch sampling's entries (include/iek.h): what they refuse, workspace sizes,
the RoPE table, and the 64-bit references against small cases worked by hand."""
import numpy as np
import pytest

import paged_ref
from inference_engine_rust_amd import engine as E

P = 1 << 20  # aligned addresses that nothing reads: every call here is refused, or has nothing to do


def cache(dtype=E.F32, pages=10, kv=2, page=16, hd=64, k=P, v=2 * P, batch=2, max_pages=5, table=3 * P):
    return E.PagedKV(dtype, pages, kv, page, hd, k, v, batch, max_pages, table)


def append(c, q=4 * P, k=5 * P, v=6 * P, heads=4, n=3, stride=512, rope=7 * P, rows=80, rotary=64, start=8 * P, count=0,
           len_out=0, q_out=9 * P, q_stride=256):
    E.paged_append(c, q, k, v, heads, n, stride, rope, rows, rotary, start, count, len_out, q_out, q_stride)


def attention(c, q=4 * P, heads=4, n_q=1, stride=256, lens=5 * P, max_len=80, pages=6 * P, shared=7 * P, max_shared=40, window=0,
              out=8 * P, ws=9 * P, size=1 << 40):
    E.paged_attention(c, q, heads, n_q, stride, lens, max_len, pages, shared, max_shared, window, 0.125, out, ws, size)


def sample(logits=P, rows=3, n=100, stride=100, t=2 * P, k=3 * P, p=4 * P, m=5 * P, r=6 * P, index=7 * P, prob=8 * P, ws=9 * P,
           size=1 << 40):
    E.sample(logits, rows, n, stride, t, k, p, m, r, index, prob, ws, size)


def refused(kind, what, call, *a, **kw):
    with pytest.raises(E.EngineError) as e:
        call(*a, **kw)
    assert e.value.kind == kind and what in str(e.value), str(e.value)


@pytest.mark.parametrize("call", [append, attention])
def test_every_entry_checks_the_cache(call):
    refused("Op", "null cache", call, None)
    refused("Op", "dtype", call, cache(dtype=E.I8))
    for hd in (0, 32, 96, 1024):
        refused("Op", "head_dim", call, cache(hd=hd))
    for page in (0, 1, 8, 24, 2048, 1 << 40):
        refused("Op", "page_size", call, cache(page=page))
    for name in ("kv", "pages", "max_pages"):
        refused("Op", "no KV heads or no pages", call, cache(**{name: 0}))
    for name, much in (("kv", 4097), ("batch", 65536), ("pages", 1 << 31), ("max_pages", (1 << 22) + 1)):
        refused("Op", "too large", call, cache(**{name: much}))
    for name in ("k", "v", "table"):
        refused("Op", "null", call, cache(**{name: 0}))
        refused("Op", "aligned", call, cache(**{name: P + 2}))
    refused("Op", "k is not 16-byte", call, cache(k=P + 8))


def test_append_refuses():
    refused("Op", "row_stride", append, cache(), stride=514)
    refused("Op", "row_stride", append, cache(), stride=252)
    refused("Op", "row_stride", append, cache(), q=0, stride=124)
    refused("Op", "q_out_stride", append, cache(), q_stride=252)
    refused("Op", "query heads", append, cache(), heads=0)
    refused("Op", "rotary_dim", append, cache(), rotary=66)
    refused("Op", "rotary_dim", append, cache(), rotary=31)
    refused("Op", "null rope", append, cache(), rope=0)
    refused("Op", "q without", append, cache(), rotary=0)
    refused("Op", "fewer rope rows", append, cache(), rows=79)
    refused("KvCache", "max len is 80", append, cache(), n=81)
    refused("Op", "too large", append, cache(max_pages=1 << 22), n=(1 << 23) + 1, rows=1 << 26)
    for name in ("k", "v", "q_out"):
        refused("Op", "null", append, cache(), **{name: 0})
    for name in ("q", "k", "v", "q_out"):
        refused("Op", "not 16-byte", append, cache(), **{name: 15 * P + 8})
    for name in ("start", "count", "len_out"):
        refused("Op", "not 4-byte", append, cache(), **{name: 15 * P + 2})
    refused("Op", "start and len_out overlap", append, cache(), start=15 * P, len_out=15 * P + 4)
    refused("Op", "count and len_out overlap", append, cache(), count=15 * P, len_out=15 * P)
    refused("Op", "q and q_out overlap", append, cache(), q_out=4 * P + 256)
    refused("Op", "q and q_out overlap", append, cache(), q_out=4 * P)  # (in place, with another stride)
    append(cache(), n=0, k=0)  # nothing to do
    append(cache(batch=0, table=0), k=0)


def test_attention_refuses():
    refused("Op", "GQA", attention, cache(), heads=3)
    refused("Op", "GQA", attention, cache(), heads=0)
    refused("Op", "GQA", attention, cache(), heads=18)
    refused("Op", "64 query", attention, cache(), n_q=65)
    refused("Op", "q_stride", attention, cache(), stride=252)
    refused("Op", "q_stride", attention, cache(), stride=258)
    refused("KvCache", "position 80 is out of bounds (max_seq_len is 80)", attention, cache(), max_len=81)
    refused("Op", "more shared", attention, cache(), max_len=39)
    for name in ("q", "lens", "out", "ws", "pages", "shared"):
        refused("Op", "null", attention, cache(), **{name: 0})
    refused("Op", "q is not 16", attention, cache(), q=P + 4)
    refused("Op", "out is not 16", attention, cache(), out=P + 8)
    refused("Op", "shared is not 4", attention, cache(), shared=P + 1)
    need = E.paged_attention_workspace(cache(), 4, 1, 80, 40)
    assert need > 0
    refused("Op", "too small", attention, cache(), size=need - 1)
    attention(cache(), n_q=0, q=0)
    attention(cache(batch=0, table=0), q=0)


def test_what_a_launch_cannot_hold_the_workspace_query_refuses_too():
    c = cache(batch=65535, kv=64, hd=512, max_pages=100)
    refused("Op", "too large", E.paged_attention_workspace, c, 512, 64, 1600, 0)
    refused("Op", "too large", attention, c, heads=512, n_q=64, stride=512 * 512, max_len=1600, max_shared=0)
    refused("KvCache", "80", E.paged_attention_workspace, cache(), 4, 1, 81, 0)


def test_workspaces_hold_less_for_less():
    for batch in (1, 7, 64, 65, 300):
        for n_q, group in ((1, 1), (1, 8), (5, 4), (64, 8)):
            c = cache(batch=batch, kv=4, hd=128, max_pages=4096)
            sizes = [E.paged_attention_workspace(c, 4 * group, n_q, n, s) for n, s in
                     ((0, 0), (1, 0), (100, 0), (1000, 0), (1000, 1), (1000, 500), (65536, 500), (65536, 60000))]
            assert sizes == sorted(sizes), sizes
    assert E.paged_attention_workspace(cache(), 4, 0, 80, 0) == 0 == E.paged_attention_workspace(cache(batch=0), 4, 1, 80, 0)


def test_sampling_refuses():
    refused("Sampling", "empty", sample, n=0)
    refused("Op", "row_stride", sample, stride=99)
    refused("Op", "too large", sample, n=(1 << 30) + 1, stride=1 << 31)
    refused("Op", "too large", sample, rows=(1 << 21) + 1)
    for name in ("logits", "t", "r", "index"):
        refused("Op", "null", sample, **{name: 0})
    for name in ("logits", "t", "k", "p", "m", "r", "index", "prob"):
        refused("Op", "not 4-byte", sample, **{name: P + 2})
    sample(rows=0, logits=0)
    refused("Sampling", "empty", E.host_sample, [], 1.0, 0.5)
    for t in (-1.0, np.inf, np.nan):
        refused("Sampling", "temperature", E.host_sample, [1.0], t, 0.5)
    for r in (-0.1, 1.0, np.nan):
        refused("Op", "uniform draw", E.host_sample, [1.0], 1.0, r)
    refused("Op", "NaN", E.host_sample, [1.0], 1.0, 0.5, top_p=np.nan)
    refused("Op", "NaN", E.host_sample, [1.0], 1.0, 0.5, min_p=np.nan)


def test_rope_table():
    t = E.rope_table(64, 64, 10000.0, 3)
    assert t.shape == (3, 32, 2) and (t[0] == [1, 0]).all()
    ang = 2 * 10000.0 ** (-np.arange(32) / 32)
    assert np.abs(t[2] - np.stack([np.cos(ang), np.sin(ang)], 1)).max() < 32 * 2.0 ** -23 * 2  # (32 rounded factors of an angle of 2)
    half = E.rope_table(64, 32, 10000.0, 3, freq_factors=np.full(16, 2.0))
    assert np.abs(half[2, 0] - [np.cos(1.0), np.sin(1.0)]).max() < 2.0 ** -23
    refused("Op", "rotary_dim", E.rope_table, 64, 128, 1e4, 3)
    refused("Op", "even", E.rope_table, 64, 33, 1e4, 3)
    refused("Op", "freq_factors", E.rope_table, 64, 32, 1e4, 3, freq_factors=np.ones(15))
    assert E.rope_table(64, 64, 1e4, 0).shape == (0, 32, 2)


def test_the_reference_of_sampling_by_hand():
    x = np.log([4.0, 1.0, 2.0, 1.0])  # weights 1, 1/4, 1/2, 1/4
    s = paged_ref.sample
    assert [s(x, 1, r)[0] for r in (0, 0.49, 0.51, 0.62, 0.63, 0.87, 0.88, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [s(x, 1, 0.99, top_k=k)[0] for k in (1, 2, 3, 4)] == [0, 2, 2, 3]  # (1 before 3 of the equal ones, but 2 is last)
    assert [s(x, 1, 0.99, top_p=p)[0] for p in (0.49, 0.51, 0.76, 0.9)] == [0, 2, 2, 3]
    assert s(x, 1, 0.5, top_p=0.76) == (0, pytest.approx(4 / 7))
    assert s(x, 1, 0.99, min_p=0.3)[0] == 2 and s(x, 1, 0.99, min_p=2)[0] == 0
    assert s(x, 0, 0.99) == (0, 1.0) and s([1, np.nan], 1, 0)[0] == s([-np.inf] * 2, 1, 0)[0] == 0xFFFFFFFF


def test_the_reference_of_attention_by_hand():
    c = paged_ref.Paged(3, 1, 16, 64, [[2, 0], [2, 7]], "f32")
    k = np.zeros((2, 20, 1, 64), np.float32)
    v = np.broadcast_to(np.arange(20, dtype=np.float32)[None, :, None, None], k.shape)
    assert c.append(k, v, [0, 0], [18, 30]) == [18, 20]  # (the second one's entries from 16 on have no page)
    out, _ = c.attention(np.ones((2, 1, 2, 64), np.float32), [18, 20], 0, 1.0)
    assert np.allclose(out[0], 17 / 2) and np.allclose(out[1], 15 / 2)
    out, _ = c.attention(np.ones((2, 2, 1, 64), np.float32), [18, 0], 4, 1.0)
    assert np.allclose(out[0, 0], (13 + 14 + 15 + 16) / 4) and np.allclose(out[0, 1], (14 + 15 + 16 + 17) / 4) and (out[1] == 0).all()


@pytest.mark.parametrize("hd", [64, 512])
@pytest.mark.parametrize("dtype", [E.F32, E.F16])
@pytest.mark.parametrize("kv,batch,n_q", [(4096, 65535, 64), (4096, 32768, 64), (2048, 65535, 1), (4096, 8192, 8)])
def test_more_columns_than_a_launch_can_have(hd, dtype, kv, batch, n_q):
    c = cache(dtype=dtype, kv=kv, hd=hd, batch=batch)
    refused("Op", "too large", E.paged_attention_workspace, c, 8 * kv, n_q, 80, 40)
