"""CPU checks of the 8-bit KV cache's entries (include/iek.h): what they refuse, workspace sizes, and the reference's
rounding against its own bound."""
import numpy as np
import pytest

import kv8_ref
from inference_engine_rust_amd import engine as E

P = 1 << 20  # aligned addresses that nothing reads: every call here is refused, or has nothing to do


def cache(dtype=E.I8, batch=2, kv=2, cap=100, hd=64, k=P, v=2 * P, ks=3 * P, vs=4 * P):
    return E.KV8Cache(dtype, batch, kv, cap, hd, k, v, ks, vs)


def append(c, k=5 * P, v=6 * P, n=4, stride=128, start=7 * P, count=0, len_out=0, weights=0):
    E.kv8_append(c, k, v, n, stride, start, count, len_out, weights)


def load(c, n=4, stride=128, k=5 * P, v=6 * P):
    E.kv8_load(c, n, stride, 0, 0, k, v)


def attention(c, q=5 * P, heads=4, n_q=1, stride=256, lens=6 * P, max_len=100, window=0, out=7 * P, w_in=0, w_out=0,
              ws=8 * P, size=None):
    if size is None:
        size = 1 << 30
    E.kv8_attention(c, q, heads, n_q, stride, lens, max_len, window, 0.125, out, w_in, w_out, ws, size)


def evict(c, to, w=16 * P, w_out=17 * P, lens=18 * P, len_out=19 * P, max_len=100, keep=50, first=1, last=10, ws=8 * P,
          size=1 << 30):
    E.kv8_evict(c, to, w, w_out, lens, len_out, max_len, keep, first, last, 0, ws, size)


def other(**kw):
    return cache(k=10 * P, v=11 * P, ks=12 * P, vs=13 * P, **kw)


def refused(kind, what, call, *a, **kw):
    with pytest.raises(E.EngineError) as e:
        call(*a, **kw)
    assert e.value.kind == kind and what in str(e.value), str(e.value)


@pytest.mark.parametrize("call", [append, load, attention, lambda c: evict(c, other())])
def test_every_entry_checks_the_cache(call):
    refused("Op", "null cache", call, None)
    refused("Op", "dtype", call, cache(dtype=E.F16))
    for hd in (0, 32, 96, 1024):
        refused("Op", "head_dim", call, cache(hd=hd))
    refused("Op", "no KV heads", call, cache(kv=0))
    refused("Op", "no KV heads", call, cache(cap=0))
    refused("Op", "too large", call, cache(batch=1 << 40))
    refused("Op", "too large", call, cache(cap=1 << 31))
    refused("Op", "too large", call, cache(batch=60000, kv=4000))
    for name in ("k", "v", "ks", "vs"):
        refused("Op", "null", call, cache(**{name: 0}))
        refused("Op", "aligned", call, cache(**{name: P + 2}))
    refused("Op", "k is not 16-byte", call, cache(k=P + 8))


def test_append_and_load_refuse():
    for call in (append, load):
        refused("Op", "stride", call, cache(), stride=130)
        refused("Op", "stride", call, cache(), stride=124)
        refused("Op", "null k rows", call, cache(), k=0)
        refused("Op", "v rows is not", call, cache(), v=P + 4)
        refused("KvCache", "100", call, cache(), n=101)
        call(cache(), n=0, k=0)  # nothing to do
        call(cache(batch=0), k=0)
    refused("Op", "start is not", append, cache(), start=P + 1)
    refused("Op", "start and len_out overlap", append, cache(), start=P, len_out=P + 4)
    refused("Op", "count and len_out overlap", append, cache(), count=P, len_out=P)


def test_attention_refuses():
    refused("Op", "GQA", attention, cache(), heads=3)
    refused("Op", "GQA", attention, cache(), heads=0)
    refused("Op", "GQA", attention, cache(), heads=18)
    refused("Op", "64 query", attention, cache(), n_q=65)
    refused("Op", "q_stride", attention, cache(), stride=252)
    refused("Op", "q_stride", attention, cache(), stride=258)
    refused("KvCache", "position 100 is out of bounds (max_seq_len is 100)", attention, cache(), max_len=101)
    for name in ("q", "lens", "out", "ws"):
        refused("Op", "null", attention, cache(), **{name: 0})
    refused("Op", "q is not 16", attention, cache(), q=P + 4)
    refused("Op", "out is not 16", attention, cache(), out=P + 8)
    refused("Op", "weights_in without", attention, cache(), w_in=P)
    refused("Op", "weights_in and weights_out overlap", attention, cache(), w_in=P, w_out=P + 4)
    need = E.kv8_attention_workspace(cache(), 4, 1, 100, False)
    refused("Op", "too small", attention, cache(), size=need - 1)
    more = E.kv8_attention_workspace(cache(), 4, 1, 100, True)
    assert more > need
    refused("Op", "too small", attention, cache(), w_out=P, size=more - 1)
    attention(cache(), n_q=0, q=0)
    attention(cache(batch=0), q=0)


def test_evict_refuses():
    refused("Op", "differ", evict, cache(), other(dtype=E.E4M3))
    refused("Op", "differ", evict, cache(), other(batch=3))
    refused("Op", "differ", evict, cache(), other(kv=1))
    refused("Op", "differ", evict, cache(), other(hd=128))
    refused("Op", "first + last", evict, cache(), other(), first=41)
    refused("Op", "first + last", evict, cache(), other(), first=1 << 63, last=1 << 63)
    refused("KvCache", "100", evict, cache(), other(), max_len=101)
    refused("KvCache", "max len is 40", evict, cache(), other(cap=40))
    refused("Op", "share some", evict, cache(), cache())  # in place, but the weights are not
    refused("Op", "share some", evict, cache(), other(), w_out=16 * P)
    refused("Op", "share some", evict, cache(), cache(cap=99), w_out=16 * P)
    refused("Op", "overlap", evict, cache(), cache(k=P + 64))
    refused("Op", "len and len_out overlap", evict, cache(), other(), len_out=18 * P + 4)
    for name in ("w", "w_out", "lens", "len_out", "ws"):
        refused("Op", "null", evict, cache(), other(), **{name: 0})
    need = E.kv8_evict_workspace(cache(), 100, 50)
    refused("Op", "too small", evict, cache(), other(), size=need - 1)
    evict(cache(batch=0), other(batch=0), w=0)


def test_workspaces_grow_with_what_they_hold():
    c = cache(batch=3, kv=8, cap=70000, hd=128)
    sizes = [E.kv8_attention_workspace(c, 32, 1, n, True) for n in (0, 1, 1000, 70000)]
    assert sizes == sorted(sizes) and sizes[-1] >= 3 * 32 * 70000 * 4
    assert E.kv8_attention_workspace(c, 64, 64, 70000, True) >= 3 * 64 * 64 * 70000 * 4
    assert E.kv8_evict_workspace(c, 70000, 60000) >= 3 * 8 * 60000 * 4
    refused("KvCache", "70000", E.kv8_attention_workspace, c, 32, 1, 70001, True)
    assert E.kv8_attention_workspace(c, 32, 0, 70000, True) == 0
    assert E.kv8_attention_workspace(cache(batch=0), 4, 1, 100, True) == 0 == E.kv8_evict_workspace(cache(batch=0), 100, 50)
    refused("KvCache", "70000", E.kv8_evict_workspace, c, 70001, 5)


@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_row_by_row_rounding_stays_under_a_step(dtype):
    """Rows appended one by one, each twice as large as any before: every earlier row is rounded again at each."""
    c = kv8_ref.Cache(1, 1, 32, 64, dtype)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 32, 1, 64)) * 2.0 ** np.arange(32)[None, :, None, None]
    for i in range(32):
        c.append(x[:, i:i + 1], x[:, i:i + 1], [i], [1])
    got, s = c.value(0, 0, 0, 32), c.scale[0][0, 0, 0]
    step = s if dtype == "i8" else np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(x[0, :, 0]) / s, 2 ** -6))) - 3) * s, s * 2.0 ** -9)
    assert (np.abs(got - x[0, :, 0]) < step).all()
    assert np.abs(x).max() <= kv8_ref.TOP[dtype] * s and np.abs(x).max() > kv8_ref.TOP[dtype] * s / 2


def test_what_a_launch_cannot_hold_the_workspace_query_refuses_too():
    """A join of 2^24 workgroups and more: 65520 KV heads of 512 with 136 columns each; and what lies below."""
    c = cache(batch=16, kv=4095, cap=4000, hd=512)
    refused("Op", "too large", E.kv8_attention_workspace, c, 8 * 4095, 17, 4000, False)
    refused("Op", "too large", attention, c, heads=8 * 4095, n_q=17, stride=512 * 8 * 4095, max_len=4000, size=1 << 62)
    # (2^29 floats of q, and 2^31 weights)
    assert E.kv8_attention_workspace(cache(batch=16, kv=4096 // 2, cap=4000, hd=512), 8 * 2048, 4, 4000, False) > 0
    assert E.kv8_attention_workspace(cache(batch=512, kv=8, cap=1 << 19, hd=64), 8, 1, 1 << 19, True) > 0
    refused("Op", "too large", E.kv8_attention_workspace, cache(kv=4097), 4097, 1, 100, False)
