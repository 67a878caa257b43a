"""The paged cache at the ends of its arguments' ranges, against tests/paged_ref.py."""
import numpy as np
import pytest

import paged_ref
from inference_engine_rust_amd import engine as E
from test_gpu_paged import Dev, attend, check, dev, filled, host, ints, queries, stream

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,rotary", [(64, 2), (64, 6), (128, 66), (256, 62), (512, 510)])
def test_dims_behind_an_odd_number_of_pairs_stay_bit_for_bit(gpu, dtype, hd, rotary):
    """The pair that follows the last rotated one: infinities, a NaN and zeros of both signs beside each other."""
    rng = np.random.default_rng(hd + rotary)
    heads, kv, n, page = 4, 2, 12, 16
    ref = paged_ref.Paged(3, kv, page, hd, [[2, 0]], dtype)
    d = Dev(ref)
    rows = rng.standard_normal((1, n, heads + 2 * kv, hd)).astype(np.float32)
    pairs = np.float32([(np.inf, 1), (1, -np.inf), (-0.0, 0.0), (0.0, -0.0), (-0.0, -0.0), (np.nan, 2), (3, np.nan), (np.inf, np.inf), (-0.0, 5),
                        (-0.0, -5), (5, -0.0), (-np.inf, -0.0)])
    rows[0, :, :, rotary:rotary + 2] = pairs[:, None]
    rope = rng.uniform(-1, 1, (2 * page, rotary // 2, 2)).astype(np.float32)
    x, table, out = dev(rows), dev(rope), torch.zeros((1, n, heads * hd), device="cuda")
    p, stride = x.data_ptr(), (heads + 2 * kv) * hd
    E.paged_append(d.h, p, p + 4 * heads * hd, p + 4 * (heads + kv) * hd, heads, n, stride, table.data_ptr(), 2 * page, rotary,
                   ints([3]).data_ptr(), 0, 0, out.data_ptr(), heads * hd, stream())
    turned = paged_ref.rotated(rows[:, :, :heads + kv], rope[3:3 + n][None])
    ref.append(turned[:, :, heads:], rows[:, :, heads + kv:], [3], [n])
    got, want = host(out).reshape(n, heads, hd), turned[0, :, :heads]
    assert np.array_equal(got, want, equal_nan=True) and np.array_equal(np.signbit(got)[want == 0], np.signbit(want)[want == 0])
    d.check(ref)
    for pool, held in zip(d.pool, (ref.k, ref.v)):
        got = host(pool.float())
        assert np.array_equal(np.signbit(got)[held == 0], np.signbit(held)[held == 0])


@pytest.mark.parametrize("dtype,bits", [("f32", 0x7F800001), ("f32", -0x7F0001), ("f32", 0x7FC00000), ("f16", 0x7C01), ("f16", -0x3FF)])
@pytest.mark.parametrize("kv,group,hd,n_q,shared", [(1, 4, 64, 3, 0), (1, 8, 64, 5, 0), (2, 8, 128, 9, 0), (1, 8, 128, 3, 40), (2, 8, 256, 5, 0),
                                                    (1, 8, 512, 7, 0)])
def test_a_nan_of_any_kind_in_v_is_a_nan(gpu, dtype, bits, kv, group, hd, n_q, shared):
    """Signalling ones with bits of their mantissa's low end alone among them, in entries that only some queries see."""
    rng = np.random.default_rng(hd)
    lens, page = [90, 75, 61], 16
    ref, pages = filled(3, dtype, kv, hd, page, lens, common=-(-shared // page))
    d = Dev(ref)
    q, scale = queries(rng, len(lens), n_q, kv * group, hd), 1 / np.sqrt(hd)
    clean, bound = ref.attention(q, lens, 0, scale, shared, pages)
    want = clean.copy()
    for b, n in enumerate(lens):
        at = n - 1 - b % n_q  # (seen by the last b + 1 tokens)
        d.pool[1][int(ref.table[b, at // page]), 0, at % page, 5:hd - 3].view(torch.int32 if dtype == "f32" else torch.int16).fill_(bits)
        want[b, n_q - 1 - b % n_q:, :group, 5:hd - 3] = np.nan
    assert np.isnan(host(d.pool[1].float())[int(ref.table[0, 89 // page]), 0, 89 % page, 5:hd - 3]).all()
    got = attend(d, q, lens, 0, scale, shared, pages)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    check(np.where(np.isnan(want), 0, got), np.where(np.isnan(want), 0, clean), bound)
