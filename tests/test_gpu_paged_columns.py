"""Attention over the paged KV cache where the launch's shape changes: many columns (a join of one a wave, more than 64
partial results of a column), own entries beside shared ones on both sides of the rule for the shared ones' workgroups,
lengths at the limits of one chunk. Against tests/paged_ref.py in 64 bits, with its bounds."""
import numpy as np
import pytest

from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,kv,group,batch,n_q,shared,own", [
    (64, 1, 8, 64, 1, 8300, 40), (128, 8, 4, 64, 1, 1200, 200), (128, 8, 4, 64, 1, 1200, 30), (256, 1, 8, 64, 1, 300, 100),
    (512, 1, 8, 64, 1, 200, 100), (64, 2, 8, 33, 1, 0, 531), (128, 1, 8, 16, 5, 300, 400), (64, 1, 8, 70, 1, 100, 300)])
def test_many_columns(gpu, dtype, hd, kv, group, batch, n_q, shared, own):
    rng = np.random.default_rng(batch + own)
    lens = [int(n) for n in shared + rng.integers(0, own + 1, batch)]
    lens[0], lens[1] = shared + own, max(0, shared - 1)
    check_attention(shared + hd, dtype, kv, group, hd, n_q, lens, page=16, shared=shared)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,group,n_q", [(64, 4, 1), (128, 4, 1), (256, 2, 1), (512, 8, 1), (128, 4, 5), (256, 8, 3)])
@pytest.mark.parametrize("around", [64, 128, 256, 512])
def test_lengths_at_one_chunks_limits(gpu, dtype, hd, group, n_q, around):
    for lens in ([around - 1], [around], [around + 1], [around, 0, around - 1]):
        check_attention(around, dtype, 2, group, hd, n_q, lens, page=32)
    check_attention(around, dtype, 2, group, hd, n_q, [around + 300, around + 17], page=32, window=around)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("group,n_q", [(8, 2), (1, 17), (4, 8), (3, 11), (8, 8), (5, 13)])
@pytest.mark.parametrize("shared,window", [(0, 0), (130, 0), (0, 100)])
def test_columns_of_a_sequence(gpu, dtype, hd, group, n_q, shared, window):
    check_attention(hd + n_q, dtype, 1, group, hd, n_q, [shared + 700, shared + 3, shared + 129, 0], page=32, shared=shared, window=window)
