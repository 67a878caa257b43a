"""Attention over f32 pages on inputs whose answer lies in the low bits of one operand (paged_planes, with its bars): many
columns of one sequence, of a shared prefix, and few columns."""
import numpy as np
import pytest

import paged_planes
import paged_ref
from test_gpu_paged import Dev, attend

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ENTRIES, PAGE = 100, 16


@pytest.mark.parametrize("turn", [0, 1])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("name", paged_planes.CASES)
@pytest.mark.parametrize("form", ["one sequence", "shared", "few columns"])
def test_low_bits(gpu, form, name, hd, turn):
    K, V, q, scale, bar = paged_planes.case(name, hd, ENTRIES, 40, turn)
    batch, n_q = {"one sequence": (1, 5), "shared": (5, 1), "few columns": (5, 1)}[form]
    # n_q - 1 entries of zeros more (each token sees another number of them)
    rest = n_q - 1
    pages = -(-(ENTRIES + rest) // PAGE)
    shared = 80 if form == "shared" else 0
    table = np.arange(batch * pages).reshape(batch, pages)
    ref = paged_ref.Paged(batch * pages, 1, PAGE, hd, table, "f32")
    for b in range(batch):
        for j in range(ENTRIES + rest):
            at = (table[b, j // PAGE], 0, j % PAGE)
            ref.k[at], ref.v[at] = (K[j], V[j]) if j < ENTRIES else (0, 0)
    got = attend(Dev(ref), q.reshape(batch, n_q, 8, hd).astype(np.float32), [ENTRIES + rest] * batch, 0, scale, shared, table[0]).reshape(40, hd)
    for t in range(n_q):
        rows = np.arange(40).reshape(batch, n_q, 8)[:, t].ravel()
        n = ENTRIES + t
        k, v = (np.concatenate([x, np.zeros((t, hd))]) for x in (K, V))
        p = paged_planes.softmax(scale * (q[rows] @ k.T))
        off, most = np.abs(got[rows] - p @ v), bar(p, v, n)
        assert (off <= most).all(), (t, np.max(off / most))
