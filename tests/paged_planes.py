"""Inputs of attention over f32 pages whose answer lies in the low bits of one operand, the leading ones cancelling, with bars
that follow from the arithmetic. A kernel that holds f32 numbers as three bf16 ones (a: cut off to 8 bits, b: the rest
rounded to 8, c: the rest of that) and adds six of the nine products finds each answer; one that loses a part or a
product does not (test_paged_planes shows it of a model of the arithmetic).

All rounding is f32's, half a unit: 2^-24 of a sum in [1, 2). A case is (K, V [entries][hd], q [columns][hd], scale, bar), bar(p, V, seen)
the largest error of the columns' outputs, p the weights in 64 bits."""
import numpy as np

U = 2.0 ** -24
A = 1 + 255 * 2.0 ** -15  # as bf16 parts 1, 255 2^-15, 0; plus i 2^-23, i < 128: i 2^-23 is the third part


def weights_bar(score):
    """Scores off by `score` at most: a weight and the sum by e^score each."""
    return lambda p, V, seen: (np.expm1(2 * score) + 2.0 ** -18) * (p @ np.abs(V))


def pair_of(c, count, turn):
    return (c + 40 * turn) % count


def k_low(rng, hd, entries, columns, turn):
    """K's third part. Two products of size A cancel, each of their parts' sums rounds twice near 1: off by 2 U, and by less than U
    of the smaller parts, where the scores are i 2 U times the scale: 3 at most."""
    i = rng.integers(0, 128, (entries, hd // 2))
    K = np.full((entries, hd), A)
    K[:, 0::2] += i * 2.0 ** -23
    q = np.zeros((columns, hd))
    for c in range(columns):
        q[c, 2 * pair_of(c, hd // 2, turn):][:2] = 1, -1
    scale = 2.0 ** 23 * 3 / 127
    return K, np.where(np.tile(i, 2) < 64, -1.0, 1.0), q, scale, weights_bar(3 * U * scale)


def q_low(rng, hd, entries, columns, turn):
    """The same of q's third part, over keys of 0 and 1."""
    b = rng.integers(0, 2, (entries, hd // 2))
    K = np.zeros((entries, hd))
    K[:, 0::2], K[:, 1::2] = b, -b
    q = np.zeros((columns, hd))
    for c in range(columns):
        q[c, 2 * pair_of(c, hd // 2, turn):][:2] = A + rng.integers(64, 128) * 2.0 ** -23, A
    scale = 2.0 ** 23 * 3 / 127
    return K, np.tile(2.0 * b - 1, 2), q, scale, weights_bar(3 * U * scale)


def both_middle(rng, hd, entries, columns, turn):
    """The product of the second parts: (1 + u)(1 + v) - (1 + u) - (1 + v) + 1 = u v. Four sums of up to 2 round by 2 U each."""
    m = rng.integers(0, 256, (entries, hd // 4))
    u, v = m * 2.0 ** -15, 255 * 2.0 ** -15
    K = np.stack([1 + u, 1 + u, np.ones_like(u), np.ones_like(u)], -1).reshape(entries, hd)
    q = np.zeros((columns, hd))
    for c in range(columns):
        q[c, 4 * pair_of(c, hd // 4, turn):][:4] = 1 + v, -1, -(1 + v), 1
    scale = 3 * 2.0 ** 30 / 255 ** 2
    return K, np.where(np.tile(m, 4) < 128, -1.0, 1.0), q, scale, weights_bar(9 * U * scale)


def pairs_of_entries(rng, hd, entries, value):
    """V with two entries a dim, value(dim) and the other's sign, the rest zero."""
    V = np.zeros((entries, hd))
    for d in range(hd):
        a, b = rng.permutation(entries)[:2]
        V[a, d], V[b, d] = value(d)
    return V


def v_low(rng, hd, entries, columns, turn):
    """V's third part, weights all 1: A and -A cancel in the sum over entries, two roundings near 1 (as many again if they are in
    different chunks or waves), and the quotient's."""
    V = pairs_of_entries(rng, hd, entries, lambda d: (A + rng.integers(64, 128) * 2.0 ** -23, -A))
    return np.zeros((entries, hd)), V, np.zeros((columns, hd)), 1.0, lambda p, V, seen: 8 * U / seen


def p_low(rng, hd, entries, columns, turn):
    """All bits of the weights (of keys with all bits and queries with two parts), against second parts of V: the two weights of a dim (0.88 to 1.14) are off by a unit of exp2, 2 U,
    each, the products that are left out are 2^-7 2^-17 = U each, the sums round twice near 1; and as much again."""
    K, q = np.zeros((entries, hd)), np.zeros((columns, hd))
    K[:, turn % hd] = np.float32(-rng.uniform(0, 2.0 ** -3, entries))
    q[:, turn % hd] = [(1, 0.5, -1, -0.5)[c % 4] * (1 + rng.integers(0, 256) * 2.0 ** -15) for c in range(columns)]

    def value(d):
        v = 1 + rng.integers(0, 256) * 2.0 ** -15
        return v, -v
    return K, pairs_of_entries(rng, hd, entries, value), q, 1.0, lambda p, V, seen: 16 * U / seen * 1.14 + 2.0 ** -20 * np.abs(p @ V)


CASES = {f.__name__: f for f in (k_low, q_low, both_middle, v_low, p_low)}


def case(name, hd, entries, columns, turn):
    K, V, q, scale, bar = CASES[name](np.random.default_rng([hd, turn]), hd, entries, columns, turn)
    for x in (K, V, q):
        assert np.array_equal(x.astype(np.float32), x)
    return K, V, q, scale, bar


def softmax(s):
    e = np.exp(s - s.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def parts(x):
    """x (f32 numbers as float64) as three bf16 numbers."""
    def bf16(y, nearest):
        bits = y.astype(np.float32).view(np.uint32).astype(np.uint64)
        if nearest:
            bits = bits + 0x7FFF + (bits >> 16 & 1)
        return (bits & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    a = bf16(x, False)
    b = bf16(x - a, True)
    return a, b, bf16(x - a - b, True)


SIX = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]


def model(K, V, q, scale, scores=SIX, sums=SIX):
    """Attention by products of parts, (K's, q's) and (V's, the weights'), their sums in 64 bits."""
    k, v, y = parts(K), parts(V), parts(q)
    s = scale * sum(y[j] @ k[i].T for i, j in scores)
    e = np.exp(s - s.max(-1, keepdims=True)).astype(np.float32).astype(np.float64)
    w = parts(e)
    return sum(w[j] @ v[i] for i, j in sums) / e.sum(-1, keepdims=True)
