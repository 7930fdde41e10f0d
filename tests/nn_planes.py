"""F32 products by 16-bit planes: a model of the six terms, and operands for
which one pair of planes carries the whole result. (numpy, on the host)

A number is cut into three planes of 8 significant bits each by truncation,
x = x0 + x1 + x2, and x * w is x2 w0 + x0 w2 + x1 w1 + x1 w0 + x0 w1 + x0 w0;
what is left out is below 2^-21 of it."""
import numpy as np

TERMS = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]  # (plane of x, plane of w)


def cut(x):
    return (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)


def planes(x):
    x = np.ascontiguousarray(x, np.float32)
    hi = cut(x)
    mid = cut(x - hi)
    return [hi, mid, x - hi - mid]


def product(x, w, terms=TERMS):
    """x @ w by the planes in `terms`, summed in 64 bits."""
    px, pw = planes(x), planes(w)
    return sum(px[i].astype(np.float64) @ pw[j].astype(np.float64) for i, j in terms)


def carried_by(term, rows, k, n, seed):
    """(x [rows, k], w [k, n]): every row of x has four numbers, in one group of
    four columns of its own, and their products with any column of w cancel but
    for the product of the planes of `term`: the result is 2^-16 or more, the
    largest products 4 or less."""
    r = np.random.default_rng(seed)
    h, v = (1 + r.integers(0, 64, rows) / 128.0), (1 + r.integers(0, 64, n) / 128.0)  # 8 significant bits
    m, q = 2.0**-8 * (1 + r.integers(0, 128, rows) / 128.0), 2.0**-8 * (1 + r.integers(0, 128, n) / 128.0)
    low, s = 2.0**-16 * (1 + r.integers(0, 128, rows) / 128.0), 2.0**-16 * (1 + r.integers(0, 128, n) / 128.0)
    z, zw = np.zeros(rows), np.zeros(n)
    a, b = {(2, 0): ([h + m + low, -(h + m), z, z], [v, v, v, v]),
            (0, 2): ([h, -h, z, z], [v + q + s, v + q, zw, zw]),
            (1, 1): ([h + m, -h, -(h + m), h], [v + q, v + q, v, v]),
            (1, 0): ([h + m, -h, z, z], [v, v, v, v]),
            (0, 1): ([h, -h, z, z], [v + q, v, zw, zw]),
            (0, 0): ([h, z, z, z], [v, v, v, v])}[term]
    x = np.zeros((rows, k), np.float32)
    first = 4 * r.integers(0, k // 4, rows)
    for i in range(4):
        x[np.arange(rows), first + i] = a[i]
    w = np.empty((k // 4 * 4, n), np.float32)
    for i in range(4):
        w[i::4] = b[i]
    w = np.concatenate([w, np.zeros((k - w.shape[0], n), np.float32)])
    return x, w
