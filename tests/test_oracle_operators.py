"""oracle/operators.py against closed forms and central differences (no GPU)."""
import numpy as np

from oracle import attention as A
from oracle import operators as P


def _pages(rng, lengths, heads, size, dim, spare=3):
    """A dense cache of each sequence, and the same keys in shuffled pages."""
    m = max(1, -(-max(lengths) // size))
    total = sum(-(-n // size) for n in lengths) + spare
    order = iter(rng.permutation(total))
    table = np.full((len(lengths), m), -1, np.int32)
    k, v = rng.standard_normal((2, total, heads, size, dim))
    dense = []
    for b, n in enumerate(lengths):
        for i in range(-(-n // size)):
            table[b, i] = next(order)
        dense.append([np.stack([x[table[b, j // size], :, j % size] for j in range(n)], 1) if n else None for x in (k, v)])
    return k, v, table, dense


def test_paged_attention_is_attention_over_the_gathered_keys():
    rng = np.random.default_rng(0)
    lengths = [1, 5, 16, 23]
    k, v, table, dense = _pages(rng, lengths, 2, 4, 8)
    q = rng.standard_normal((4, 6, 8))
    got = P.paged_attention(q, k, v, table, np.array(lengths, np.int32))
    for b, n in enumerate(lengths):
        kd, vd = (np.repeat(x, 3, 0)[None] for x in dense[b])
        want = A.attention_f64(q[b][None, :, None], kd, vd, causal=False, scale=8 ** -0.5)
        np.testing.assert_allclose(got[b], want[0, :, 0], rtol=1e-12, atol=1e-12)


def test_paged_attention_masks():
    rng = np.random.default_rng(1)
    k, v, table, dense = _pages(rng, [12], 1, 4, 8)
    q = rng.standard_normal((1, 1, 8))
    full = P.paged_attention(q, k, v, table, [12])
    assert np.array_equal(P.paged_attention(q, k, v, table, [12], window=12), full)
    # one key left: its value; none left: zeros; a page taken away: the others
    np.testing.assert_allclose(P.paged_attention(q, k, v, table, [12], window=1)[0, 0], dense[0][1][0, 11])
    assert not P.paged_attention(q, k, v, table, [0]).any()
    assert not P.paged_attention(q, k, v, np.full_like(table, -1), [12]).any()
    hole = table.copy()
    hole[0, 1] = 99
    s = (dense[0][0][0] @ q[0, 0]) / np.sqrt(8)
    e = np.exp(s) * ~np.isin(np.arange(12), [4, 5, 6, 7])
    np.testing.assert_allclose(P.paged_attention(q, k, v, hole, [12])[0, 0], e @ dense[0][1][0] / e.sum())


def test_append_last_row_stays():
    k = np.zeros((2, 1, 4, 2))
    new = np.arange(10.0).reshape(5, 1, 2)
    k2, v2 = P.paged_append(k, k, new, -new, [5, -1, 5, 8, 0])
    assert (k2[1, 0, 1] == new[2, 0]).all() and (k2[0, 0, 0] == new[4, 0]).all() and np.count_nonzero(k2) == 4
    assert (v2 == -k2).all() and not k.any()


def test_norm_closed_form_and_gradient():
    y, t = P.add_rms_norm(np.array([[3.0, 4.0]]), np.zeros((1, 2)), np.array([1.0, 2.0]), 0.0)
    np.testing.assert_allclose(y, [[3 / np.sqrt(12.5), 8 / np.sqrt(12.5)]])
    rng = np.random.default_rng(2)
    x, r, dy, ds = rng.standard_normal((4, 3, 7))
    g = rng.standard_normal(7)
    dx, dg = P.add_rms_norm_grad(dy, ds, x + r, g, 1e-2)

    def loss(x, g):
        y, t = P.add_rms_norm(x, r, g, 1e-2)
        return (y * dy).sum() + (t * ds).sum()
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-6
        np.testing.assert_allclose((loss(x + e, g) - loss(x - e, g)) / 2e-6, dx[i], atol=1e-7)
    for i in range(7):
        e = np.zeros_like(g)
        e[i] = 1e-6
        np.testing.assert_allclose((loss(x, g + e) - loss(x, g - e)) / 2e-6, dg[i], atol=1e-7)


def test_logprobs_closed_form_and_gradient():
    lp, H, lse, top, ids = P.token_logprobs(np.zeros((2, 8)), np.array([3, 9]), 3)
    np.testing.assert_allclose(lp, [-np.log(8), 0.0])
    np.testing.assert_allclose(H, np.log(8))
    np.testing.assert_allclose(lse, np.log(8))
    assert (ids == [[0, 1, 2]] * 2).all() and np.allclose(top, -np.log(8))
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 6))
    x[1, 2] = -np.inf
    tok = np.array([4, 0, -1])
    g, h = rng.standard_normal((2, 3))
    _, H, lse = P.token_logprobs(x, tok)
    dx = P.token_logprobs_grad(x, tok, lse, H, g, h)

    def loss(x):
        lp, H, _ = P.token_logprobs(x, tok)
        return (lp * g).sum() + (H * h).sum()
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-6
        np.testing.assert_allclose((loss(x + e) - loss(x - e)) / 2e-6, dx[i], atol=1e-8)
    assert dx[1, 2] == 0 and np.allclose(dx.sum(1), 0)
