"""The operator custom calls on the GPU against oracle/operators.py (float64
on the same rounded inputs).

Tolerances. u is half a step of the result's type (bf16 2^-8, f16 2^-11, f32
2^-24), w = 2^-24. A sum of n products in 32 bits is off by at most n w of the
sum of their magnitudes, in any order. A weight exp(x - max) is off by what x
is off by, plus 4 w for the exponential; where the weights are rounded to 16
bits before the product with the values, by u more, in the sum and in the
product. Each bound is written where it is used, doubled for the rounding of
the bound's own terms."""
import time

import numpy as np
import pytest

from oracle import operators as P
from oracle import ops
from pjrtx_amd.hlo import Builder
from pjrtx_amd.pjrt import DeviceArray

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
W = 2.0 ** -24
NP = {"bf16": np.uint16, "f16": np.float16, "f32": np.float32, "s32": np.int32, "s64": np.int64, "s8": np.int8}


def put(x, dtype):
    """x rounded to the type, as the client takes it."""
    if dtype == "bf16":
        return ops.f32_to_bf16_bits(np.asarray(x, np.float32))
    return np.asarray(x, np.float32).astype(NP[dtype])


def val(a):
    """What an array of put() or of a result stands for, in float64."""
    return ops.bf16_bits_to_f32(a).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


def call(client, build, arrays, dtypes, noalloc=True):
    """The program's results by execute, and by the allocation-free execute on
    the caller's memory: the same bits."""
    b = Builder()
    out = build(b, [b.param(a.shape, d) for a, d in zip(arrays, dtypes)])
    out = list(out) if isinstance(out, (tuple, list)) else [out]
    exe = client.compile(b.build(out))
    res = exe(*arrays, dtypes=[d if d == "bf16" else None for d in dtypes])
    if noalloc:
        p = client.p
        args = [DeviceArray.from_numpy(p, a) for a in arrays]
        outs = [DeviceArray(p, r.nbytes) for r in res]
        exe.execute_noalloc([a.ptr for a in args], [o.ptr for o in outs])
        p.hip_check(p.lib.pjrtx_hip_synchronize(0))
        for r, o in zip(res, outs):
            np.testing.assert_array_equal(o.to_numpy(r.dtype, r.shape).view(np.uint8), r.view(np.uint8))
        for d in args + outs:
            d.free()
    return res


def close(got, want, tol):
    got = val(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want) & ~(got == want)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


# --------------------------------------------------------- paged attention

def cache(rng, lengths, kv_heads, size, dim, dtype, extra=1, poison=True):
    """Shuffled pages, entries past a sequence's last page -1, and NaN in every
    slot that no key holds."""
    used = [-(-n // size) for n in lengths]
    total = sum(used) + 3
    order = iter(rng.permutation(total))
    table = np.full((len(lengths), max(1, max(used, default=0) + extra)), -1, np.int32)
    k, v = rng.standard_normal((2, total, kv_heads, size, dim)).astype(np.float32)
    held = np.zeros((total, size), bool)
    for b, n in enumerate(lengths):
        for i in range(used[b]):
            table[b, i] = next(order)
            held[table[b, i], : n - i * size] = True
    if poison:
        for x in (k, v):
            x[np.broadcast_to(~held[:, None, :], x.shape[:3])] = np.nan
    return put(k, dtype), put(v, dtype), table


def attention_tolerance(q, k, v, want, dtype, scale, length):
    """scale q.k: D products and the scaling, each side of the difference with
    the max; the weights' exponential; their rounding twice; the sums over the
    keys; the result's rounding."""
    kk, vv = np.nan_to_num(val(k)), np.nan_to_num(val(v))
    reach = abs(scale) * np.abs(val(q)).sum(-1).max(initial=0) * np.abs(kk).max(initial=0)
    weights = 2 * ((q.shape[-1] + 4) * W * reach + 4 * W + (U[dtype] if dtype != "f32" else 0) + (length + 8) * W)
    return 2 * weights * np.abs(vv).max(initial=0) + U[dtype] * np.abs(want)


def attend(client, q, k, v, table, lengths, dtype, scale=None, window=0, **kw):
    lengths = np.asarray(lengths, np.int32)
    (got,) = call(client, lambda b, p: b.paged_attention(*p, scale=scale, window=window), [q, k, v, table, lengths],
                  [dtype] * 3 + ["s32"] * 2, **kw)
    want = P.paged_attention(val(q), np.nan_to_num(val(k)), np.nan_to_num(val(v)), table, lengths, scale, window)
    s = q.shape[-1] ** -0.5 if scale is None else scale
    close(got, want, attention_tolerance(q, k, v, want, dtype, s, int(lengths.max(initial=0))))
    return got


LENGTHS = [1, 0, 2, 31, 32, 33, 127, 129, 300]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kv_heads,group,dim,size", [
    (2, 1, 128, 16), (2, 4, 64, 16), (1, 8, 128, 32), (3, 5, 96, 24), (1, 16, 64, 8), (1, 33, 128, 16), (2, 2, 256, 1),
    (1, 2, 192, 48), (1, 16, 256, 16), (1, 17, 192, 24), (2, 3, 32, 16), (1, 9, 32, 4), (2, 40, 64, 16), (1, 70, 96, 12), (1, 32, 256, 16), (2, 3, 80, 7), (1, 1, 1, 5), (1, 2, 500, 16), (1, 3, 33, 130)])
def test_paged_attention_shapes(client, dtype, kv_heads, group, dim, size):
    rng = np.random.default_rng(dim * 7 + size)
    k, v, table = cache(rng, LENGTHS, kv_heads, size, dim, dtype)
    q = put(rng.standard_normal((len(LENGTHS), kv_heads * group, dim)), dtype)
    attend(client, q, k, v, table, LENGTHS, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 5, 32, 40, 100, 1000])
@pytest.mark.parametrize("size,dim", [(16, 128), (12, 64), (16, 40)])
def test_paged_attention_window(client, dtype, window, size, dim):
    rng = np.random.default_rng(window)
    k, v, table = cache(rng, LENGTHS, 2, size, dim, dtype)
    q = put(rng.standard_normal((len(LENGTHS), 4, dim)), dtype)
    got = attend(client, q, k, v, table, LENGTHS, dtype, window=window)
    # pages before the window may be taken away: their keys are not read
    for b, n in enumerate(LENGTHS):
        table[b, : max(0, n - window) // size] = -7
    again = attend(client, q, k, v, table, LENGTHS, dtype, window=window)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [8, 16, 64])
def test_paged_attention_pages_that_are_none(client, dtype, size):
    rng = np.random.default_rng(5)
    lengths = [200, 200, 200, 64, 10 ** 6, -5]
    k, v, table = cache(rng, [200, 200, 200, 64, 200, 0], 2, size, 64, dtype)
    table[0, 1:3] = [-1, 10 ** 9]              # holes in the middle
    table[1] = -(2 ** 31)                      # nothing left
    table[2, 0] = k.shape[0]                   # one past the last
    full = table[4, : 200 // size]
    table[4] = np.resize(full, table.shape[1])  # a length beyond the table; pages shared and met again
    q = put(rng.standard_normal((6, 6, 64)), dtype)
    got = attend(client, q, k, v, table, lengths, dtype)
    assert not val(got[1]).any() and not val(got[5]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_paged_attention_scores(client, dtype):
    """Large, negative and equal scores; scale 0 and below."""
    rng = np.random.default_rng(6)
    lengths = [40, 300, 7]
    k, v, table = cache(rng, lengths, 1, 16, 64, dtype)
    q = rng.standard_normal((3, 3, 64))
    for factor, scale in ((1.0, 0.0), (1.0, -0.5), (100.0, None), (0.0, None)):
        attend(client, put(q * factor, dtype), k, v, table, lengths, dtype, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 40])
def test_paged_attention_infinities(client, dtype, dim):
    """A key of -inf score weighs nothing; where every score is -inf, or one is
    NaN or +inf, the answer is NaN, as softmax's is."""
    rng = np.random.default_rng(7)
    lengths = [50, 50, 50, 50]
    k, v, table = cache(rng, lengths, 1, 16, dim, dtype)
    kf = val(k)
    kf[..., 0] = 1.0
    kf[table[0, 1], 0, 3, 0] = -np.inf
    kf[table[1, :4], 0, :, 0] = -np.inf
    kf[table[2, 2], 0, 5, 0] = np.inf
    kf[table[3, 0], 0, 0, 1] = np.nan
    with np.errstate(all="ignore"):
        k = put(kf, dtype)
        q = np.abs(rng.standard_normal((4, 2, dim))) + 0.1
        (got,) = call(client, lambda b, p: b.paged_attention(*p), [put(q, dtype), k, v, table, np.array(lengths, np.int32)],
                      [dtype] * 3 + ["s32"] * 2)
    assert np.isnan(val(got[1:])).all() and np.isfinite(val(got[0])).all()
    table[0, 1], hole = -1, table[0, 1]
    kk = np.delete(val(k)[hole, 0], 3, 0)
    rest = [j for j in range(50) if j != 16 + 3]
    rows = [(hole if j // 16 == 1 else table[0, j // 16], j % 16) for j in rest]
    s = np.array([val(k)[pg, 0, i] for pg, i in rows]) @ val(put(q, dtype))[0].T * dim ** -0.5
    e = np.exp(s - s.max(0))
    want = (e.T @ np.array([val(v)[pg, 0, i] for pg, i in rows])) / e.sum(0)[:, None]
    assert np.isfinite(kk).all()
    finite = put(np.where(np.isfinite(kf), kf, 0), dtype)
    close(got[0], want, attention_tolerance(put(q[:1], dtype), finite, v, want, dtype, dim ** -0.5, 50))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths", [[5000], [3000, 1, 0, 17], [700] * 9 + [2500], [64] * 300, [1] * 70 + [900] * 3])
@pytest.mark.parametrize("group,dim", [(4, 128), (20, 64), (50, 32), (2, 72)])
def test_paged_attention_split_lengths(client, dtype, lengths, group, dim):
    """Long sequences cut into splits, many sequences, both beside short ones."""
    rng = np.random.default_rng(len(lengths))
    k, v, table = cache(rng, lengths, 1, 16, dim, dtype, extra=40)
    q = put(rng.standard_normal((len(lengths), group, dim)), dtype)
    got = attend(client, q, k, v, table, lengths, dtype)
    assert np.array_equal(got, attend(client, q, k, v, table, lengths, dtype))


def test_paged_attention_results_do_not_depend_on_the_pages_order(client):
    rng = np.random.default_rng(9)
    k, v, table = cache(rng, [700, 90], 2, 16, 128, "bf16")
    q = put(rng.standard_normal((2, 8, 128)), "bf16")
    got = attend(client, q, k, v, table, [700, 90], "bf16")
    perm = rng.permutation(k.shape[0])
    inv = np.argsort(perm)
    moved = np.where(table >= 0, inv[np.maximum(table, 0)], -1).astype(np.int32)
    assert np.array_equal(got, attend(client, q, k[perm], v[perm], moved, [700, 90], "bf16"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [40, 64, 128, 500])
def test_paged_attention_large_scores(client, dtype, dim):
    """Two keys of one score far past the rest, and past what exp2 takes: each
    weighs a half."""
    rng = np.random.default_rng(3)
    k, v = (put(x, dtype) for x in rng.standard_normal((2, 4, 1, 16, dim)))
    k[:, :, :, :] = put(np.full((4, 1, 16, dim), -2.0 ** 18), dtype)
    k[1, 0, 3], k[2, 0, 9] = (put(np.full(dim, 2.0 ** 17), dtype),) * 2
    q = put(np.full((1, 2, dim), 2.0 ** 17), dtype)
    table, n = np.array([[0, 1, 2, 3]], np.int32), np.array([60], np.int32)
    (got,) = call(client, lambda b, p: b.paged_attention(*p, scale=1.0), [q, k, v, table, n], [dtype] * 3 + ["s32"] * 2)
    want = (val(v)[1, 0, 3] + val(v)[2, 0, 9]) / 2
    close(got, np.broadcast_to(want, (1, 2, dim)), (U[dtype] + 2 * W) * np.abs(want) + 2 * W * np.abs(val(v)[1, 0, 3]))



@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kv_heads,group,dim,size", [(2, 4, 64, 16), (1, 20, 128, 8), (2, 1, 256, 16), (1, 3, 96, 24), (2, 2, 80, 16)])
def test_paged_attention_weights_are_not_rounded_to_the_type(client, dtype, kv_heads, group, dim, size):
    """Scores that are exact: small integers times a power of two. A weight is
    then off by its exponent's rounding (two of |x| w), its exponential's 4 w
    and, in 16 bits, by the square of the type's u, what two pieces of it leave;
    the sums by (n + 8) w. All of it counts by the weight's own share of the
    answer, in the numerator and in the denominator."""
    rng = np.random.default_rng(dim)
    lengths = [1, 3, 9, 33, 80, 500]
    k, v, table = cache(rng, lengths, kv_heads, size, dim, dtype, poison=False)
    k = put(rng.integers(-2, 3, k.shape), dtype)
    q = put(rng.integers(-2, 3, (len(lengths), kv_heads * group, dim)), dtype)
    scale = 2.0 ** -4
    (got,) = call(client, lambda b, p: b.paged_attention(*p, scale=scale), [q, k, v, table, np.array(lengths, np.int32)],
                  [dtype] * 3 + ["s32"] * 2)
    want = P.paged_attention(val(q), val(k), val(v), table, lengths, scale)
    share = P.paged_attention(val(q), val(k), np.abs(val(v)), table, lengths, scale)  # sum of p |v|
    x = 1.45 * scale * 4 * dim
    u2 = 0 if dtype == "f32" else U[dtype] ** 2
    weight = u2 + (2 * x + 4 + np.array(lengths)[:, None, None] + 8) * W
    close(got, want, 2 * weight * 2 * share + U[dtype] * np.abs(want))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [1, 20])
def test_paged_attention_many_small_weights(client, dtype, group):
    """One key of weight 1 and value 0 before 7,999 of weight e^-18, which is
    below f16's smallest number, and value 100. Sequences enough that one
    workgroup walks each: all of one page table."""
    n, size, dim, batch = 8000, 64, 64, 600
    pages = n // size
    k, v = np.zeros((2, pages, 1, size, dim))
    k[..., 0], v[...] = -18, 100
    k[0, 0, 0, 0] = v[0, 0, 0] = 0
    q = np.zeros((batch, group, dim))
    q[..., 0] = 1
    table = np.repeat(np.arange(pages, dtype=np.int32)[None], batch, 0)
    (got,) = call(client, lambda b, p: b.paged_attention(*p, scale=1.0),
                  [put(q, dtype), put(k, dtype), put(v, dtype), table, np.full(batch, n, np.int32)], [dtype] * 3 + ["s32"] * 2)
    s = (n - 1) * np.exp(-18.0)
    want = np.full((batch, group, dim), 100 * s / (1 + s))
    # sums of n weights in 32 bits, each off by its exponent's 2 x 26 w, its
    # exponential's 4 w and by u squared; the result's rounding
    u2 = 0 if dtype == "f32" else U[dtype] ** 2
    close(got, want, (2 * ((n + 56) * W + u2) + U[dtype]) * want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,group,size", [(64, 2, 16), (128, 20, 16), (256, 1, 8), (96, 3, 24), (40, 2, 16)])
def test_paged_attention_infinite_values(client, dtype, dim, group, size):
    """An attended key's infinite value makes its column's answer infinite, two
    of either sign, or a NaN, make it NaN; the other columns are as without."""
    rng = np.random.default_rng(dim)
    lengths = [50, 300, 33]
    k, v, table = cache(rng, lengths, 1, size, dim, dtype, poison=False)
    q = put(0.3 * rng.standard_normal((3, group, dim)), dtype)
    plain = P.paged_attention(val(q), val(k), val(v), table, lengths)
    vf = val(v)
    vf[table[0, 1], 0, 1, 3] = np.inf
    vf[table[1, 0], 0, 2, 5], vf[table[1, 2], 0, 1, 5] = np.inf, -np.inf
    vf[table[1, 1], 0, 0, 7] = -np.inf
    vf[table[2, 0], 0, 0, 9], vf[table[2, 0], 0, 1, 11] = np.nan, np.inf
    n = np.array(lengths, np.int32)
    (got,) = call(client, lambda b, p: b.paged_attention(*p), [q, k, put(vf, dtype), table, n], [dtype] * 3 + ["s32"] * 2)
    got = val(got)
    assert np.isposinf(got[0, :, 3]).all() and np.isneginf(got[1, :, 7]).all() and np.isposinf(got[2, :, 11]).all()
    assert np.isnan(got[1, :, 5]).all() and np.isnan(got[2, :, 9]).all()
    special = np.zeros((3, group, dim), bool)
    special[0, :, 3] = special[1, :, [5, 7]] = special[2, :, [9, 11]] = True
    tol = attention_tolerance(q, k, v, plain, dtype, dim ** -0.5, 300)
    assert (np.abs(got - plain) <= tol)[~special].all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size,dim", [(8, 64), (16, 128), (48, 64), (5, 96), (7, 40)])
def test_paged_attention_full_tables_at_the_pools_end(client, dtype, size, dim):
    """Sequences that fill their table, the last page the pool's last, with
    tables that end inside a 32-key tile."""
    rng = np.random.default_rng(size)
    for width in (1, 3, 11):
        pages, n = 2 * width, width * size
        k, v = (put(x, dtype) for x in rng.standard_normal((2, pages, 1, size, dim)))
        table = np.stack([rng.permutation(width), width + np.arange(width)]).astype(np.int32)
        q = put(rng.standard_normal((2, 3, dim)), dtype)
        attend(client, q, k, v, table, [n, n], dtype)
        attend(client, q, k, v, table, [n - 1, 2 ** 31 - 1], dtype, window=max(1, n // 2))


def test_paged_attention_rows_past_32_bits(client):
    """Pages of more than 2^32 bytes, written and read at their end."""
    pages, size, dim = 140000, 64, 256
    assert 2 * pages * size * dim > 2 ** 32
    b = Builder()
    knew, vnew, slots = b.param((128, 1, dim), "bf16"), b.param((128, 1, dim), "bf16"), b.param((128,), "s32")
    q, table, lengths = b.param((1, 4, dim), "bf16"), b.param((1, 3), "s32"), b.param((1,), "s32")
    zero = b.constant(0.0, "bf16")
    kp, vp = (b.broadcast_in_dim(zero, (pages, 1, size, dim), []) for _ in range(2))
    kp, vp = b.paged_append(kp, vp, knew, vnew, slots)
    exe = client.compile(b.build([b.paged_attention(q, kp, vp, table, lengths)]))
    rng = np.random.default_rng(10)
    kn, vn = (put(rng.standard_normal((128, 1, dim)), "bf16") for _ in range(2))
    qa = put(rng.standard_normal((1, 4, dim)), "bf16")
    last = pages - 2
    sl = (last * size + np.arange(128)).astype(np.int32)
    tb = np.array([[last, last + 1, -1]], np.int32)
    (got,) = exe(kn, vn, sl, qa, tb, np.array([100], np.int32), dtypes=["bf16", "bf16", None, "bf16", None, None])
    kd, vd = (x.reshape(2, 64, 1, dim).transpose(0, 2, 1, 3) for x in (kn, vn))
    want = P.paged_attention(val(qa), val(kd), val(vd), np.array([[0, 1]]), [100])
    close(got, want, attention_tolerance(qa, kd, vd, want, "bf16", dim ** -0.5, 100))


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("dtype,slot_type", [("bf16", "s32"), ("f16", "s64"), ("f32", "s32")])
@pytest.mark.parametrize("n,kv_heads,dim,size", [(1, 2, 64, 16), (7, 3, 80, 5), (300, 1, 33, 16), (1025, 2, 8, 32),
                                                 (4000, 1, 1, 64)])
def test_append(client, dtype, slot_type, n, kv_heads, dim, size):
    rng = np.random.default_rng(n)
    pages = max(3, -(-n // size))
    k, v = (put(x, dtype) for x in rng.standard_normal((2, pages, kv_heads, size, dim)))
    kn, vn = (put(x, dtype) for x in rng.standard_normal((2, n, kv_heads, dim)))
    # slots met again, negative ones and ones past the end among them
    slots = rng.integers(-2, pages * size + 2, n).astype(NP[slot_type])
    if n > 4:
        slots[[0, n // 2, n - 1]] = 3
        slots[1] = np.iinfo(NP[slot_type]).max
        slots[2] = np.iinfo(NP[slot_type]).min
    for donate in (False, True):
        b = Builder()
        p = [b.param(k.shape, dtype, donate=donate), b.param(k.shape, dtype, donate=donate), b.param(kn.shape, dtype),
             b.param(kn.shape, dtype), b.param((n,), slot_type)]
        exe = client.compile(b.build(list(b.paged_append(*p))))
        got = exe(k, v, kn, vn, slots, dtypes=[dtype if dtype == "bf16" else None] * 4 + [None])
        for g, w in zip(got, P.paged_append(k, v, kn, vn, slots)):
            assert np.array_equal(g.view(np.uint8), w.view(np.uint8))


def test_append_allocation_free_writes_the_callers_pages(client):
    """Outputs at the donated pages' own addresses: written there, other slots
    untouched. Outputs elsewhere: the pages stay as they were."""
    p = client.p
    rng = np.random.default_rng(3)
    k, v = (put(x, "bf16") for x in rng.standard_normal((2, 9, 2, 16, 64)))
    kn, vn = (put(x, "bf16") for x in rng.standard_normal((2, 5, 2, 64)))
    slots = np.array([3, 143, -1, 60, 3], np.int32)
    b = Builder()
    ps = [b.param(k.shape, "bf16", donate=True) for _ in range(2)] + [b.param(kn.shape, "bf16") for _ in range(2)]
    exe = client.compile(b.build(list(b.paged_append(*ps, b.param((5,), "s32")))))
    want = P.paged_append(k, v, kn, vn, slots)
    args = [DeviceArray.from_numpy(p, a) for a in (k, v, kn, vn, slots)]
    outs = [DeviceArray(p, k.nbytes) for _ in range(2)]

    def run(out_ptrs):
        exe.execute_noalloc([a.ptr for a in args], out_ptrs)
        p.hip_check(p.lib.pjrtx_hip_synchronize(0))

    def read(d):
        return d.to_numpy(np.uint16, k.shape)
    run([o.ptr for o in outs])
    assert all(np.array_equal(read(o), w) for o, w in zip(outs, want))
    assert np.array_equal(read(args[0]), k) and np.array_equal(read(args[1]), v)
    used = exe.execute_noalloc([a.ptr for a in args], [args[0].ptr, args[1].ptr])
    p.hip_check(p.lib.pjrtx_hip_synchronize(0))
    assert all(np.array_equal(read(a), w) for a, w in zip(args[:2], want)) and used < k.nbytes
    # the other way round: each output is the other's argument
    run([args[1].ptr, args[0].ptr])
    wk, wv = P.paged_append(*want, kn, vn, slots)
    assert np.array_equal(read(args[1]), wk) and np.array_equal(read(args[0]), wv)
    for d in args + outs:
        d.free()


def test_append_time_grows_as_its_rows_do(client):
    """2^20 rows are 16 times 2^16 of them, and the search for later rows of a
    slot no more: the square of 16 would be 256. Best of several, in one
    process, against the shorter call."""
    def best(n):
        b = Builder()
        pages, shape = (n // 64, 1, 64, 8), (n, 1, 8)
        p = [b.param(pages, "bf16", donate=True) for _ in range(2)] + [b.param(shape, "bf16") for _ in range(2)]
        exe = client.compile(b.build(list(b.paged_append(*p, b.param((n,), "s32")))))
        d = [DeviceArray(client.p, 16 * n) for _ in range(4)]
        d.append(DeviceArray.from_numpy(client.p, np.random.default_rng(n).permutation(n).astype(np.int32)))
        times = []
        for _ in range(6):
            client.p.hip_check(client.p.lib.pjrtx_hip_synchronize(0))
            t = time.perf_counter()
            exe.execute_noalloc([a.ptr for a in d], [d[0].ptr, d[1].ptr])
            client.p.hip_check(client.p.lib.pjrtx_hip_synchronize(0))
            times.append(time.perf_counter() - t)
        for a in d:
            a.free()
        return min(times)
    short, long = best(1 << 16), best(1 << 20)
    assert long <= 48 * short, (short, long)


@pytest.mark.parametrize("n", [8192, 8193, 50000])
def test_append_many_rows_of_equal_slots(client, n):
    """The last of the rows of a slot stays, however far apart they lie."""
    rng = np.random.default_rng(n)
    pages = (40, 2, 8, 4)
    k, v = (put(x, "bf16") for x in rng.standard_normal((2, *pages)))
    kn, vn = (put(x, "bf16") for x in rng.standard_normal((2, n, 2, 4)))
    slots = rng.integers(-3, 40 * 8 + 3, n).astype(np.int64)
    slots[n // 2:] = np.where(slots[n // 2:] % 2 == 0, -1, slots[n // 2:])  # even ones only in the first half
    got = call(client, lambda b, p: b.paged_append(*p), [k, v, kn, vn, slots], ["bf16"] * 4 + ["s64"])
    for g, w in zip(got, P.paged_append(k, v, kn, vn, slots)):
        assert np.array_equal(g, w)


# -------------------------------------------------------------------- norm

ROWS = [(1, 2048), (5, 1), (3, 7), (9, 64), (6, 500), (4, 513), (2, 1024), (3, 2056), (2, 4096), (3, 8191), (2, 16384),
        (1, 40001)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,dim", ROWS)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rms_norm(client, dtype, rows, dim, residual):
    rng = np.random.default_rng(dim)
    x, r = (put(a, dtype) for a in rng.standard_normal((2, rows, dim)) * 2)
    x[0] = 0
    if residual and rows > 1:
        r[0] = 0                              # a row of zeros: eps alone
    g = put(1 + 0.2 * rng.standard_normal(dim), dtype)
    args = [x, r, g] if residual else [x, g]
    eps = 1e-5
    want, total = P.add_rms_norm(val(x), val(r) if residual else None, val(g), eps)
    # the sum's rounding, dim squares, then a few operations
    rel = 2 * (2 * W + (dim + 16) * W)
    got = call(client, lambda b, p: b.add_rms_norm(p[0], p[1] if residual else None, p[-1], eps), args, [dtype] * len(args))
    close(got[0], want, (rel + U[dtype]) * np.abs(want) + 1e-30 + (6e-8 if dtype == "f16" else 0))
    if residual:
        close(got[1], total, U[dtype] * np.abs(total) + (6e-8 if dtype == "f16" else 0))
    q = call(client, lambda b, p: b.add_rms_norm(p[0], p[1] if residual else None, p[-1], eps, quantize=True), args,
             [dtype] * len(args))
    scale = np.abs(want).max(-1) / 127
    close(q[1], scale, 2 * (rel + 4 * W) * scale)
    assert q[0].dtype == np.int8
    safe = np.where(scale > 0, scale, 1)[:, None]
    # half a step, and what the quotient of up to 127 is off by
    assert (np.abs(q[0] - want / safe) <= 0.5 + 127 * 2 * (2 * rel + 8 * W)).all()
    assert np.abs(q[0].astype(int)).max() <= 127
    if residual:
        assert np.array_equal(q[2].view(np.uint8), got[1].view(np.uint8))


def test_add_rms_norm_keeps_leading_dims_and_takes_none(client):
    rng = np.random.default_rng(1)
    x, r = (put(a, "f32") for a in rng.standard_normal((2, 2, 3, 40)))
    g = put(np.ones(40), "f32")
    got = call(client, lambda b, p: b.add_rms_norm(*p, quantize=True), [x, r, g], ["f32"] * 3)
    assert [a.shape for a in got] == [(2, 3, 40), (2, 3), (2, 3, 40)]
    (one,) = call(client, lambda b, p: b.add_rms_norm(p[0], None, p[1]), [x[0, 0], g], ["f32"] * 2)
    close(one, P.add_rms_norm(val(x[0, 0]), None, val(g), 1e-5)[0], 1e-5)
    e = np.zeros((0, 40), np.float32)
    got = call(client, lambda b, p: b.add_rms_norm(*p), [e, e, g], ["f32"] * 3, noalloc=False)
    assert got[0].shape == (0, 40)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_add_rms_norm_not_finite(client, dtype):
    x = np.ones((4, 300))
    x[1, 7], x[2, 8], x[3, 9] = np.nan, np.inf, -np.inf
    x, r, g = put(x, dtype), put(np.zeros((4, 300)), dtype), put(np.ones(300), dtype)
    y, t = call(client, lambda b, p: b.add_rms_norm(*p), [x, r, g], [dtype] * 3)
    assert np.isnan(val(y)[1]).all() and np.isnan(val(y)[2, 8]) and np.isnan(val(y)[3, 9])
    assert (val(y)[2, :8] == 0).all() and np.array_equal(val(t), val(x), equal_nan=True)
    y8, scale, _ = call(client, lambda b, p: b.add_rms_norm(*p, quantize=True), [x, r, g], [dtype] * 3)
    assert np.isnan(scale[1:]).all() and scale[0] > 0 and (y8[0] == 127).all()


def test_add_rms_norm_infinite_gain_quantizes(client):
    """An infinite scale: +-127 stand for the infinities, 0 for what no value
    stands for."""
    x = np.full((2, 300), -1.0, np.float32)
    x[1, 5] = 0
    g = np.ones(300, np.float32)
    g[5], g[9] = np.inf, -np.inf
    y8, scale = call(client, lambda b, p: b.add_rms_norm(p[0], None, p[1], quantize=True), [x, g], ["f32"] * 2)
    assert scale[0] == np.inf and np.isnan(scale[1])
    assert y8[0, 5] == -127 and y8[0, 9] == 127 and not np.delete(y8[0], [5, 9]).any()


def test_add_rms_norm_small_rows_quantize(client):
    """Scales near the smallest floats: the quotients stay finite."""
    x = np.zeros((4, 64), np.float32)
    x[0, :2], x[1, :2], x[2, :2] = [1e-38, 5e-39], [1e-30, -1e-30], [2e-36, 1e-36]
    g = np.ones(64, np.float32)
    y8, scale = call(client, lambda b, p: b.add_rms_norm(p[0], None, p[1], 1.0, quantize=True), [x, g], ["f32"] * 2)
    back = y8 * scale[:, None].astype(np.float64)
    assert np.isfinite(scale).all() and (np.abs(back - x) <= 0.51 * scale[:, None] + 2e-44).all() and not y8[3].any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,dim", ROWS + [(1200, 96), (2000, 256), (700, 2048)])
@pytest.mark.parametrize("dsum", [True, False])
def test_add_rms_norm_grad(client, dtype, rows, dim, dsum):
    rng = np.random.default_rng(rows * dim)
    dy, ds, t = (put(a, dtype) for a in rng.standard_normal((3, rows, dim)))
    g = put(1 + 0.2 * rng.standard_normal(dim), dtype)
    eps = 1e-5
    args = [dy, ds, t, g] if dsum else [dy, t, g]
    dx, dg = call(client, lambda b, p: b.add_rms_norm_grad(p[0], p[1] if dsum else None, p[-2], p[-1], eps), args,
                  [dtype] * len(args))
    want, wg = P.add_rms_norm_grad(val(dy), val(ds) if dsum else None, val(t), val(g), eps)
    r = 1 / np.sqrt((val(t) ** 2).mean(-1, keepdims=True) + eps)
    n, dn = np.abs(val(t)) * r, np.abs(val(dy) * val(g))
    parts = (np.abs(val(ds)) if dsum else 0) + r * (dn + n * (dn * n).mean(-1, keepdims=True))
    small = 6e-8 if dtype == "f16" else 0
    close(dx, want, 2 * (dim + 24) * W * parts + U[dtype] * np.abs(want) + small)
    # n is off by dim squares' sum, the columns by their rows' sums
    mag = (np.abs(val(dy)) * n).sum(0)
    close(dg, wg, 2 * (dim + 24 + rows) * W * mag + U[dtype] * np.abs(wg) + small)


def test_add_rms_norm_grad_of_no_rows(client):
    e, g = np.zeros((0, 40), np.float32), np.ones(40, np.float32)
    dx, dg = call(client, lambda b, p: b.add_rms_norm_grad(p[0], None, p[1], p[2]), [e, e, g], ["f32"] * 3, noalloc=False)
    assert dx.shape == (0, 40) and not dg.any()


def test_add_rms_norm_grad_is_the_norms_difference(client):
    """Central differences of the kernel's own forward pass in 32 bits: a step
    of 2^-6 leaves 2 w |loss terms| / 2^-6 of rounding and a third-order term
    of at most the step squared."""
    rng = np.random.default_rng(4)
    x, r, dy, ds = rng.standard_normal((4, 2, 24)).astype(np.float32)
    g = (1 + 0.1 * rng.standard_normal(24)).astype(np.float32)
    b = Builder()
    fwd = client.compile(b.build(list(b.add_rms_norm(b.param((2, 24), "f32"), b.param((2, 24), "f32"), b.param((24,), "f32"), 0.1))))
    y, t = fwd(x, r, g)
    (dx, dg) = call(client, lambda b, p: b.add_rms_norm_grad(*p, eps=0.1), [dy, ds, t, g], ["f32"] * 4)

    def loss(x, g):
        y, t = fwd(x, r, g)
        return float((y.astype(np.float64) * dy).sum() + (t.astype(np.float64) * ds).sum())
    h = 2.0 ** -6
    for i in range(0, 24, 5):
        e = np.zeros_like(x)
        e[1, i] = h
        assert abs((loss(x + e, g) - loss(x - e, g)) / (2 * h) - dx[1, i]) < 50 * h * h
        e = np.zeros_like(g)
        e[i] = h
        assert abs((loss(x, g + e) - loss(x, g - e)) / (2 * h) - dg[i]) < 50 * h * h


# ---------------------------------------------------- token log probabilities

def logprob_tolerances(x, lse):
    """Of lse and of the entropy: sums of exponentials, a thread's in turn (a
    32nd of a chunk at a time), then over the threads and the splits; each
    exponential's argument is off by 4 w of its distance to the largest."""
    V = x.shape[1]
    depth = 32 * -(-V // 8192) + 80
    d = np.where(np.isfinite(x), lse[:, None] - x, 0)
    far = (np.exp(-d) * np.abs(d)).sum(1)            # the mean distance
    lse_tol = 2 * (depth * W + 6 * W * (1 + far)) + 4 * W * np.abs(lse)
    return lse_tol, 2 * (depth + 8) * W * (1 + 2 * far) + 8 * W * (1 + (np.exp(-d) * d * d).sum(1))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 5, 5), (2, 255, 0), (4, 1000, 20), (5, 8192, 7), (3, 8193, 128),
                                          (2, 32000, 5), (2, 50257, 20), (1, 128256, 64), (70, 999, 3)])
def test_token_logprobs(client, dtype, rows, vocab, k):
    rng = np.random.default_rng(vocab)
    x = put(rng.standard_normal((rows, vocab)) * 4, dtype)
    tok = rng.integers(0, vocab, rows).astype(np.int32)
    if rows > 2:
        tok[:2] = [-1, vocab]
    got = call(client, lambda b, p: b.token_logprobs(*p, top_k=k), [x, tok], [dtype, "s32"])
    want = P.token_logprobs(val(x), tok, k)
    lse_tol, ent_tol = logprob_tolerances(val(x), want[2])
    close(got[2], want[2], lse_tol)
    close(got[0], want[0], lse_tol + W * np.abs(want[0]))
    close(got[1], want[1], ent_tol)
    if rows > 2:
        assert got[0][0] == 0 and got[0][1] == 0
    if k:
        assert got[4].dtype == np.int32 and np.array_equal(got[4], want[4])
        close(got[3], want[3], lse_tol[:, None] + W * np.abs(want[3]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3000, 20000, 100000])
@pytest.mark.parametrize("shape", ["equal", "two", "rising", "falling", "late", "levels"])
def test_token_logprobs_ties_and_orders(client, dtype, vocab, shape):
    """Equal logits (the lowest ids), and orders that keep passing the bound."""
    rng = np.random.default_rng(8)
    i = np.arange(vocab)
    x = {"equal": 0 * i + 0.5, "two": np.where(i % 3 == 1, 2.0, -1.0), "rising": i / vocab * 8, "falling": -i / vocab * 8,
         "late": np.where(i >= vocab - 30, 3.0 + i * 1e-6, 0.0), "levels": rng.integers(0, 4, vocab) / 2.0}[shape]
    x = put(np.stack([x, x[::-1]]), dtype)
    got = call(client, lambda b, p: b.token_logprobs(*p, top_k=40), [x, np.zeros(2, np.int64)], [dtype, "s64"])
    want = P.token_logprobs(val(x), np.zeros(2, int), 40)
    assert np.array_equal(got[4], want[4])
    lse_tol, ent_tol = logprob_tolerances(val(x), want[2])
    close(got[1], want[1], ent_tol)
    close(got[3], want[3], lse_tol[:, None] + W * np.abs(want[3]))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_token_logprobs_not_finite(client, dtype):
    """Masked logits weigh nothing, the type's lowest value as -inf; NaN or +inf
    makes the row's numbers NaN, and a row of -inf has no distribution."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((6, 9000))
    lowest = {"bf16": -3.3895314e38, "f16": -65504.0, "f32": -3.4028235e38}[dtype]
    x[0, 3:] = -np.inf
    x[1, ::2] = -np.inf
    x[2, 5:] = lowest
    x[3, 8500] = np.nan
    x[4, 10] = np.inf
    x[5] = -np.inf
    x = put(x, dtype)
    tok = np.array([1, 0, 2, 0, 0, 0], np.int32)
    got = call(client, lambda b, p: b.token_logprobs(*p, top_k=5), [x, tok], [dtype, "s32"])
    with np.errstate(all="ignore"):
        want = P.token_logprobs(val(x[:3]), tok[:3], 5)
    lse_tol, ent_tol = logprob_tolerances(val(x[:3]), want[2])
    close(got[2][:3], want[2], lse_tol)
    close(got[0][:3], want[0], lse_tol + W * np.abs(np.nan_to_num(want[0], neginf=0)))
    close(got[1][:3], want[1], ent_tol)
    assert np.array_equal(got[4][:3], want[4]) and got[0][1] == -np.inf and np.isneginf(got[3][0, 3:]).all()
    assert np.isnan(got[0][3:]).all() and np.isnan(got[1][3:]).all() and np.isnan(got[2][3:5]).all() and got[2][5] == -np.inf
    assert got[4][3, 0] == 8500 and got[4][4, 0] == 10 and np.array_equal(got[4][5], np.arange(5))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 8192), (5, 8200), (300, 333), (2, 50257)])
def test_token_logprobs_grad(client, dtype, rows, vocab):
    rng = np.random.default_rng(vocab)
    x = put(rng.standard_normal((rows, vocab)) * 3, dtype)
    if vocab > 5:
        xf = val(x)
        xf[0, 2] = -np.inf
        x = put(xf, dtype)
    tok = rng.integers(0, vocab, rows).astype(np.int64)
    if rows > 2:
        tok[:2] = [-3, vocab]
    g, h = rng.standard_normal((2, rows)).astype(np.float32)
    h[-1] = 0
    with np.errstate(all="ignore"):
        _, H, lse = P.token_logprobs(val(x), tok)
        H, lse = H.astype(np.float32), lse.astype(np.float32)
        want = P.token_logprobs_grad(val(x), tok, lse.astype(np.float64), H.astype(np.float64), g, h)
        p = np.exp(val(x) - lse[:, None])
        d = np.where(p > 0, np.abs(val(x) - lse[:, None]), 0)
    (got,) = call(client, lambda b, p: b.token_logprobs_grad(*p), [x, tok, lse, H, g, h], [dtype, "s64"] + ["f32"] * 4)
    part = np.abs(g)[:, None] + np.abs(h)[:, None] * (d + np.abs(H)[:, None])
    hit = np.zeros_like(p)
    known = (tok >= 0) & (tok < vocab)
    hit[np.flatnonzero(known), tok[known]] = np.abs(g[known])
    close(got, want, 2 * W * (p * part * (8 + 4 * d) + hit) + U[dtype] * np.abs(want) + (6e-8 if dtype == "f16" else 1e-38))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_token_logprobs_grad_of_rows_left_out(client, dtype):
    """Padded rows: no gradient reaches them, and none comes out, also where
    they hold no distribution."""
    x = np.ones((5, 9000))
    x[0], x[1, 5], x[2, 7] = -np.inf, np.nan, np.inf
    tok = np.array([3, -1, 9000, -1, 4], np.int32)
    g, h = np.array([0, 5, -5, 7, 0], np.float32), np.zeros(5, np.float32)
    with np.errstate(all="ignore"):
        _, H, lse = (a.astype(np.float32) for a in P.token_logprobs(x, tok))
    (dx,) = call(client, lambda b, p: b.token_logprobs_grad(*p), [put(x, dtype), tok, lse, H, g, h],
                 [dtype, "s32"] + ["f32"] * 4)
    assert np.isnan(lse[:3]).all() and (val(dx) == 0).all()


def test_token_logprobs_grad_is_the_forward_passs_difference(client):
    rng = np.random.default_rng(11)
    x = rng.standard_normal((2, 30)).astype(np.float32)
    tok = np.array([4, 29], np.int32)
    g, h = rng.standard_normal((2, 2)).astype(np.float32)
    b = Builder()
    fwd = client.compile(b.build(list(b.token_logprobs(b.param((2, 30), "f32"), b.param((2,), "s32")))))
    _, H, lse = fwd(x, tok)
    (dx,) = call(client, lambda b, p: b.token_logprobs_grad(*p), [x, tok, lse, H, g, h], ["f32", "s32"] + ["f32"] * 4)

    def loss(x):
        lp, H, _ = fwd(x, tok)
        return float((lp.astype(np.float64) * g).sum() + (H.astype(np.float64) * h).sum())
    s = 2.0 ** -6
    for i in (0, 4, 17, 29):
        for r in range(2):
            e = np.zeros_like(x)
            e[r, i] = s
            assert abs((loss(x + e) - loss(x - e)) / (2 * s) - dx[r, i]) < 10 * s * s


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,k", [(50, 3), (9000, 0), (20001, 12), (600000, 4)])
def test_token_logprobs_large_logits(client, dtype, vocab, k):
    """Rows of nothing but a mask's value, and logits at any size: the
    distances to the largest count, not the logits' own size."""
    rng = np.random.default_rng(9)
    low = -3.38e38
    x = np.stack([np.full(vocab, -1e30), np.full(vocab, low), np.full(vocab, -low), np.full(vocab, -1e9),
                  1e9 + 64.0 * rng.integers(0, 3, vocab), np.where(np.arange(vocab) % 7, low, -low),
                  np.where(np.arange(vocab) % 5, low, 3.0), 1000 + rng.standard_normal(vocab),
                  -200 + rng.standard_normal(vocab), np.where(np.arange(vocab) == vocab - 1, 1e30, -5.0)])
    x = put(x, dtype)
    tok = rng.integers(0, vocab, len(x)).astype(np.int32)
    got = call(client, lambda b, p: b.token_logprobs(*p, top_k=k), [x, tok], [dtype, "s32"])
    want = P.token_logprobs(val(x), tok, k)
    # Nothing but lse itself is off by a part of its size: the tolerances are
    # those of the distances to the largest logit.
    m = val(x).max(1, keepdims=True)
    tol, ent_tol = logprob_tolerances(val(x) - m, np.log(np.exp(val(x) - m).sum(1)))
    close(got[2], want[2], tol + 4 * W * np.abs(want[2]))
    # Lowest less largest is -6.76e38, which rounds to -inf: past 2^128 - 2^103.
    rounded = np.where(want[0] < -(2.0 ** 128 - 2.0 ** 103), -np.inf, want[0])
    close(got[0], rounded, tol + 4 * W * np.abs(want[0]))
    close(got[1], want[1], ent_tol)
    if k:
        assert np.array_equal(got[4], want[4])
        close(got[3], want[3], tol[:, None] + 4 * W * np.abs(want[3]))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab,k,step", [(300, 4, 0.5), (9000, 0, 6.5), (40000, 0, 8.5), (40000, 4, 8.5)])
@pytest.mark.parametrize("equal", [1, 3])
def test_token_logprobs_wherever_the_largest_logit_lies(client, dtype, vocab, k, step, equal):
    """Rows with all their weight on `equal` tokens, at a largest logit of any
    size: log p is -log(equal) whatever that size is. The other weights are
    e^-110, below every float, so a sum of one weight over itself is 1 and log
    p is 0; of three it is off by their 3 roundings, the quotient's and the
    logarithm's 4 w of itself."""
    rng = np.random.default_rng(vocab)
    top = np.arange(-128, 128.5, step)
    x = np.repeat(top[:, None] - 110, vocab, 1)
    at = np.stack([rng.permutation(vocab)[:equal] for _ in top])
    at[::2] = (at[::2, :1] // 4 * 4 + np.arange(equal)) % vocab  # neighbours: one thread's
    np.put_along_axis(x, at, top[:, None], 1)
    x = put(x, dtype)
    assert np.array_equal(val(x).max(1), top)
    tok = at[:, -1].astype(np.int32)
    got = call(client, lambda b, p: b.token_logprobs(*p, top_k=k), [x, tok], [dtype, "s32"])
    want = np.log(equal)
    tol = 0 if equal == 1 else 2 * (4 + 4 * want) * W
    assert (np.abs(got[0] + want) <= tol).all(), np.abs(got[0] + want).max()
    assert (got[0] <= 0).all() and (np.abs(got[1] - want) <= tol + W).all()
    assert (np.abs(got[2] - (top + want)) <= tol + W * np.abs(top + want)).all()
    if k:
        assert (np.abs(got[3][:, :equal] + want) <= tol).all()
        assert np.array_equal(got[4][:, :equal], np.sort(at, 1))


@pytest.mark.parametrize("vocab", [300, 9000, 40000])
def test_token_logprobs_entropy_is_not_negative(client, vocab):
    """0 where one token has all the weight, at a largest logit of any size."""
    top = np.arange(-130, 130.5, 0.5)
    x = np.repeat(top[:, None] - 110, vocab, 1).astype(np.float32)
    x[:, 7] = top
    got = call(client, lambda b, p: b.token_logprobs(*p), [x, np.full(len(top), 7, np.int32)], ["f32", "s32"])
    assert (got[1] >= 0).all() and (got[1] <= W).all() and (got[0] == 0).all()


# ---------------------------------------------------- the caller's addresses

def _off(client, a, by):
    """Device memory that holds `a` from `by` bytes on."""
    raw = np.zeros(a.nbytes + by, np.uint8)
    raw[by:] = np.ascontiguousarray(a).view(np.uint8).ravel()
    return DeviceArray.from_numpy(client.p, raw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("what", ["attention", "any", "append", "norm", "quantized", "norm_grad", "long_grad", "logprobs",
                                  "logprobs_grad"])
def test_addresses_are_an_elements(client, dtype, what):
    """Arguments and outputs at any element's address: the bits of aligned ones."""
    rng = np.random.default_rng(12)
    r = lambda *shape: put(rng.standard_normal(shape), dtype)  # noqa: E731
    ints = lambda *v: np.array(v, np.int32)  # noqa: E731
    f = lambda n: rng.standard_normal(n).astype(np.float32)  # noqa: E731
    table = np.array([[3, 1, 0, 2], [2, 0, 3, -1]], np.int32)
    dim = 64 if what == "attention" else 40
    args, build = {
        "attention": ([r(2, 6, dim), r(4, 2, 16, dim), r(4, 2, 16, dim), table, ints(60, 33)], lambda b, p: [b.paged_attention(*p)]),
        "any": ([r(2, 6, dim), r(4, 2, 16, dim), r(4, 2, 16, dim), table, ints(60, 33)], lambda b, p: [b.paged_attention(*p)]),
        "append": ([r(4, 2, 16, 32), r(4, 2, 16, 32), r(5, 2, 32), r(5, 2, 32), ints(3, 9, 3, 60, -1)],
                   lambda b, p: b.paged_append(*p)),
        "norm": ([r(5, 1032), r(5, 1032), r(1032)], lambda b, p: b.add_rms_norm(*p)),
        "quantized": ([r(5, 1032), r(5, 1032), r(1032)], lambda b, p: b.add_rms_norm(*p, quantize=True)),
        "norm_grad": ([r(9, 520), r(9, 520), r(9, 520), r(520)], lambda b, p: b.add_rms_norm_grad(*p)),
        "long_grad": ([r(3, 9000), r(3, 9000), r(3, 9000), r(9000)], lambda b, p: b.add_rms_norm_grad(*p)),
        "logprobs": ([r(3, 9000), ints(1, 2, 3)], lambda b, p: b.token_logprobs(*p, top_k=7)),
        "logprobs_grad": ([r(3, 9000), ints(1, 2, 3), f(3) + 9, f(3), f(3), f(3)], lambda b, p: [b.token_logprobs_grad(*p)]),
    }[what]
    names = {np.dtype(np.uint16): "bf16", np.dtype(np.float32): "f32", np.dtype(np.int32): "s32"}
    b = Builder()
    exe = client.compile(b.build(list(build(b, [b.param(a.shape, names[a.dtype]) for a in args]))))
    want = exe(*args, dtypes=["bf16" if a.dtype == np.uint16 else None for a in args])
    size = 2 if dtype == "bf16" else 4
    for by in (size, 3 * size):
        ins = [_off(client, a, by * a.dtype.itemsize // size) for a in args]
        outs = [DeviceArray(client.p, w.nbytes + by * w.dtype.itemsize // size) for w in want]
        exe.execute_noalloc([d.ptr + by * a.dtype.itemsize // size for d, a in zip(ins, args)],
                            [d.ptr + by * w.dtype.itemsize // size for d, w in zip(outs, want)])
        client.p.hip_check(client.p.lib.pjrtx_hip_synchronize(0))
        for d, w in zip(outs, want):
            at = by * w.dtype.itemsize // size
            got = d.to_numpy(np.uint8, (w.nbytes + at,))[at:]
            assert np.array_equal(got, w.view(np.uint8).ravel())
        for d in ins + outs:
            d.free()


@pytest.mark.parametrize("by", [2, 6, 16, 256])
def test_results_that_other_steps_read(client, by):
    """A norm of keys that is a result, at any address, and attention's operand,
    whose kernels load whole vectors: the bits of aligned ones."""
    rng = np.random.default_rng(14)
    x, q, v = (put(rng.standard_normal((1, 256, 4, 128)), "bf16") for _ in range(3))
    g, zero = put(np.ones(128), "bf16"), np.array(0, np.int32)
    b = Builder()
    ps = [b.param(x.shape, "bf16") for _ in range(3)] + [b.param((128,), "bf16"), b.param((), "s32")]
    (k,) = b.add_rms_norm(ps[0], None, ps[3])
    o = b.custom_call("pjrtx.mlx_metal.scaled_dot_product_attention", [ps[1], k, ps[2], ps[4]], x.shape, "bf16")
    w = b.dot_general(b.reshape(k, (1024, 128)), b.reshape(ps[1], (1024, 128)), contract=((0,), (0,)))
    exe = client.compile(b.build([k, o, w]))
    want = exe(x, q, v, g, zero, dtypes=["bf16"] * 4 + [None])
    ins = [DeviceArray.from_numpy(client.p, a) for a in (x, q, v, g, zero)]
    outs = [DeviceArray(client.p, a.nbytes + by) for a in want]
    for _ in range(2):
        exe.execute_noalloc([d.ptr for d in ins], [d.ptr + by for d in outs])
        client.p.hip_check(client.p.lib.pjrtx_hip_synchronize(0))
        for d, a in zip(outs, want):
            assert np.array_equal(d.to_numpy(np.uint8, (a.nbytes + by,))[by:], a.view(np.uint8).ravel())
    for d in ins + outs:
        d.free()


# ------------------------------------------------------------ inside a loop

def test_append_and_attention_inside_a_while_loop(client):
    """Steps of a decode loop on the device: each appends a row and attends."""
    rng = np.random.default_rng(13)
    steps, dim = 20, 64
    k, v = (put(x, "bf16") for x in rng.standard_normal((2, 6, 2, 8, dim)))
    table = np.array([[4, 1, 5, 0, 2, 3]], np.int32)
    rows = put(rng.standard_normal((steps, 2, dim)), "bf16")
    q = put(rng.standard_normal((1, 4, dim)), "bf16")
    b = Builder()
    kp, vp = b.param(k.shape, "bf16", donate=True), b.param(v.shape, "bf16", donate=True)
    tb, rp, qp = b.param(table.shape, "s32"), b.param(rows.shape, "bf16"), b.param(q.shape, "bf16")
    n, size, one, zero = b.constant(steps, "s32"), b.constant(8, "s32"), b.constant(1, "s32"), b.constant(0, "s32")
    outs = b.broadcast_in_dim(b.constant(0.0, "bf16"), (steps, 4, dim), [])

    def body(i, kc, vc, o):
        row = b.dynamic_slice(rp, [i, zero, zero], (1, 2, dim))
        page = b.dynamic_slice(tb, [zero, b.divide(i, size)], (1, 1))
        slot = b.add(b.multiply(b.reshape(page, ()), size), b.remainder(i, size))
        kc, vc = b.paged_append(kc, vc, row, row, b.reshape(slot, (1,)))
        a = b.paged_attention(qp, kc, vc, tb, b.reshape(b.add(i, one), (1,)))
        return [b.add(i, one), kc, vc, b.dynamic_update_slice(o, a, [i, zero, zero])]

    end = b.while_loop([zero, kp, vp, outs], lambda i, *_: b.compare("LT", i, n), body)
    got_k, got_v, got = client.compile(b.build([end[1], end[2], end[3]]))(k, v, table, rows, q,
                                                                          dtypes=["bf16", "bf16", None, "bf16", "bf16"])
    slots = np.array([table[0, i // 8] * 8 + i % 8 for i in range(steps)])
    wk, wv = P.paged_append(k, v, rows, rows, slots)
    assert np.array_equal(got_k, wk) and np.array_equal(got_v, wv)
    for i in range(steps):
        want = P.paged_attention(val(q), val(wk), val(wv), table, [i + 1])
        close(got[i:i + 1], want, attention_tolerance(q, wk, wv, want, "bf16", dim ** -0.5, i + 1))
