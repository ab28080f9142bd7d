"""How many bits each path of paged attention keeps, against 64 bits.  Results are f32, so that no rounding of them hides the others.

A row is O = sum_j w_j c_j / sum_j p_j, in f32 but for the weights of the second product.  Those are, and are off by at most

    16-bit cache, bf16 program       p in bf16                                  2^-8 p
    16-bit cache, f16 program        p in f16, 2^14 under the largest           2^-11 p + 2^-39 max p
    8-bit cache, few rows            p v_scale in f16, 2^14 under the largest   2^-11 p vs + 2^-39 max (p vs)
    8-bit cache, chunks, f16         p v_scale in bf16 and what that lost       2^-16 p vs
    8-bit cache, chunks, bf16        p v_scale in bf16                          2^-8 p vs

(the spacing of f16 is 2^-24 below 2^-14, so half of it 2^-25; the largest weight stands at 2^14).  A score is an f32 sum of D products
times a scale: D 2^-24 S with S = scale sum_d |q_d k_d|; forming the exponent, the hardware's exponential and logarithm are within
2^-20 (1 + S), over few rows of codes 2^-20 (1 + S + |log v_scale|), and move p by that share, numerator and denominator alike.  The
sum of n weights in the order of the tiles: n 2^-24 of the sum of magnitudes, at most 2^-14 here beyond 1024 keys (f32 sums of partial
sums of a few hundred terms each)."""
import numpy as np
import pytest

import tessera_oracle as orc
from test_gpu_paged import attend, from_bits, make, reference, to_bits

pytestmark = pytest.mark.gpu

FORMATS = [("storage", "bf16"), ("storage", "f16"), ("i8", "bf16"), ("i8", "f16"), ("e4m3", "bf16"), ("e4m3", "f16")]


def few_rows(c, hq, new):
    D = c.dims[3]
    return hq // c.dims[2] * max(new) <= (128 if D <= 64 else 64 if D <= 128 else 32)


def hold(o, lse, ref, c, hq, new, slots, tail=1.0):
    """The table above.  ``tail``: most keys a row sees times the largest weight's share of one (the absolute part's factor)."""
    O, L, A, S = ref
    few, D = few_rows(c, hq, new), c.dims[3]
    f16_weights = few if c.fmt != "storage" else c.dtype == "f16"
    unit = 2.0 ** -11 if f16_weights else 2.0 ** -16 if c.fmt != "storage" and c.dtype == "f16" else 2.0 ** -8
    every = np.concatenate(slots)
    keys = max(len(s) for s in slots)
    at = (every // c.dims[1], every % c.dims[1])
    vs = np.abs(c.vs[at].astype(np.float64)) if c.fmt != "storage" else np.ones(1)
    logs = float(np.abs(np.log(np.maximum(vs, 1e-25))).max()) if few and c.fmt != "storage" else 0.0
    score = D * 2.0 ** -24 * S + 2.0 ** -20 * (1 + S + logs)
    sums = 2.0 ** -24 * min(keys, 1024)
    tol = (unit + sums + 2 * score[..., None]) * A + 1e-30
    if f16_weights:
        top = {"storage": 6.0, "i8": 127.0, "e4m3": 448.0}[c.fmt] if c.fmt != "storage" else float(np.abs(from_bits(c.v[at], c.dtype)).max())
        tol = tol + 2.0 ** -39 * keys * tail * float(vs.max()) * top
    assert np.all(np.abs(o - O) <= tol), float(np.max(np.abs(o - O) / tol))
    seen = np.isfinite(L)
    assert np.array_equal(seen, np.isfinite(lse))
    assert np.all(np.abs(lse[seen] - L[seen]) <= (score + sums + 2.0 ** -21 * np.abs(np.where(seen, L, 0)) + 1e-6)[seen])


# rows of few keys: nothing averages a weight's rounding away
SHORT = [([1] * 12, list(range(1, 13)), 4, 2, 64), ([1, 2, 4], [3, 9, 20], 8, 2, 128), ([1] * 3, [2, 5, 33], 4, 2, 256),
         ([70], [70], 4, 2, 64), ([40, 90], [45, 90], 8, 2, 128), ([40], [40], 4, 2, 256), ([2] * 20, [6 + b for b in range(20)], 4, 2, 128)]


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("new,kv,hq,hkv,D", SHORT)
def test_weights_keep_their_bits(lane, fmt, dtype, new, kv, hq, hkv, D):
    c, table, slots, q = make(lane, new, kv, hq=hq, hkv=hkv, D=D, page=16, fmt=fmt, dtype=dtype, seed=31)
    o, lse = attend(lane, c, table, q, new, kv, hq)
    hold(o, lse, reference(c, slots, q, new, kv, hq), c, hq, new, slots)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("new,kv,hq,hkv,D", [([1, 1, 3], [4, 60, 9], 4, 2, 64), ([1], [7000], 4, 1, 128), ([1] * 6, [40, 2500, 800, 3, 1, 900], 8, 2, 128),
                                             ([90], [100], 4, 2, 64), ([60], [3000], 4, 1, 128)])
def test_values_of_all_magnitudes(lane, fmt, dtype, new, kv, hq, hkv, D):
    """V rows from 1e-4 (codes: 1e-6) to 1e4, K rows over a factor of a hundred: scales of one call orders of magnitude apart, uncut and cut sequences,
    and a key that takes most of the probability while its V is among the smallest."""
    rng = np.random.default_rng(kv[0])
    c, table, slots, q = make(lane, new, kv, hq=hq, hkv=hkv, D=D, page=16, fmt=fmt, dtype=dtype, seed=32, spread=0.5)
    low = -6 if fmt != "storage" else -4 if dtype == "bf16" else -2
    first = 0
    for s, n in zip(slots, new):
        k = rng.standard_normal((len(s), hkv, D)) * 10.0 ** rng.uniform(-1, 1, (len(s), hkv, 1))
        v = rng.standard_normal((len(s), hkv, D)) * 10.0 ** rng.uniform(low, 4, (len(s), hkv, 1))
        j = len(s) // 2
        for h in range(hkv):                                   # aligned with the last token's first query head of the group
            x = from_bits(q[first + n - 1, h * hq // hkv], dtype).astype(np.float64)
            k[j, h] = x * 12 / (D ** -0.5 * (x @ x))
            v[j, h] = rng.standard_normal(D) * 10.0 ** low
        c.put(s, k.astype(np.float32), v.astype(np.float32))
        first += n
    o, lse = attend(lane, c, table, q, new, kv, hq)
    hold(o, lse, reference(c, slots, q, new, kv, hq), c, hq, new, slots)


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("new,kv", [([1], [131072]), ([1, 1], [5000, 300]), ([2] * 20, [900] * 20), ([33], [40000])])
def test_a_long_flat_tail_under_one_key(lane, fmt, dtype, new, kv):
    """One key 17.4 above all others: each of the others has 2.8e-8 of its weight, all together 3.6e-3 at 131072 keys, and they hold every
    column in which that key's value is zero."""
    hq, hkv, D = 4, 2, 64
    rng = np.random.default_rng(5)
    c, table, slots, _ = make(lane, new, kv, hq=hq, hkv=hkv, D=D, page=256, fmt=fmt, dtype=dtype, seed=33)
    x = rng.standard_normal((hkv, D))
    q = to_bits(np.broadcast_to(x.repeat(hq // hkv, 0), (sum(new), hq, D)), dtype)
    held = from_bits(to_bits(x, dtype), dtype).astype(np.float64)
    for b, s in enumerate(slots):
        k = np.zeros((len(s), hkv, D), np.float32)
        v = (1 + 0.5 * rng.random((len(s), hkv, D))).astype(np.float32)
        v[:, :, 3] = 2.0                                       # every V scale the same
        at = len(s) // 3
        k[at] = held * (17.4 / (D ** -0.5 * (held * held).sum(-1, keepdims=True)))
        v[at, :, ::2] = 0
        c.put(s, k, v)
    o, lse = attend(lane, c, table, q, new, kv, hq)
    ref = reference(c, slots, q, new, kv, hq)
    hold(o, lse, ref, c, hq, new, slots)
    if fmt != "storage" and few_rows(c, hq, new) or fmt == "storage" and dtype == "f16":
        assert np.all(np.abs(o[..., ::2] - ref[0][..., ::2]) <= 2.0 ** -7 * np.abs(ref[0][..., ::2]) + 1e-30)


@pytest.mark.parametrize("scale", (-0.3, 0.0, 1e-7, 2.0))
@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("new,kv", [([1, 2], [70, 300]), ([1], [3000]), ([100], [180])])
def test_any_finite_scale_over_every_format(lane, scale, fmt, dtype, new, kv):
    c, table, slots, q = make(lane, new, kv, hq=4, hkv=2, D=64, page=16, fmt=fmt, dtype=dtype, seed=34)
    o, lse = attend(lane, c, table, q, new, kv, 4, scale=scale)
    hold(o, lse, reference(c, slots, q, new, kv, 4, scale=scale), c, 4, new, slots)


@pytest.mark.parametrize("fmt", ("storage", "i8", "e4m3"))
@pytest.mark.parametrize("softcap", (0.0, 20.0, 1e6))
@pytest.mark.parametrize("new,kv", [([1, 1], [100, 0]), ([1], [5000]), ([2] * 5, [900] * 5), ([60, 1], [200, 3]), ([50], [6000])])
def test_scores_under_any_sentinel_over_every_format(lane, fmt, softcap, new, kv):
    """Every visible score is near -8e32, or at the cap's lower end: finite and equal, so a row is the mean of the values it sees."""
    c, table, slots, q = make(lane, new, kv, hq=4, hkv=2, D=64, page=16, fmt=fmt, dtype="bf16", seed=35)
    q = to_bits(np.full(q.shape, 1e15), "bf16")
    for s in slots:
        at = (s // 16, s % 16)
        if fmt == "storage":
            c.k[at] = to_bits(np.float32(-1e17), "bf16")
        else:
            codes, scales = orc.kv_quantise(np.full((1, 64), -1e17, np.float32), fmt)
            c.k[at], c.ks[at] = codes.view(np.uint8)[0], scales[0]
    o, lse = attend(lane, c, table, q, new, kv, 4, softcap=softcap)
    first, unit = 0, 2.0 ** -8
    for b, n in enumerate(new):
        keys, values = c.values(slots[b])
        for i in range(n):
            lo, hi = orc.key_bounds(i, n, kv[b], True, 0)
            if hi < lo:
                assert not o[first + i].any() and np.all(lse[first + i] == -np.inf)
                continue
            score = float(keys[lo, 0].sum()) * float(from_bits(q[:1, 0, 0], "bf16")[0]) * 64 ** -0.5
            want = max(score, -softcap) if softcap else score
            seen = values[lo:hi + 1].repeat(2, axis=1)
            assert np.all(np.abs(o[first + i] - seen.mean(0)) <= (unit + (len(seen) + 4) * 2.0 ** -24) * np.abs(seen).mean(0) + 1e-7)
            assert np.all(np.abs(lse[first + i] - want - (np.log(len(seen)) if softcap else 0)) <= 64 * 2.0 ** -24 * abs(want) + 1e-4)
        first += n
