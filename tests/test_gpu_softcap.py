"""Attention under soft caps from ordinary ones to caps far above every score, paged and contiguous, against 64 bits.

cap tanh(s / cap) of a score s is s itself, nearly, where the cap is large, so a result's error may not grow with the cap.  Bounds, in
the score's units: an f32 sum of D products is off by at most D 2^-24 S, S = scale sum_d |q_d k_d|, and |d cap tanh(s / cap) / ds| <= 1;
forming the exponent costs a few roundings of it, within 2^-20 (1 + S); under a cap of at most 64 the form -1 / (1 + e^(2 s / cap)) is off by up to
2^-24 from each of its three steps and is multiplied by 2 cap: 2^-21 cap.  Such an error moves a probability by that share,
numerator and denominator alike, and the LSE by itself.  A probability is rounded once (bf16 2^-8, f16 2^-11 of itself)."""
import numpy as np
import pytest

import tessera_oracle as orc
from tessera_amd import bf16 as b16
from test_gpu_paged import attend, make, reference

pytestmark = pytest.mark.gpu

CAPS = (0.5, 30.0, 64.0, 64.5, 1e3, 1e5, 1e8, 1e30, 3e38)


def hold(o, lse, ref, D, cap, unit, absolute=1e-6):
    O, L, A, S = ref
    score = D * 2.0 ** -24 * S + 2.0 ** -20 * (1 + S) + (2.0 ** -21 * cap if cap <= 64 else 0.0)
    tol = (unit + 2 * score[..., None]) * A + absolute
    assert np.all(np.abs(o - O) <= tol), float(np.max(np.abs(o - O) / tol))
    off = np.abs(lse - L) / (score + 2.0 ** -21 * np.abs(L) + 1e-6)
    assert np.all(off <= 1), float(off.max())


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("fmt,dtype", [("storage", "f16"), ("storage", "bf16"), ("e4m3", "bf16"), ("i8", "f16")])
@pytest.mark.parametrize("new,kv,D", [([1, 3, 1], [1, 400, 700], 64), ([140, 65], [300, 65], 128), ([60], [200], 256)])
@pytest.mark.parametrize("spread", (1.0, 50.0))
def test_paged(lane, cap, fmt, dtype, new, kv, D, spread):
    """Few rows and tiles; scores of a few and of a hundred and more (the bend of the caps between)."""
    c, table, slots, q = make(lane, new, kv, hq=4, hkv=2, D=D, page=16, fmt=fmt, dtype=dtype, seed=21, spread=spread)
    o, lse = attend(lane, c, table, q, new, kv, 4, softcap=cap)
    unit = 2.0 ** -11 if fmt == "storage" and dtype == "f16" else 2.0 ** -8
    hold(o, lse, reference(c, slots, q, new, kv, 4, softcap=cap), D, cap, unit, 1e-6 + 2.0 ** -25 * max(kv) * 6)


@pytest.mark.parametrize("cap", CAPS + (np.inf,))
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("Sq,Sk,D,bias", [(1, 40, 64, False), (150, 300, 64, True), (200, 200, 128, False), (70, 130, 256, False), (33, 90, 80, False)])
def test_contiguous(lane, cap, dtype, Sq, Sk, D, bias):
    """The same for K and V of one length for the batch, with an additive bias behind the cap; a cap of infinity is none."""
    from tessera_amd import ops
    rng = np.random.default_rng(Sq)
    hq, hkv = 4, 2
    to = (lambda x: b16.from_float32(x.astype(np.float32))) if dtype == "bf16" else (lambda x: x.astype(np.float16))
    back = (lambda x: x.to_float32()) if dtype == "bf16" else (lambda x: x.astype(np.float32))
    q, k, v = to(rng.standard_normal((1, hq, Sq, D)) * 20), to(rng.standard_normal((1, hkv, Sk, D))), to(rng.standard_normal((1, hkv, Sk, D)))
    B = rng.standard_normal((1, hq, Sq, Sk)).astype(np.float32) if bias else None
    o, lse = ops.gqa_attention(q, k, v, causal=True, logit_softcap=cap, attn_bias=B, return_lse=True, out="f32")
    first = lambda x: np.ascontiguousarray(back(x)[0].swapaxes(0, 1)).astype(np.float64)  # noqa: E731
    Q, K, V = first(q), first(k), first(v)
    O, A = np.zeros((Sq, hq, D)), np.zeros((Sq, hq, D))
    L, S = np.zeros((Sq, hq)), np.zeros((Sq, hq))
    for i in range(Sq):
        lo, hi = orc.key_bounds(i, Sq, Sk, True, 0)
        for h in range(hq):
            kh, vh = K[lo:hi + 1, h // 2], V[lo:hi + 1, h // 2]
            s = kh @ Q[i, h] * D ** -0.5
            S[i, h] = np.max(np.abs(kh) @ np.abs(Q[i, h])) * D ** -0.5
            if np.isfinite(cap):
                s = cap * np.tanh(s / cap)
            if bias:
                s = s + B[0, h, i, lo:hi + 1]
            p = np.exp(s - s.max())
            L[i, h] = s.max() + np.log(p.sum())
            p /= p.sum()
            O[i, h], A[i, h] = p @ vh, p @ np.abs(vh)
    unit = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
    hold(np.ascontiguousarray(np.asarray(o)[0].swapaxes(0, 1)), np.ascontiguousarray(np.asarray(lse)[0].T), (O, L, A, S), D, cap, unit,
         1e-6 + 2.0 ** -25 * Sk * 6)
