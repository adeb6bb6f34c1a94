"""Infinite keys against small query elements: a score of -inf leaves its position out however small the element is."""
import math

import numpy as np
import pytest

from test_gpu_paged import HALF, KINDS, U, Pool, _attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("dim,rep", [(64, 2), (128, 9), (256, 1)])
@pytest.mark.parametrize("small", [2.0 ** -10, 2.0 ** -24, 1e-9, 2.0 ** -41, 1e-20, 1e-36])
def test_attention_infinite_keys_and_small_query_elements(act, cache, dim, rep, small, cuda_ok):
    """f32 queries over 16-bit caches are split into terms of which the first may be 0; the first is what decides here.
    Elements of a query of 16 bits that are 0 in its type are given as the smallest that are not."""
    lens = [40, 33, 20]
    pool = Pool(lens, 16, 1, dim, cache, seed=dim + rep)
    q = np.abs(np.random.default_rng(rep).standard_normal((3, rep, dim))).astype(np.float32) + 0.5
    least = max(small, 2.0 ** -24) if act == "f16" else small
    q[:, :, 0], q[:, :, 5] = least, -least
    pg = pool.table
    pool.full[0][pg[0, 1], 0, 3, 0] = -math.inf   # position 19 of sequence 0: -inf
    pool.full[0][pg[0, 0], 0, 2, 5] = math.inf    # position 2: -inf as well
    for p in range(33):                           # all of sequence 1
        pool.full[0][pg[1, p // 16], 0, p % 16, p % 2 * 5] = math.inf if p % 2 else -math.inf
    qd, out, lse = _attend(pool, act, rep, 0.125, q=q)
    assert (qd[:, :, 0] > 0).all()
    assert (out[1] == 0).all() and (lse[1] == -np.inf).all()
    for s, use in ((0, np.setdiff1d(np.arange(40), [2, 19])), (2, np.arange(20))):
        k, v = pool.rows(0, s, lens[s])[0][use], pool.rows(1, s, lens[s])[0][use]
        for h in range(rep):
            x = 0.125 * (k @ qd[s, h])
            e = np.exp(x - x.max())
            ref, n = e @ v / e.sum(), len(use)
            ds = (dim + 4) * U * (0.125 * np.abs(k) @ np.abs(qd[s, h])).max()
            tol = (2 * ds + (2 * n + 32) * U + 2.0 ** -16) * (e @ np.abs(v) / e.sum()) + HALF[act] * np.abs(ref)
            assert (np.abs(out[s, h] - ref) <= tol).all(), (s, h, out[s, h], ref)
            assert abs(lse[s, h] - (x.max() + math.log(e.sum()))) <= ds + (2 * n + 32) * U + 4 * U * abs(lse[s, h])
